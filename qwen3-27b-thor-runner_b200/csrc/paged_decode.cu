// Attention of few new tokens over the paged cache (decode, verification of drafted tokens): one pass over keys and values, split
// over the sequences' lengths and joined.
//
//   out_r = sum_j 2^(t_rj - m_r) v_j / sum_j 2^(t_rj - m_r),   t_rj = scale * log2(e) * q_r . k_j,   m_r a running maximum
//
// The bound is HBM: a key and its value are 4 * head_dim bytes and meet only the rows of one key-value head, group * new tokens of
// them, up to 16 of which share a tile of mma.sync m16n8k16 (two FLOPs a byte and row; the warp MMA reaches a hundred times that).  So
// everything serves the stream of keys and values:
//  * Work is cut into units of 16 tokens for each of the block's warps (or pairs of warps), over all sequences, heads and row tiles in order, and each
//    block (one per SM) takes a run of consecutive units of about the same cost, counted on the device from the lengths as they are.  A block so holds
//    whole (sequence, head, row tile) items and at most two parts of split ones.
//  * A warp loads its own 16 tokens by TMA, a page's or half a page's piece at a time, into a ring of its own and multiplies them alone, with a running
//    maximum and sum of its own: no barrier between warps inside an item, two stages always under way (128 KB of loads in flight on an SM), and
//    the loads run on across the borders of items.  Pages that are no multiple of eight tokens come by cp.async, 16 bytes a thread (at pages of 16
//    and 32 tokens nearly as fast: 64 sequences, heads of 256, TMA 83, cp.async 82 us; 243 sequences, heads of 128, 109 and 111).
//  * Scores, maxima, sums and results stay in registers.  The weights 2^(t - m) enter the second product as two BF16 operands, the rounded weight and
//    what its rounding left (2^-16 of it is lost): one operand alone would be off by up to 2^-8, as much as the result's own rounding (error against 64
//    bits 0.0022 instead of 0.0017).  With up to eight rows in a tile the second operand lies in the places of the other eight rows and costs
//    nothing on the tensor core, otherwise the product is done twice; 64 sequences, 12 rows of 256: 84.3 us with one operand, 85.7 with two; 243 sequences, 4 rows of
//    128: 110.8, 112.2.  The sums take the weights unrounded in FP32.  The maximum follows only when a score passes it by 8 (weights up to 2^8), which spares
//    nearly every rescaling of the results.
//  * At an item's end the warps' results are added in shared memory in warp order.  Parts of a split item go to the handle's scratch and are added
//    in block order by a second kernel.
// Measured, call after call (1.86 to 1.92 GHz under the power cap): 64 sequences of 128 to 16384 tokens, 24 heads over 2 of 256, 86 us, 0.75 of the copy rate in
// cache bytes; 243 sequences, 32 heads over 8 of 128, 113 us, 0.76, and of 64 102 us; one sequence of 131,000 tokens 55 us, 0.74; one of 1501 16 us, a chain of
// latencies (lengths, pages, a few units, the sums, the join) and not bytes.
// Tokens past the length, and those of pages out of bounds, are zero-filled and masked, whatever memory holds there.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "nvfp4_internal.h"
#include "paged_plan.h"
#include "ptx.cuh"
#include "umma.cuh"

namespace nvfp4 {

bool make_cache_map(CUtensorMap* m, const paged::Batch& b, const void* base, int slots, int parts);

namespace {

using namespace paged;

constexpr int kGroup = 16;           // tokens of a unit and warp

// Heads of 256 are shared by two warps, half the elements each: both halves' results and queries in one warp's registers spill.  The pair
// adds its two halves of the scores in shared memory; all else runs as with heads of 128.
template <int D>
struct Form {
    static constexpr int kWarps = 8, kThreads = kWarps * 32;
    static constexpr int kHalves = D == 256 ? 2 : 1;
    static constexpr int kWidth = D / kHalves;                         // elements of a head that a warp works on
    static constexpr int kGroups = kWarps / kHalves;                   // warps, or pairs of them, with tokens of their own
    static constexpr int kChunk = kGroups * kGroup;                    // tokens of a unit
    static constexpr int kHalfStage = kGroup * kWidth * 2, kStageBytes = 2 * kHalfStage;      // a warp's keys and values of one unit
    static constexpr int kStages = 192 * 1024 / (kWarps * kStageBytes);
    static constexpr int kTiles = kWidth / 8;                          // 8-column tiles of a warp's result
    static constexpr int kRounds = D == 64 ? 1 : 2;                    // rounds in which the warps' results are added
    static constexpr int kRoundTiles = kTiles / kRounds;
    static constexpr int kAllTiles = D / 8, kWarpTiles = kAllTiles / kWarps;                  // tiles of the sum that a warp writes
    static constexpr int kMergeBytes = kWarps * kRoundTiles * 512;
    static constexpr int kAhead = 16;                                  // sequences from the run's first one on that are looked up at once
    static constexpr int kSmem = kWarps * kStages * kStageBytes + kMergeBytes + kWarps * kRows * 8 + kWarps * kStages * 12 + 64 + kAhead * 16 + 1024;
};
static_assert(Form<256>::kSmem <= 232448 && Form<128>::kSmem <= 232448 && Form<64>::kSmem <= 232448, "shared memory");
static_assert(Form<256>::kStages == 3 && Form<128>::kStages == 3 && Form<64>::kStages == 6, "ring");
static_assert(Form<256>::kMergeBytes >= 2 * Form<256>::kWarps * 1024, "the pairs' scores lie where the results are added");

// Scratch of the handle: for each block the split item that begins in it, then two part slots per block: results [D / 8 tiles][32 lanes] of the
// registers' four values, maxima and sums of the 16 rows.
struct SplitItem {
    int count;               // blocks that share it; 0: none begins here
    int q0, rows, head, tile;
    int pad[3];
};
constexpr size_t kSplitBytes = kMaxBlocks * sizeof(SplitItem);
constexpr int kPartFloats = kRows * 256 + 2 * kRows;

struct DecodeParams {
    AttentionArgs a;
    float scale_log2;
    int min_cost;            // places of cost that a block takes at least
    int most_rows;           // sequences with more rows (new tokens x group) belong to another kernel
    int piece;               // tokens of one box of the tensor maps: 16, or 8 where pages are multiples of 8 only; 0: cp.async
    SplitItem* split;
    float* parts;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 y = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&y);
}

// Row r of an item's (token, head in the group) rows, as one lane of four sees it: two columns of every tile of eight.
struct Row {
    long long gate_at, out_at;
    bool there;
    __device__ __forceinline__ Row(const AttentionArgs& a, int q0, int rows, int head, int r) {
        there = r < rows;
        const int t = there ? (a.group == 1 ? r : r / a.group) : 0, h = head * a.group + (there ? r - t * a.group : 0), c = (threadIdx.x & 3) * 2;
        gate_at = (long long)(q0 + t) * a.g_stride + (long long)h * a.g_head + c;
        out_at = (long long)(q0 + t) * a.o_stride + (long long)h * a.o_head + c;
    }
    __device__ __forceinline__ uint32_t gate(const AttentionArgs& a, int tile) const {
        return a.gate && there ? *reinterpret_cast<const uint32_t*>(a.gate + gate_at + tile * 8) : 0u;
    }
    // gated, rounded once
    __device__ __forceinline__ void write(const AttentionArgs& a, int tile, uint32_t gate, float x, float y) const {
        if (a.gate) {
            x /= 1.0f + __expf(-__uint_as_float(gate << 16));
            y /= 1.0f + __expf(-__uint_as_float(gate & 0xFFFF0000u));
        }
        if (there) *reinterpret_cast<uint32_t*>(a.out + out_at + tile * 8) = pack_bf16(x, y);
    }
};

// A walk over the units of a run of places.
template <int D>
struct Cursor {
    Sequence q;
    Items n;
    long long at;                    // the item's place
    int s, item, chunk, to;          // units [chunk, to) of it are left
    int head, tile, limit;           // limit: tokens that some row of its tile sees
    static __device__ __forceinline__ Items items(const DecodeParams& p, const Sequence& q) {
        return items_of(p.a.b, q, p.a.group, Form<D>::kChunk, p.most_rows);
    }
    __device__ __forceinline__ void set_item(const DecodeParams& p, long long c0, long long c1) {
        head = n.tiles == 1 ? item : item / n.tiles;
        tile = item - head * n.tiles;
        limit = q.q_len == 1 ? sees(q, 0) : sees(q, (min((tile + 1) * kRows, q.q_len * p.a.group) - 1) / p.a.group);
        const Units u = units_in(at, n, c0, c1);
        chunk = u.from;
        to = u.to;
    }
    // To the next item that has units in the run [c0, c1); false behind the last one.
    __device__ __forceinline__ bool next_item(const DecodeParams& p, long long c0, long long c1, const Sequence* ahead, int base) {
        at += n.cost();
        if (at + n.extra >= c1) return false;
        if (++item == n.items) {
            item = 0;
            do {
                ++s;
                q = s - base < Form<D>::kAhead ? ahead[s - base] : sequence(p.a.b, s);
                n = items(p, q);
            } while (n.items == 0 && s + 1 < p.a.b.sequences);
        }
        set_item(p, c0, c1);
        return true;
    }
};

template <int D, bool TMA>
__global__ void __launch_bounds__(Form<D>::kThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const __grid_constant__ DecodeParams p) {
    using F = Form<D>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);     // the swizzle's pattern repeats every 1024 bytes
    const AttentionArgs& a = p.a;
    const Batch& b = a.b;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = warp / F::kHalves, col0 = warp % F::kHalves * F::kWidth;        // whose tokens and elements are this warp's
    unsigned char* ring = smem + warp * F::kStages * F::kStageBytes;
    float4* merge = reinterpret_cast<float4*>(smem + F::kWarps * F::kStages * F::kStageBytes);
    float* s_max = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(merge) + F::kMergeBytes);   // [warp][row]
    float* s_sum = s_max + F::kWarps * kRows;
    unsigned int* s_ok = reinterpret_cast<unsigned int*>(s_sum + F::kWarps * kRows);                     // [warp][stage]: tokens whose page is one
    uint64_t* full = reinterpret_cast<uint64_t*>(s_ok + F::kWarps * F::kStages) + warp * F::kStages;
    int* s_abort = reinterpret_cast<int*>(s_ok + 3 * F::kWarps * F::kStages);
    Sequence* ahead = reinterpret_cast<Sequence*>(s_abort + 16);
    if (tid == 0) *s_abort = 0;
    if (TMA && lane == 0) {
        for (int i = 0; i < F::kStages; ++i) ptx::mbar_init(&full[i], 1);
        ptx::fence_mbar_init();
        if (warp == 0) {
            ptx::prefetch_tensormap(&tmk);
            ptx::prefetch_tensormap(&tmv);
        }
    }

    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // ---- this block's run: prefix sums over the sequences, several of them per thread where there are many
    long long* prefix = reinterpret_cast<long long*>(merge);
    Cursor<D>* found = reinterpret_cast<Cursor<D>*>(prefix + F::kWarps);
    const int run = (b.sequences + F::kThreads - 1) / F::kThreads;
    const int s0 = min(tid * run, b.sequences), s1 = min(s0 + run, b.sequences);
    long long mine = 0;
    Cursor<D> at;
    for (int s = s0; s < s1; ++s) {
        at.s = s;
        at.q = sequence(b, s);
        at.n = Cursor<D>::items(p, at.q);
        mine += (long long)at.n.items * at.n.cost();
        // one block says so, the one that is the last to have work of its own
        if (blockIdx.x + 1 == gridDim.x && cut_off(b, s)) *b.places = kStatusPlace;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) prefix[warp] = upto;
    __syncthreads();
    long long cost = 0, before = 0;
#pragma unroll
    for (int w = 0; w < F::kWarps; ++w) {
        if (w < warp) before += prefix[w];
        cost += prefix[w];
    }
    upto += before;
    const int blocks = cost == 0 ? 0 : blocks_of(cost, gridDim.x, p.min_cost);
    if (tid == 0) p.split[blockIdx.x].count = 0;
    if ((int)blockIdx.x >= blocks) return;
    const long long c0 = run_begin(cost, blocks, blockIdx.x), c1 = run_begin(cost, blocks, blockIdx.x + 1);
    if (upto - mine <= c0 && c0 < upto) {            // exactly one thread
        long long left = c0 - (upto - mine);
        for (int s = s0; run > 1; ++s) {             // with one sequence a thread it is at hand
            at.s = s;
            at.q = sequence(b, s);
            at.n = Cursor<D>::items(p, at.q);
            const long long here = (long long)at.n.items * at.n.cost();
            if (left < here) break;
            left -= here;
        }
        at.item = (int)(left / at.n.cost());
        at.at = c0 - (left - (long long)at.item * at.n.cost());
        at.set_item(p, c0, c1);
        *found = at;
    }
    __syncthreads();
    at = *found;
    const int base = at.s;
    if (tid < F::kAhead && base + tid < b.sequences) ahead[tid] = sequence(b, base + tid);
    __syncthreads();                                 // and the scores of pairs go where the cursor was
    bool more = true;
    Cursor<D> ld = at;                               // where the loads are
    bool ld_more = more;

    // ---- loads: the page number of this lane's token (cp.async: lanes 0..15) or piece is asked for one unit ahead
    int page_ahead = -1, slot_ahead = 0;
    bool seen_ahead = false;
    const int step = TMA ? p.piece : 1;                          // tokens that a lane looks up
    auto look_up = [&]() {
        const int tok = ld.chunk * F::kChunk + group * kGroup + (TMA ? lane * step : lane & 15);
        seen_ahead = ld_more && tok < ld.limit && (!TMA || lane * step < kGroup);
        page_ahead = -1;
        if (seen_ahead) {
            const int entry = divide(tok, b.div);
            slot_ahead = tok - entry * b.page_size;
            page_ahead = b.table[(long long)ld.s * b.table_stride + entry];
        }
    };
    auto load = [&](int stage) {
        if (ld_more) {
            const bool there = seen_ahead && (unsigned)page_ahead < (unsigned)b.num_pages;
            if (seen_ahead && !there) *b.places = kStatusPlace;
            unsigned int ok = __ballot_sync(0xffffffffu, there);
            unsigned char* ks = ring + stage * F::kStageBytes;
            unsigned char* vs = ks + F::kHalfStage;
            const int tok0 = ld.chunk * F::kChunk + group * kGroup;
            if (TMA) {
                const unsigned int pieces = ok;
                ok = step == kGroup ? (pieces & 1u) * 0xFFFFu : (pieces & 1u) * 0xFFu | (pieces >> 1 & 1u) * 0xFF00u;
                if (ld.limit - tok0 < kGroup) ok &= ld.limit > tok0 ? (1u << (ld.limit - tok0)) - 1u : 0u;
                if (lane == 0) {
                    s_ok[warp * F::kStages + stage] = ok;
                    ptx::mbar_arrive_expect_tx(&full[stage], (unsigned)__popc(pieces) * (unsigned)step * F::kWidth * 4u);
                }
                __syncwarp();
                if (step == kGroup) {
                    if (there) {                             // lane 0
                        ptx::tma_load_5d(ks, &tmk, &full[stage], 0, slot_ahead, col0 / 64, ld.head, page_ahead);
                        ptx::tma_load_5d(vs, &tmv, &full[stage], 0, slot_ahead, col0 / 64, ld.head, page_ahead);
                    }
                } else {
                    // lane = (piece, keys or values, 64 of the head's elements)
                    const int from = lane / (F::kWidth / 32);        // 2 * (kWidth / 64) boxes of a piece
                    const int pg = __shfl_sync(0xffffffffu, page_ahead, from & 1), sl = __shfl_sync(0xffffffffu, slot_ahead, from & 1);
                    const int part = lane % (F::kWidth / 64), which = lane / (F::kWidth / 64) % 2;
                    if (from < 2 && (pieces >> from & 1u))
                        ptx::tma_load_5d((which ? vs : ks) + part * (kGroup * 128) + from * 1024, which ? &tmv : &tmk, &full[stage], 0, sl, col0 / 64 + part, ld.head, pg);
                }
            } else {
                ok &= 0xFFFFu;
                if (lane == 0) s_ok[warp * F::kStages + stage] = ok;
                const long long off = there ? (long long)page_ahead * b.page_stride + (long long)slot_ahead * b.token_stride + (long long)ld.head * b.head_stride + col0 : 0;
                if (tok0 < ld.limit) {                       // no page at all: zeros too, the values are multiplied
                    constexpr int kPer = F::kWidth / 8;      // 16-byte pieces of a token
#pragma unroll
                    for (int i = 0; i < kGroup * kPer / 32; ++i) {
                        const int tok = (i * 32 + lane) / kPer, piece = (i * 32 + lane) % kPer;
                        const long long o = __shfl_sync(0xffffffffu, off, tok);
                        const uint32_t bytes = (ok >> tok) & 1u ? 16u : 0u;
                        const int to = (piece >> 3) * (kGroup * 128) + tok * 128 + (((piece & 7) ^ (tok & 7)) << 4);
                        ptx::cp_async_16(ks + to, b.k + o + piece * 8, bytes);
                        ptx::cp_async_16(vs + to, b.v + o + piece * 8, bytes);
                    }
                }
            }
            if (++ld.chunk == ld.to) ld_more = ld.next_item(p, c0, c1, ahead, base);
            look_up();
        }
        if (!TMA) cp_async_commit();
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < F::kStages - 1; ++i) load(i);

    // ---- units
    uint32_t qf[F::kWidth / 16][4];
    float o[F::kTiles][4];
    float m0 = 0, m1 = 0, l0 = 0, l1 = 0;            // of rows lane / 4 and lane / 4 + 8
    int see0 = 0, see1 = 0;
    int stage = 0, next = F::kStages - 1;
    uint32_t parity = 0;
    unsigned int unit = 0;                           // units multiplied so far
    const int row = lane >> 2;
    // what a new item begins with: its rows of q, and which keys they see
    auto begin_item = [&]() {
        const int r0 = at.tile * kRows + row, rows = at.q.q_len * a.group, head = at.head;
        const uint16_t *x0 = nullptr, *x1 = nullptr;
        see0 = see1 = 0x7fffffff;                    // rows that are none see all there is, of a query of zeros
        if (r0 < rows) {
            const int t = a.group == 1 ? r0 : r0 / a.group;
            x0 = a.q + (long long)(at.q.q0 + t) * a.q_stride + (long long)(head * a.group + r0 - t * a.group) * a.q_head;
            see0 = sees(at.q, t);
        }
        if (r0 + 8 < rows) {
            const int t = a.group == 1 ? r0 + 8 : (r0 + 8) / a.group;
            x1 = a.q + (long long)(at.q.q0 + t) * a.q_stride + (long long)(head * a.group + r0 + 8 - t * a.group) * a.q_head;
            see1 = sees(at.q, t);
        }
#pragma unroll
        for (int k = 0; k < F::kWidth / 16; ++k) {
            const int c = col0 + k * 16 + (lane & 3) * 2;
            qf[k][0] = x0 ? *reinterpret_cast<const uint32_t*>(x0 + c) : 0u;
            qf[k][1] = x1 ? *reinterpret_cast<const uint32_t*>(x1 + c) : 0u;
            qf[k][2] = x0 ? *reinterpret_cast<const uint32_t*>(x0 + c + 8) : 0u;
            qf[k][3] = x1 ? *reinterpret_cast<const uint32_t*>(x1 + c + 8) : 0u;
        }
    };
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.0f;
    };
    begin_item();
    clear();
    int from = at.chunk;                             // the first unit of the item that is this block's
    bool low = at.q.q_len * a.group - at.tile * kRows <= 8;      // the tile's rows are the first eight at most
    while (more) {
        if (TMA) {
            // run out: nothing more is asked for; the warp goes on through its units, whose results are worth nothing, so that no other waits for it
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[stage], parity, s_abort, b.status, 0xA10u))) ld_more = false;
        } else {
            cp_async_wait<F::kStages - 2>();
        }
        __syncwarp();
        load(next);
        next = next + 1 == F::kStages ? 0 : next + 1;
        const int tok0 = at.chunk * F::kChunk + group * kGroup;
        if (tok0 < at.limit) {
            const uint32_t ks = ptx::smem_u32(ring + stage * F::kStageBytes), vs = ks + F::kHalfStage;
            const unsigned int ok = s_ok[warp * F::kStages + stage];
            if (TMA && ok != 0xFFFFu) {
                // what lies behind the length or on no page: a weight of zero times anything finite only
                for (int i = lane; i < kGroup * F::kWidth / 8; i += 32) {
                    const int tok = (i >> 3) & (kGroup - 1);
                    if (!(ok >> tok & 1u))
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vs + (i >> 7) * (kGroup * 128) + tok * 128 + (i & 7) * 16), "r"(0u) : "memory");
                }
                ptx::fence_proxy_async_smem();       // in front of the next load into this stage
                __syncwarp();
            }
            float sc[2][2][4] = {};                  // [even / odd step][8 tokens][element]
            {
                const int tok = ((lane >> 4) << 3) + (lane & 7);
                uint32_t off[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) off[i] = ks + tok * 128 + (((i * 2 + ((lane >> 3) & 1)) ^ (tok & 7)) << 4);
#pragma unroll
                for (int k = 0; k < F::kWidth / 16; ++k) {
                    uint32_t r[4];
                    ldmatrix_x4(r, off[k & 3] + (k >> 2) * (kGroup * 128));
                    ptx::mma_bf16_16x8x16(sc[k & 1][0], qf[k], r[0], r[1]);
                    ptx::mma_bf16_16x8x16(sc[k & 1][1], qf[k], r[2], r[3]);
                }
            }
            float t[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[n][e] = sc[0][n][e] + sc[1][n][e];
            if (F::kHalves == 2) {                   // both warps go through the same units, so they meet here; two buffers in turn
                float4* mine = merge + (warp * 2 + (unit & 1)) * 64 + lane;
                mine[0] = make_float4(t[0][0], t[0][1], t[0][2], t[0][3]);
                mine[32] = make_float4(t[1][0], t[1][1], t[1][2], t[1][3]);
                ptx::named_barrier_sync(1 + group, 64);
                const float4* other = merge + ((warp ^ 1) * 2 + (unit & 1)) * 64 + lane;
                const float4 x = other[0], y = other[32];
                t[0][0] += x.x; t[0][1] += x.y; t[0][2] += x.z; t[0][3] += x.w;
                t[1][0] += y.x; t[1][1] += y.y; t[1][2] += y.z; t[1][3] += y.w;
                ++unit;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[n][e] *= p.scale_log2;
            if (__any_sync(0xffffffffu, tok0 + kGroup > min(see0, see1)) || ok != 0xFFFFu) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = n * 8 + (lane & 3) * 2 + (e & 1);
                        if (tok0 + j >= (e < 2 ? see0 : see1) || !((ok >> j) & 1u)) t[n][e] = -INFINITY;
                    }
            }
            float g0 = fmaxf(fmaxf(t[0][0], t[0][1]), fmaxf(t[1][0], t[1][1]));
            float g1 = fmaxf(fmaxf(t[0][2], t[0][3]), fmaxf(t[1][2], t[1][3]));
            g0 = fmaxf(g0, __shfl_xor_sync(0xffffffffu, g0, 1));
            g1 = fmaxf(g1, __shfl_xor_sync(0xffffffffu, g1, 1));
            g0 = fmaxf(g0, __shfl_xor_sync(0xffffffffu, g0, 2));
            g1 = fmaxf(g1, __shfl_xor_sync(0xffffffffu, g1, 2));
            if (__any_sync(0xffffffffu, g0 > m0 + 8.0f || g1 > m1 + 8.0f)) {
                const float n0 = fmaxf(m0, g0), n1 = fmaxf(m1, g1);
                const float c0 = n0 == m0 ? 1.0f : ex2(m0 - n0), c1 = low ? c0 : n1 == m1 ? 1.0f : ex2(m1 - n1);
                m0 = n0;
                m1 = n1;
                l0 *= c0;
                l1 *= c1;
#pragma unroll
                for (int i = 0; i < F::kTiles; ++i) {
                    o[i][0] *= c0;
                    o[i][1] *= c0;
                    o[i][2] *= c1;
                    o[i][3] *= c1;
                }
            }
            const float b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
            const int tok = lane & 15;
            uint32_t off[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) off[i] = vs + tok * 128 + (((i * 2 + (lane >> 4)) ^ (tok & 7)) << 4);
            // The weights are two BF16 operands, the rounded ones and what their rounding left, which lies in the places of rows 8 to 15 where the
            // tile has none.
            auto multiply = [&](auto halves) {
                constexpr int kRowHalves = decltype(halves)::value;          // 1: rows 0 to 7 only
                uint32_t w[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int h = 0; h < kRowHalves; ++h) {
                        const float x = ex2(t[n][2 * h] - (h ? b1 : b0)), y = ex2(t[n][2 * h + 1] - (h ? b1 : b0));
                        (h ? l1 : l0) += x + y;
                        const uint32_t rounded = pack_bf16(x, y);
                        w[0][2 * n + h] = rounded;
                        w[kRowHalves - 1][2 * n + h + 2 - kRowHalves] = pack_bf16(x - __uint_as_float(rounded << 16), y - __uint_as_float(rounded & 0xFFFF0000u));
                    }
#pragma unroll
                for (int c = 0; c < F::kTiles; c += 2) {
                    uint32_t r[4];
                    ldmatrix_x4_trans(r, off[c / 2 & 3] + (c >> 3) * (kGroup * 128));
#pragma unroll
                    for (int i = 0; i < kRowHalves; ++i) {
                        ptx::mma_bf16_16x8x16(o[c], w[i], r[0], r[1]);
                        ptx::mma_bf16_16x8x16(o[c + 1], w[i], r[2], r[3]);
                    }
                }
            };
            if (low) multiply(std::integral_constant<int, 1>{});
            else multiply(std::integral_constant<int, 2>{});
        }
        if (++stage == F::kStages) {
            stage = 0;
            parity ^= 1u;
        }
        if (++at.chunk < at.to) continue;

        // ---- the item (or this block's part of it) is through
        const bool whole = from == 0 && at.to == at.n.chunks;
        const int rows = at.q.q_len * a.group, low_rows = rows - at.tile * kRows;
        const Row row0(a, at.q.q0, rows, at.head, at.tile * kRows + row), row1(a, at.q.q0, rows, at.head, at.tile * kRows + row + 8);
        const int first = block_of(cost, blocks, at.at + at.n.extra);
        const int count = whole ? 1 : block_of(cost, blocks, at.at + at.n.extra + at.n.chunks - 1) - first + 1;
        float* part = p.parts + (size_t)part_slot(first, blockIdx.x) * kPartFloats;
        if (!whole && first == (int)blockIdx.x && tid == 0) p.split[blockIdx.x] = SplitItem{count, at.q.q0, rows, at.head, at.tile, {0, 0, 0}};
        // the i-th tile whose sum this warp writes: as the rounds go through them
        auto tile_of = [&](int i) {
            constexpr int kPer = F::kWarpTiles / F::kRounds;
            const int tile = i % kPer * F::kWarps + warp;
            return tile / F::kRoundTiles * F::kTiles + i / kPer * F::kRoundTiles + tile % F::kRoundTiles;
        };
        uint32_t gates[F::kWarpTiles][2];            // of this thread's values, asked for in front of the barriers
        if (whole) {
#pragma unroll
            for (int i = 0; i < F::kWarpTiles; ++i) {
                gates[i][0] = row0.gate(a, tile_of(i));
                gates[i][1] = row1.gate(a, tile_of(i));
            }
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

        // the next item's rows of q are on their way while this one's results are added
        more = at.next_item(p, c0, c1, ahead, base);
        from = at.chunk;
        if (more) begin_item();
        float f0[F::kGroups], f1[F::kGroups], top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.0f, sum1 = 0.0f;
        // LOW: the tile's rows are the first eight at most (a group of eight or less in decode): half the values, added in one round.
        auto add_warps = [&](auto low) {
            constexpr bool kLow = decltype(low)::value;
            constexpr int kRounds = kLow ? 1 : F::kRounds, kRoundTiles = F::kTiles / kRounds, kPer = F::kWarpTiles / kRounds;
            float2* merge2 = reinterpret_cast<float2*>(merge);
#pragma unroll
            for (int rd = 0; rd < kRounds; ++rd) {
                __syncthreads();                     // the round before is out of the shared arrays
#pragma unroll
                for (int i = 0; i < kRoundTiles; ++i) {
                    const float(&x)[4] = o[rd * kRoundTiles + i];
                    if (kLow) merge2[(warp * kRoundTiles + i) * 32 + lane] = make_float2(x[0] + x[2], x[1] + x[3]);
                    else merge[(warp * kRoundTiles + i) * 32 + lane] = make_float4(x[0], x[1], x[2], x[3]);
                }
                if (rd == 0 && col0 == 0 && (lane & 3) == 0) {
                    s_max[group * kRows + row] = m0;
                    s_max[group * kRows + row + 8] = m1;
                    s_sum[group * kRows + row] = l0;
                    s_sum[group * kRows + row + 8] = l1;
                }
                __syncthreads();
                if (rd == 0) {
#pragma unroll
                    for (int w = 0; w < F::kGroups; ++w) {
                        f0[w] = s_max[w * kRows + row];
                        f1[w] = s_max[w * kRows + row + 8];
                        top0 = fmaxf(top0, f0[w]);
                        top1 = fmaxf(top1, f1[w]);
                    }
#pragma unroll
                    for (int w = 0; w < F::kGroups; ++w) {
                        f0[w] = f0[w] == -INFINITY ? 0.0f : ex2(f0[w] - top0);
                        f1[w] = f1[w] == -INFINITY ? 0.0f : ex2(f1[w] - top1);
                        sum0 += s_sum[w * kRows + row] * f0[w];
                        sum1 += s_sum[w * kRows + row + 8] * f1[w];
                    }
                    if (whole) {
                        const float inv0 = sum0 == 0.0f ? 0.0f : 1.0f / sum0, inv1 = sum1 == 0.0f ? 0.0f : 1.0f / sum1;
#pragma unroll
                        for (int w = 0; w < F::kGroups; ++w) {
                            f0[w] *= inv0;
                            f1[w] *= inv1;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const int mine = rd * kPer + i, nt = tile_of(mine), half = nt / F::kTiles, in_half = nt % F::kTiles - rd * kRoundTiles;
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < F::kGroups; ++w) {
                        const int from = ((w * F::kHalves + half) * kRoundTiles + in_half) * 32 + lane;
                        float4 y;
                        if (kLow) {
                            const float2 z = merge2[from];
                            y = make_float4(z.x, z.y, 0.0f, 0.0f);
                        } else {
                            y = merge[from];
                        }
                        x.x = fmaf(y.x, f0[w], x.x);
                        x.y = fmaf(y.y, f0[w], x.y);
                        x.z = fmaf(y.z, f1[w], x.z);
                        x.w = fmaf(y.w, f1[w], x.w);
                    }
                    if (whole) {
                        row0.write(a, nt, gates[mine][0], x.x, x.y);
                        if (!kLow) row1.write(a, nt, gates[mine][1], x.z, x.w);
                    } else {
                        __stcg(reinterpret_cast<float4*>(part) + nt * 32 + lane, x);
                    }
                }
            }
        };
        if (low_rows <= 8) add_warps(std::true_type{});
        else add_warps(std::false_type{});
        if (!whole && warp == 0) {
            if ((lane & 3) == 0) {
                float* ml = part + kRows * D;
                __stcg(ml + row, top0);
                __stcg(ml + row + 8, top1);
                __stcg(ml + kRows + row, sum0);
                __stcg(ml + kRows + row + 8, sum1);
            }
        }
        if (F::kHalves == 2) __syncthreads();        // the next item's scores go where the results were added
        clear();
        low = at.q.q_len * a.group - at.tile * kRows <= 8;
    }
    if (!TMA) cp_async_wait<0>();
    if (TMA && *reinterpret_cast<volatile int*>(s_abort)) {            // loads may still be on their way into this block's shared memory
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
}

// Adds the parts of split items in the order of their blocks.  A kernel of its own behind the other one: there the last block to arrive would
// read up to a hundred parts of 16 KB through one SM (17 us for a single long sequence, in two levels).  Here an item's 8-column tiles are spread over
// blocks.  Few parts: a warp for each tile, all its parts under way at once.  Many: a block for one or two tiles, its warps share the parts.  (Heads of 256 spill 24
// bytes at the 128 registers that two blocks an SM leave.)
constexpr int kJoinWarps = 8, kJoinAhead = 10;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32, 2)
paged_join_kernel(const __grid_constant__ DecodeParams p, int blocks) {
    constexpr int kTiles = D == 256 ? 2 : 1, kSlices = D / 8 / kTiles, kFewSlices = D / 8 / kJoinWarps;
    __shared__ SplitItem s_item[kMaxBlocks];
    __shared__ int s_first[kMaxBlocks], s_count[2][kMaxBlocks / 32];
    __shared__ unsigned short s_work[kMaxBlocks * kSlices];             // item, slice: item * kSlices + slice
    __shared__ float4 s_sum[kJoinWarps][kTiles][32];
    __shared__ float s_top[kJoinWarps][kRows], s_den[kJoinWarps][kRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = lane >> 2;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    static_assert(kMaxBlocks == kJoinWarps * 32, "a thread looks at a block");
    static_assert(kMaxBlocks * kSlices <= 65536, "16-bit work numbers");
    SplitItem mine{};
    if (tid < blocks) {
        const int4 x = __ldcg(reinterpret_cast<const int4*>(p.split + tid));
        mine.count = x.x; mine.q0 = x.y; mine.rows = x.z; mine.head = x.w;
        mine.tile = __ldcg(&p.split[tid].tile);
    }
    // items and pieces of work in front of this thread's
    const int slices = mine.count == 0 ? 0 : mine.count <= kJoinAhead ? kFewSlices : kSlices;
    int upto = slices;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    const unsigned int vote = __ballot_sync(0xffffffffu, mine.count > 0);
    if (lane == 31) {
        s_count[0][warp] = __popc(vote);
        s_count[1][warp] = upto;
    }
    __syncthreads();
    int works = 0, item0 = __popc(vote & ((1u << lane) - 1u)), work0 = upto - slices;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        if (w < warp) {
            item0 += s_count[0][w];
            work0 += s_count[1][w];
        }
        works += s_count[1][w];
    }
    if (mine.count > 0) {
        s_item[item0] = mine;
        s_first[item0] = tid;
        for (int i = 0; i < slices; ++i) s_work[work0 + i] = (unsigned short)(item0 * kSlices + i);
    }
    __syncthreads();
    for (int work = blockIdx.x; work < works; work += gridDim.x) {
        const int number = s_work[work], slice = number % kSlices;
        const SplitItem it = s_item[number / kSlices];
        const int first = s_first[number / kSlices];
        const Row row0(p.a, it.q0, it.rows, it.head, it.tile * kRows + row), row1(p.a, it.q0, it.rows, it.head, it.tile * kRows + row + 8);
        if (it.count <= kJoinAhead) {
            const int tile = slice * kJoinWarps + warp;
            const uint32_t gate0 = row0.gate(p.a, tile), gate1 = row1.gate(p.a, tile);
            float4 y[kJoinAhead];
            float m[kJoinAhead / 2], l[kJoinAhead / 2], top = -INFINITY, den = 0.0f;      // part 2j + lane / 16, row lane % 16, in place j
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j)
                y[j] = ptx::ldcg_if(j < it.count, reinterpret_cast<const float4*>(p.parts + (size_t)part_slot(first, first + j) * kPartFloats) + tile * 32 + lane);
#pragma unroll
            for (int j = 0; j < kJoinAhead / 2; ++j) {
                const int i = 2 * j + (lane >> 4);
                const float* ml = p.parts + (size_t)part_slot(first, first + i) * kPartFloats + kRows * D + (lane & 15);
                m[j] = ptx::ldcg_if(i < it.count, ml, -INFINITY);
                l[j] = ptx::ldcg_if(i < it.count, ml + kRows, 0.0f);
                top = fmaxf(top, m[j]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
#pragma unroll
            for (int j = 0; j < kJoinAhead / 2; ++j) {
                m[j] = m[j] == -INFINITY ? 0.0f : ex2(m[j] - top);
                den += m[j] * l[j];
            }
            den += __shfl_xor_sync(0xffffffffu, den, 16);
            const float norm = den == 0.0f ? 0.0f : 1.0f / den;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                const float w0 = __shfl_sync(0xffffffffu, m[j / 2], j % 2 * 16 + row), w1 = __shfl_sync(0xffffffffu, m[j / 2], j % 2 * 16 + row + 8);
                if (j >= it.count) continue;
                x.x = fmaf(y[j].x, w0, x.x);
                x.y = fmaf(y[j].y, w0, x.y);
                x.z = fmaf(y[j].z, w1, x.z);
                x.w = fmaf(y[j].w, w1, x.w);
            }
            const float n0 = __shfl_sync(0xffffffffu, norm, row), n1 = __shfl_sync(0xffffffffu, norm, row + 8);
            row0.write(p.a, tile, gate0, x.x * n0, x.y * n0);
            row1.write(p.a, tile, gate1, x.z * n1, x.w * n1);
            continue;
        }
        const int tile0 = slice * kTiles;
        uint32_t gates[2] = {0u, 0u};
        if (warp < kTiles) {
            gates[0] = row0.gate(p.a, tile0 + warp);
            gates[1] = row1.gate(p.a, tile0 + warp);
        }
        // parts warp, warp + 8, ...; maxima and sums: part 2j + lane / 16 of these, row lane % 16, in place j
        float top = -INFINITY, den = 0.0f;           // of row lane % 16 over this half's parts, then over all of the warp's
        float4 x[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) x[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = warp; i0 < it.count; i0 += kJoinWarps * kJoinAhead) {
            float4 y[kJoinAhead][kTiles];
            float m[kJoinAhead / 2], l[kJoinAhead / 2];
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                const int i = i0 + j * kJoinWarps;
                const float4* from = reinterpret_cast<const float4*>(p.parts + (size_t)part_slot(first, first + i) * kPartFloats) + tile0 * 32 + lane;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) y[j][t] = ptx::ldcg_if(i < it.count, from + t * 32);
            }
#pragma unroll
            for (int j = 0; j < kJoinAhead / 2; ++j) {
                const int i = i0 + (2 * j + (lane >> 4)) * kJoinWarps;
                const float* ml = p.parts + (size_t)part_slot(first, first + i) * kPartFloats + kRows * D + (lane & 15);
                m[j] = ptx::ldcg_if(i < it.count, ml, -INFINITY);
                l[j] = ptx::ldcg_if(i < it.count, ml + kRows, 0.0f);
            }
            float now = top;
#pragma unroll
            for (int j = 0; j < kJoinAhead / 2; ++j) now = fmaxf(now, m[j]);
            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 16));
            const float back = top == -INFINITY ? 0.0f : ex2(top - now);
            top = now;
            den *= back;
#pragma unroll
            for (int j = 0; j < kJoinAhead / 2; ++j) {
                m[j] = m[j] == -INFINITY ? 0.0f : ex2(m[j] - now);
                den += m[j] * l[j];
            }
            const float b0 = __shfl_sync(0xffffffffu, back, row), b1 = __shfl_sync(0xffffffffu, back, row + 8);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) x[t] = make_float4(x[t].x * b0, x[t].y * b0, x[t].z * b1, x[t].w * b1);
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                const float w0 = __shfl_sync(0xffffffffu, m[j / 2], j % 2 * 16 + row), w1 = __shfl_sync(0xffffffffu, m[j / 2], j % 2 * 16 + row + 8);
                if (i0 + j * kJoinWarps >= it.count) continue;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    x[t].x = fmaf(y[j][t].x, w0, x[t].x);
                    x[t].y = fmaf(y[j][t].y, w0, x[t].y);
                    x[t].z = fmaf(y[j][t].z, w1, x[t].z);
                    x[t].w = fmaf(y[j][t].w, w1, x[t].w);
                }
            }
        }
        den += __shfl_xor_sync(0xffffffffu, den, 16);
        __syncthreads();                             // the work before is out of the shared arrays
#pragma unroll
        for (int t = 0; t < kTiles; ++t) s_sum[warp][t][lane] = x[t];
        if (lane < kRows) {
            s_top[warp][lane] = top;
            s_den[warp][lane] = den;
        }
        __syncthreads();
        if (warp < kTiles) {
            float t0 = -INFINITY, t1 = -INFINITY, d0 = 0.0f, d1 = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) {
                t0 = fmaxf(t0, s_top[w][row]);
                t1 = fmaxf(t1, s_top[w][row + 8]);
            }
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) {
                const float a0 = s_top[w][row], a1 = s_top[w][row + 8];
                const float w0 = a0 == -INFINITY ? 0.0f : ex2(a0 - t0), w1 = a1 == -INFINITY ? 0.0f : ex2(a1 - t1);
                const float4 v = s_sum[w][warp][lane];
                d0 += w0 * s_den[w][row];
                d1 += w1 * s_den[w][row + 8];
                sum.x = fmaf(v.x, w0, sum.x);
                sum.y = fmaf(v.y, w0, sum.y);
                sum.z = fmaf(v.z, w1, sum.z);
                sum.w = fmaf(v.w, w1, sum.w);
            }
            const float n0 = d0 == 0.0f ? 0.0f : 1.0f / d0, n1 = d1 == 0.0f ? 0.0f : 1.0f / d1;
            row0.write(p.a, tile0 + warp, gates[0], sum.x * n0, sum.y * n0);
            row1.write(p.a, tile0 + warp, gates[1], sum.z * n1, sum.w * n1);
        }
    }
}

template <class... P, class... A>
cudaError_t launch_behind(void (*kernel)(P...), int grid, int threads, int smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D>
cudaError_t launch(const DecodeParams& p, const nvfp4_device_info& dev, cudaStream_t s) {
    const int blocks = dev.sm_count < kMaxBlocks ? dev.sm_count : kMaxBlocks, parts = p.piece == kGroup ? Form<D>::kWidth / 64 : 1;
    CUtensorMap tmk{}, tmv{};
    cudaError_t e;
    if (p.piece && make_cache_map(&tmk, p.a.b, p.a.b.k, p.piece, parts) && make_cache_map(&tmv, p.a.b, p.a.b.v, p.piece, parts))
        e = launch_behind(paged_decode_kernel<D, true>, blocks, Form<D>::kThreads, Form<D>::kSmem, s, tmk, tmv, p);
    else
        e = launch_behind(paged_decode_kernel<D, false>, blocks, Form<D>::kThreads, Form<D>::kSmem, s, tmk, tmv, p);
    if (e != cudaSuccess) return e;
    return launch_behind(paged_join_kernel<D>, 2 * blocks, kJoinWarps * 32, 0, s, p, blocks);
}

}  // namespace

// k or v as [page][head][64-element part][slot][64]: a box of `slots` slots and `parts` parts of one head of one page, rows of 128 bytes swizzled.
// False where the map cannot describe the cache.
bool make_cache_map(CUtensorMap* m, const paged::Batch& b, const void* base, int slots, int parts) {
    umma::EncodeFn enc = umma::get_encode();
    if (!enc) return false;
    const long long token = b.page_size > 1 ? b.token_stride : 64, head = b.kv_heads > 1 ? b.head_stride : 64, page = b.num_pages > 1 ? b.page_stride : 64;
    const cuuint64_t dims[5] = {64, (cuuint64_t)b.page_size, (cuuint64_t)(b.head_dim / 64), (cuuint64_t)b.kv_heads, (cuuint64_t)b.num_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)token * 2, 128, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)slots, (cuuint32_t)parts, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
    for (const cuuint64_t x : strides)
        if (x >= 1ull << 40) return false;
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t paged_scratch_bytes(int sm_count) { return kSplitBytes + (size_t)(sm_count < kMaxBlocks ? sm_count : kMaxBlocks) * 2 * kPartFloats * sizeof(float); }

cudaError_t configure_paged_decode() {
    cudaError_t e = configure_large_smem(paged_decode_kernel<64, true>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<128, true>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<256, true>, Form<256>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<64, false>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<128, false>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<256, false>, Form<256>::kSmem);
    return e;
}

cudaError_t launch_paged_decode(const paged::AttentionArgs& a, int most_rows, const nvfp4_device_info& dev, void* scratch, int* launches, cudaStream_t s) {
    DecodeParams p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.min_cost = item_cost(a.b.head_dim) + 1;
    p.most_rows = most_rows;
    p.piece = a.b.page_size % 16 == 0 ? 16 : a.b.page_size % 8 == 0 ? 8 : 0;
    p.split = static_cast<SplitItem*>(scratch);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + kSplitBytes);
    *launches = 2;
    return a.b.head_dim == 64 ? launch<64>(p, dev, s) : a.b.head_dim == 128 ? launch<128>(p, dev, s) : launch<256>(p, dev, s);
}

}  // namespace nvfp4
