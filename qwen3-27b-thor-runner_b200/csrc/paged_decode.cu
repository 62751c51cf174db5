// Attention of few new tokens over the paged cache (decode, verification of drafted tokens): one pass over keys and values, split
// over the sequences' lengths and joined.
//
//   out_r = sum_j 2^(t_rj - m_r) v_j / sum_j 2^(t_rj - m_r),   t_rj = scale * log2(e) * q_r . k_j,   m_r a running maximum
//
// The bound is HBM: a key and its value are 4 * head_dim bytes and meet only the rows of one key-value head, group * new tokens of
// them, up to 16 of which share a tile of mma.sync m16n8k16 (two FLOPs a byte and row; the warp MMA reaches a hundred times that).  So
// everything serves the stream of keys and values:
//  * Work is cut into units of 16 tokens for each of the block's warps, over all sequences, heads and row tiles in order, and each
//    block (one per SM) takes the same number of consecutive units, counted on the device from the lengths as they are.  A block so
//    holds whole (sequence, head, row tile) items and at most two parts of split ones.
//  * A warp loads its own 16 tokens with cp.async into a ring of its own and multiplies them alone, with a running maximum and sum of
//    its own: no barrier between warps inside an item, two stages always under way (128 KB of loads in flight on an SM), and the loads
//    run on across the borders of items.
//  * Scores, maxima, sums and results stay in registers.  The weights 2^(t - m) are rounded to BF16 as the MMA's operand (2^-9 relative
//    to each, below the rounding of the result); the sums take them unrounded in FP32.  The maximum follows only when a score passes it by 8
//    (weights up to 2^8), which spares nearly every rescaling of the results.
//  * At an item's end the warps' results are added in shared memory in warp order.  Parts of a split item go to the handle's scratch; the block
//    that arrives last adds them in block order, so the order of arrival changes nothing.
// Tokens past the length, and those of pages out of bounds, are zero-filled and masked, whatever memory holds there.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

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
    static constexpr int kSmem = kWarps * kStages * kStageBytes + kMergeBytes + kWarps * kRows * 8 + kWarps * kStages * 12 + 64 + 1024;
};
static_assert(Form<256>::kSmem <= 232448 && Form<128>::kSmem <= 232448 && Form<64>::kSmem <= 232448, "shared memory");
static_assert(Form<256>::kStages == 3 && Form<128>::kStages == 3 && Form<64>::kStages == 6, "ring");
static_assert(Form<256>::kMergeBytes >= 2 * Form<256>::kWarps * 1024, "the pairs' scores lie where the results are added");

// Scratch of the handle: the counters, then two part slots per block: results [16 rows, D] in the layout of the registers,
// maxima and sums.
constexpr int kPartFloats = kRows * 256 + 2 * kRows;
constexpr size_t kCounterBytes = (kCounters * 4 + 255) / 256 * 256;

struct DecodeParams {
    AttentionArgs a;
    float scale_log2;
    int min_cost;            // places of cost that a block takes at least
    int most_rows;           // sequences with more rows (new tokens x group) belong to another kernel
    int piece;               // tokens of one box of the tensor maps: 16, or 8 where pages are multiples of 8 only; 0: cp.async
    unsigned int* counters;
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
    __device__ __forceinline__ bool next_item(const DecodeParams& p, long long c0, long long c1) {
        at += n.cost();
        if (at + kItemCost >= c1) return false;
        if (++item == n.items) {
            item = 0;
            do {
                q = sequence(p.a.b, ++s);
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
    int* s_word = reinterpret_cast<int*>(s_ok + F::kWarps * F::kStages + 2 * F::kWarps * F::kStages);
    if (tid == 0) s_word[15] = 0;
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
    if (cost == 0) return;
    const int blocks = blocks_of(cost, gridDim.x, p.min_cost);
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
    __syncthreads();                                 // the scores of pairs go to the same place
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
            if (seen_ahead && !there) atomicCAS(b.status, 0u, kStatusPlace);
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
                if (ok) {
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
            if (++ld.chunk == ld.to) ld_more = ld.next_item(p, c0, c1);
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
    bool fresh = true;
    int stage = 0, next = F::kStages - 1;
    uint32_t parity = 0;
    unsigned int unit = 0;                           // units multiplied so far
    const int row = lane >> 2;
    int from = at.chunk;                             // the first unit of the item that is this block's
    while (more) {
        if (fresh) {                                 // a new item: its rows of q
            fresh = false;
            from = at.chunk;
            const int r0 = at.tile * kRows + row, rows = at.q.q_len * a.group, head = at.head;
            const uint16_t *x0 = nullptr, *x1 = nullptr;
            see0 = see1 = 0x7fffffff;                // rows that are none see all there is, of a query of zeros
            if (r0 < rows) {
                const int t = r0 / a.group;
                x0 = a.q + (long long)(at.q.q0 + t) * a.q_stride + (long long)(head * a.group + r0 - t * a.group) * a.q_head;
                see0 = sees(at.q, t);
            }
            if (r0 + 8 < rows) {
                const int t = (r0 + 8) / a.group;
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
#pragma unroll
            for (int t = 0; t < F::kTiles; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.0f;
        }
        if (TMA) {
            ptx::mbar_wait(&full[stage], parity, s_word + 15, b.status, 0xA10u);
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
                const float c0 = n0 == m0 ? 1.0f : ex2(m0 - n0), c1 = n1 == m1 ? 1.0f : ex2(m1 - n1);
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
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                t[n][0] = ex2(t[n][0] - b0);
                t[n][1] = ex2(t[n][1] - b0);
                t[n][2] = ex2(t[n][2] - b1);
                t[n][3] = ex2(t[n][3] - b1);
                l0 += t[n][0] + t[n][1];
                l1 += t[n][2] + t[n][3];
            }
            const uint32_t pf[4] = {pack_bf16(t[0][0], t[0][1]), pack_bf16(t[0][2], t[0][3]), pack_bf16(t[1][0], t[1][1]), pack_bf16(t[1][2], t[1][3])};
            const int tok = lane & 15;
            uint32_t off[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) off[i] = vs + tok * 128 + (((i * 2 + (lane >> 4)) ^ (tok & 7)) << 4);
#pragma unroll
            for (int c = 0; c < F::kTiles; c += 2) {
                uint32_t r[4];
                ldmatrix_x4_trans(r, off[c / 2 & 3] + (c >> 3) * (kGroup * 128));
                ptx::mma_bf16_16x8x16(o[c], pf, r[0], r[1]);
                ptx::mma_bf16_16x8x16(o[c + 1], pf, r[2], r[3]);
            }
        }
        if (++stage == F::kStages) {
            stage = 0;
            parity ^= 1u;
        }
        if (++at.chunk < at.to) continue;

        // ---- the item (or this block's part of it) is through
        fresh = true;
        const bool whole = from == 0 && at.to == at.n.chunks;
        const int r_first = at.tile * kRows + row, rows = at.q.q_len * a.group, head = at.head;
        // row r's place in out or gate
        auto row_of = [&](int r, long long stride, long long head_stride) {
            const int t = a.group == 1 ? r : r / a.group;
            return (long long)(at.q.q0 + t) * stride + (long long)(head * a.group + r - t * a.group) * head_stride + (lane & 3) * 2;
        };
        // the i-th tile whose sum this warp writes: as the rounds go through them
        auto tile_of = [&](int i) {
            constexpr int kPer = F::kWarpTiles / F::kRounds;
            const int tile = i % kPer * F::kWarps + warp;
            return tile / F::kRoundTiles * F::kTiles + i / kPer * F::kRoundTiles + tile % F::kRoundTiles;
        };
        // the gates of this thread's values, asked for in front of the barriers
        uint32_t gates[F::kWarpTiles][2];
        auto ask_gates = [&]() {
            if (!a.gate) return;
            const uint16_t* g0 = a.gate + (r_first < rows ? row_of(r_first, a.g_stride, a.g_head) : 0);
            const uint16_t* g1 = a.gate + (r_first + 8 < rows ? row_of(r_first + 8, a.g_stride, a.g_head) : 0);
#pragma unroll
            for (int i = 0; i < F::kWarpTiles; ++i) {
                gates[i][0] = r_first < rows ? *reinterpret_cast<const uint32_t*>(g0 + tile_of(i) * 8) : 0u;
                gates[i][1] = r_first + 8 < rows ? *reinterpret_cast<const uint32_t*>(g1 + tile_of(i) * 8) : 0u;
            }
        };
        uint16_t* const out0 = a.out + (r_first < rows ? row_of(r_first, a.o_stride, a.o_head) : 0);
        uint16_t* const out1 = a.out + (r_first + 8 < rows ? row_of(r_first + 8, a.o_stride, a.o_head) : 0);
        // two columns of a row's result, gated, rounded once
        auto write = [&](bool there, uint16_t* to, uint32_t gate, float x, float y) {
            if (a.gate) {
                x /= 1.0f + __expf(-__uint_as_float(gate << 16));
                y /= 1.0f + __expf(-__uint_as_float(gate & 0xFFFF0000u));
            }
            if (there) *reinterpret_cast<uint32_t*>(to) = pack_bf16(x, y);
        };
        if (whole) ask_gates();
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

        const int first = block_of(cost, blocks, at.at + kItemCost);
        const int count = whole ? 1 : block_of(cost, blocks, at.at + kItemCost + at.n.chunks - 1) - first + 1;
        float* part = p.parts + (size_t)(blockIdx.x * 2 + (first == (int)blockIdx.x ? 1 : 0)) * kPartFloats;
        float f0[F::kGroups], f1[F::kGroups], top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int rd = 0; rd < F::kRounds; ++rd) {
            __syncthreads();                         // the round before is out of the shared arrays
#pragma unroll
            for (int i = 0; i < F::kRoundTiles; ++i) {
                const float(&x)[4] = o[rd * F::kRoundTiles + i];
                merge[(warp * F::kRoundTiles + i) * 32 + lane] = make_float4(x[0], x[1], x[2], x[3]);
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
            for (int i = 0; i < F::kWarpTiles / F::kRounds; ++i) {
                const int tile = i * F::kWarps + warp, half = tile / F::kRoundTiles, in_half = tile % F::kRoundTiles;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < F::kGroups; ++w) {
                    const float4 y = merge[((w * F::kHalves + half) * F::kRoundTiles + in_half) * 32 + lane];
                    x.x = fmaf(y.x, f0[w], x.x);
                    x.y = fmaf(y.y, f0[w], x.y);
                    x.z = fmaf(y.z, f1[w], x.z);
                    x.w = fmaf(y.w, f1[w], x.w);
                }
                const int mine = rd * (F::kWarpTiles / F::kRounds) + i, nt = tile_of(mine);
                if (whole) {
                    write(r_first < rows, out0 + nt * 8, gates[mine][0], x.x, x.y);
                    write(r_first + 8 < rows, out1 + nt * 8, gates[mine][1], x.z, x.w);
                } else {
                    __stcg(reinterpret_cast<float4*>(part) + nt * 32 + lane, x);
                }
            }
        }
        if (!whole) {
            if (warp == 0 && (lane & 3) == 0) {
                float* ml = part + kRows * D;
                __stcg(ml + row, top0);
                __stcg(ml + row + 8, top1);
                __stcg(ml + kRows + row, sum0);
                __stcg(ml + kRows + row + 8, sum1);
            }
            auto part_of = [&](int i) { return p.parts + (size_t)((first + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats; };
            // whether this block is the last of n at a counter, which is then at zero again
            auto last_of = [&](unsigned int* counter, int n) {
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    s_word[0] = atomicAdd(counter, 1u) == (unsigned)(n - 1);
                    if (s_word[0]) *counter = 0u;
                }
                __syncthreads();
                const bool last = s_word[0] != 0;
                if (last) __threadfence();
                return last;
            };
            float* weight = reinterpret_cast<float*>(merge);            // [part][row], then the rows' 1 / sum behind them
            // adds parts i0, i0 + by, ...: into the result, or into part i0
            auto add_parts = [&](int i0, int by, int n, bool final) {
                if (final) ask_gates();
                if (warp == 0) {
                    const int r = lane & 15;
                    float m[kMaxAdded / 2], l[kMaxAdded / 2], top = -INFINITY, sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < kMaxAdded / 2; ++j) {
                        const int i = 2 * j + (lane >> 4);
                        const float* ml = part_of(i0 + min(i, n - 1) * by) + kRows * D;
                        m[j] = i < n ? __ldcg(ml + r) : -INFINITY;
                        l[j] = __ldcg(ml + kRows + r);
                    }
#pragma unroll
                    for (int j = 0; j < kMaxAdded / 2; ++j) top = fmaxf(top, m[j]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
#pragma unroll
                    for (int j = 0; j < kMaxAdded / 2; ++j) {
                        const int i = 2 * j + (lane >> 4);
                        const float f = m[j] == -INFINITY ? 0.0f : ex2(m[j] - top);
                        if (i < n) weight[i * kRows + r] = f;
                        sum += f * l[j];
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    if (lane < 16) weight[n * kRows + r] = !final ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
                    __syncwarp();
                    if (!final && lane < 16) {
                        __stcg(part_of(i0) + kRows * D + r, top);
                        __stcg(part_of(i0) + kRows * D + kRows + r, sum);
                    }
                }
                __syncthreads();
                constexpr int kT = F::kWarpTiles, kP = 16 / kT;      // loads under way: 16 of 16 bytes a thread
                const float w0n = weight[n * kRows + row], w1n = weight[n * kRows + row + 8];
                float4 x[kT];
#pragma unroll
                for (int t = 0; t < kT; ++t) x[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int i = 0; i < n; i += kP) {
                    float4 y[kP][kT];
#pragma unroll
                    for (int j = 0; j < kP; ++j) {
                        const float4* from = reinterpret_cast<const float4*>(part_of(i0 + min(i + j, n - 1) * by)) + lane;
#pragma unroll
                        for (int t = 0; t < kT; ++t) y[j][t] = __ldcg(from + tile_of(t) * 32);
                    }
#pragma unroll
                    for (int j = 0; j < kP; ++j) {
                        if (i + j >= n) continue;
                        const float w0 = weight[(i + j) * kRows + row], w1 = weight[(i + j) * kRows + row + 8];
#pragma unroll
                        for (int t = 0; t < kT; ++t) {
                            x[t].x = fmaf(y[j][t].x, w0, x[t].x);
                            x[t].y = fmaf(y[j][t].y, w0, x[t].y);
                            x[t].z = fmaf(y[j][t].z, w1, x[t].z);
                            x[t].w = fmaf(y[j][t].w, w1, x[t].w);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < kT; ++t) {
                    if (final) {
                        write(r_first < rows, out0 + tile_of(t) * 8, gates[t][0], x[t].x * w0n, x[t].y * w0n);
                        write(r_first + 8 < rows, out1 + tile_of(t) * 8, gates[t][1], x[t].z * w1n, x[t].w * w1n);
                    } else {
                        __stcg(reinterpret_cast<float4*>(part_of(i0)) + tile_of(t) * 32 + lane, x[t]);
                    }
                }
            };
            const Join join = join_of(count);
            const int my_run = ((int)blockIdx.x - first) / join.run_len, in_run = min(join.run_len, count - my_run * join.run_len);
            if (last_of(p.counters + run_counter(first, my_run, join.run_len), in_run)) {
                if (join.runs == 1) {
                    add_parts(0, 1, count, true);
                } else {
                    if (in_run > 1) add_parts(my_run * join.run_len, 1, in_run, false);
                    if (last_of(p.counters + item_counter(first), join.runs)) add_parts(0, join.run_len, join.runs, true);
                }
            }
        }
        if (F::kHalves == 2) __syncthreads();        // the next item's scores go where the results were added
        more = at.next_item(p, c0, c1);
    }
    if (!TMA) cp_async_wait<0>();
}

template <int D, bool TMA>
cudaError_t launch(const CUtensorMap& tmk, const CUtensorMap& tmv, const DecodeParams& p, int blocks, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(Form<D>::kThreads);
    cfg.dynamicSmemBytes = Form<D>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, TMA>, tmk, tmv, p);
}

template <int D>
cudaError_t launch(const DecodeParams& p, int blocks, cudaStream_t s) {
    CUtensorMap tmk{}, tmv{};
    if (p.piece && make_cache_map(&tmk, p.a.b, p.a.b.k, p.piece, p.piece == kGroup ? Form<D>::kWidth / 64 : 1) &&
        make_cache_map(&tmv, p.a.b, p.a.b.v, p.piece, p.piece == kGroup ? Form<D>::kWidth / 64 : 1))
        return launch<D, true>(tmk, tmv, p, blocks, s);
    return launch<D, false>(tmk, tmv, p, blocks, s);
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

size_t paged_scratch_bytes(int sm_count) { return kCounterBytes + (size_t)sm_count * 2 * kPartFloats * sizeof(float); }

cudaError_t configure_paged_decode() {
    cudaError_t e = configure_large_smem(paged_decode_kernel<64, true>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<128, true>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<256, true>, Form<256>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<64, false>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<128, false>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<256, false>, Form<256>::kSmem);
    return e;
}

cudaError_t launch_paged_decode(const paged::AttentionArgs& a, const nvfp4_device_info& dev, void* scratch, int* launches, cudaStream_t s) {
    DecodeParams p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.min_cost = 4;
    p.most_rows = 0x7fffffff;
    p.piece = a.b.page_size % 16 == 0 ? 16 : a.b.page_size % 8 == 0 ? 8 : 0;
    p.counters = static_cast<unsigned int*>(scratch);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + kCounterBytes);
    const int blocks = dev.sm_count < kMaxBlocks ? dev.sm_count : kMaxBlocks;
    *launches = 1;
    return a.b.head_dim == 64 ? launch<64>(p, blocks, s) : a.b.head_dim == 128 ? launch<128>(p, blocks, s) : launch<256>(p, blocks, s);
}

}  // namespace nvfp4
