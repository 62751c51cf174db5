// Attention of many new tokens over the paged cache (prompts, chunks of prompts, batches that mix them with others): causal attention on the
// tensor cores, one pass over keys and values with a running maximum and sum.
//
//   S = Q K^T,   P = 2^(scale * log2(e) * S - m),   O = O * 2^(m_old - m) + P V,   l = l * 2^(m_old - m) + P 1,   out = O / l
//
// A tile is 128 rows of (new token, query head of the group): the group's heads share keys and values, so a short chunk of a prompt fills
// tiles too.  Heads of 256 take one tile at a time (512 columns of tensor memory: results 256, scores 2 x 128), smaller heads two tiles that share
// every key and value (results 2 x D, scores 2 x 128).  Keys come 128 at a time (a unit).
//   warp 0       TMA producer: the tiles of q once per item; keys and values through a ring of slots of 32 KB (16 KB for heads of 64; keys: 128 tokens
//                of up to 128 elements; values: whole heads of up to 128 tokens, so a slot holds whole steps of the second product), page by page.
//   warp 1       issues S = Q K^T: tcgen05.mma 128 x 128 x 16, both operands from shared memory.
//   warp 2       issues O += P V: 128 x D x 16, P from tensor memory over the scores it came from, V in shared memory as it lies in the cache (its
//                tokens are the operand's long way round).  A warp of its own: an MMA costs its issuer 50-60 clocks whatever its size, a wait 130, a
//                commit 75; one warp for both, with 16 KB slots, took 5000 clocks a unit whose products take 2048.
//   warps 3..    four warps per tile, thread = row = lane of tensor memory: maximum, 2^x, sum, P.  The results follow the maximum only when it grows
//                by more than 8 (weights up to 2^8), which is rare behind the first units.
// With one tile the scores of unit j+1 are formed while unit j's weights are, with two tiles one's products run beside the other's weights.
//
// Work is shared as in the attention of few tokens: units of all (sequence, tile, head) items in order, a prompt's later tiles with more of
// them, cut into equal runs, one persistent block per SM; parts of split items (FP32 results, maxima, sums) are added by a second kernel.
// Keys behind a tile's last one and those of pages out of bounds are masked, and their values zeroed in shared memory, whatever lies there.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "nvfp4_internal.h"
#include "paged_plan.h"
#include "ptx.cuh"
#include "umma.cuh"

namespace nvfp4 {

bool make_cache_map(CUtensorMap* m, const paged::Batch& b, const void* base, int slots, int parts);

#ifndef NVFP4_NT
#define NVFP4_NT 2
#endif
namespace {

using namespace paged;

constexpr int kTile = 128;           // rows of a tile

template <int D>
struct Form {
    static constexpr int kSlotBytes = D == 64 ? 16384 : 32768;
    static constexpr int kWidth = D == 64 ? 64 : 128;            // elements of a slot of keys
    static constexpr int kNT = D == 256 ? 1 : NVFP4_NT;                 // tiles of an item
    static constexpr int kThreads = 96 + 256;
    static constexpr int kBufs = kNT == 2 ? 1 : D == 256 ? 2 : 3;       // buffers of scores of a tile
    static constexpr int kParts = D / kWidth;                    // slots of a unit's keys, and of its values
    static constexpr int kQTile = kTile * D * 2;
    static constexpr int kSlots = (224 * 1024 - kNT * kQTile) / kSlotBytes;
    static constexpr int kVTokens = kLongChunk / kParts;         // tokens of a slot of values
    static constexpr int kSCols = kNT == 2 ? 256 : kBufs * 128;  // columns of scores, those of results behind them
    static constexpr int kOCol = kSCols, kOStep = D == 64 ? 64 : 128;
    static constexpr int kOkRing = kSlots / kParts > 8 ? 16 : 8; // units whose page masks are kept: more than the ring holds
    static constexpr int kControl = 2048;
    static constexpr int kSmem = kNT * kQTile + kSlots * kSlotBytes + kControl + 1024;
};
static_assert(Form<256>::kSmem <= 232448 && Form<64>::kSmem <= 232448, "shared memory");
constexpr int kMaxPartFloats = kTile * 260;          // results, maxima and sums of one tile of 256 columns or two of 128

struct LongSplit {
    int count, q0, q_len, tile, head;
    int pad[3];
};
constexpr size_t kSplitBytes = kMaxBlocks * sizeof(LongSplit);

struct PrefillParams {
    AttentionArgs a;
    float scale_log2;
    int above_rows;                  // sequences with no more rows belong to another kernel
    int tile_tokens;                 // new tokens of a tile: 128 / group
    int k_rows, v_rows;              // tokens of a box of keys, of values
    int min_cost;
    LongSplit* split;
    float* parts;
};

// A walk over the units of a run of places.
template <int D>
struct Cursor {
    Sequence q;
    LongItems n;
    long long at;                    // the item's place
    int s, tile, head, limit, chunks, chunk, to;                 // units [chunk, to) of it are this block's; limit: keys that the tile's last token sees
    static __device__ __forceinline__ LongItems items(const PrefillParams& p, const Sequence& q) {
        return long_items_of(p.a.b, q, p.a.group, p.tile_tokens * Form<D>::kNT, p.above_rows);
    }
    __device__ __forceinline__ void set_item(long long c0, long long c1) {
        limit = long_limit(q, n, tile);
        chunks = long_chunks(limit);
        const long long u = at + kLongCost;
        chunk = (int)min(max(c0 - u, 0LL), (long long)chunks);
        to = (int)min(max(c1 - u, 0LL), (long long)chunks);
    }
    __device__ __forceinline__ bool next_item(const PrefillParams& p, long long c0, long long c1) {
        at += chunks + kLongCost;
        if (at + kLongCost >= c1) return false;
        if (++head == n.heads) {
            head = 0;
            if (++tile == n.tiles) {
                tile = 0;
                do {
                    q = sequence(p.a.b, ++s);
                    n = items(p, q);
                } while (n.tiles == 0 && s + 1 < p.a.b.sequences);
            }
        }
        set_item(c0, c1);
        return true;
    }
    // tiles of the item that have rows
    __device__ __forceinline__ int live(const PrefillParams& p) const {
        return Form<D>::kNT == 2 && q.q_len - tile * n.tile_tokens > p.tile_tokens ? 2 : 1;
    }
};

// ---------------------------------------------------------------- tcgen05, from a converged warp; one elected lane issues
// Four steps of 16 elements: A and B with rows of 128 swizzled bytes along the product's sum.
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
        "add.u64 a1, %1, 2;\n\tadd.u64 a2, %1, 4;\n\tadd.u64 a3, %1, 6;\n\t"
        "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Four steps of 16 tokens: A (P) from tensor memory, 8 columns a step; B (V) with its tokens 128 bytes apart, 2048 bytes a step.
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
        "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
        "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives once all MMAs issued so far have completed.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(ptx::smem_u32(bar)) : "memory");
}
// A slot of values: 64 elements a row, the next 64 `tokens` rows on, groups of eight tokens 1024 bytes apart (the operand's long way round).
__device__ __forceinline__ uint64_t values_desc(uint32_t addr, uint32_t tokens) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(tokens * 128 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
#define NVFP4_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define NVFP4_S8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {       // without the wait
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31}, [%32];"
        : NVFP4_R8(r, 0), NVFP4_R8(r, 8), NVFP4_R8(r, 16), NVFP4_R8(r, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31,%32};" ::"r"(taddr), NVFP4_S8(r, 0), NVFP4_S8(r, 8), NVFP4_S8(r, 16), NVFP4_S8(r, 24)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), NVFP4_S8(r, 0), NVFP4_S8(r, 8)
                 : "memory");
}
// What a load delivers is read behind the wait only: the registers pass through it.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 ::"memory");
    asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                   "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 ::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 y = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two FP32 values in one register pair, one instruction for both.
__device__ __forceinline__ uint64_t pair_bits(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair(float a, float b) { return pair_bits(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
    uint32_t x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(p));
    a = __uint_as_float(x);
    b = __uint_as_float(y);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 32 columns of a row's result, gated, rounded once.
__device__ __forceinline__ void ask_gates(const AttentionArgs& a, bool there, long long gate_at, uint4 (&g)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = a.gate && there ? *reinterpret_cast<const uint4*>(a.gate + gate_at + i * 8) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ void write32(const AttentionArgs& a, long long out_at, const uint4 (&g)[4], const float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[i * 8 + e];
        if (a.gate) {
            const uint32_t w[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[2 * e] = __fdividef(y[2 * e], 1.0f + __expf(-__uint_as_float(w[e] << 16)));
                y[2 * e + 1] = __fdividef(y[2 * e + 1], 1.0f + __expf(-__uint_as_float(w[e] & 0xFFFF0000u)));
            }
        }
        *reinterpret_cast<uint4*>(a.out + out_at + i * 8) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
    }
}

template <int D>
__global__ void __launch_bounds__(Form<D>::kThreads, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                     const __grid_constant__ PrefillParams p) {
    using F = Form<D>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* s_q = smem;
    unsigned char* ring = smem + F::kNT * F::kQTile;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + F::kSlots * F::kSlotBytes);
    uint64_t* empty = full + F::kSlots;
    uint64_t* q_full = empty + F::kSlots;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;                  // [3] scores are there
    uint64_t* p_ready = s_full + 3;                  // [3] weights are there, results scaled to them
    uint64_t* s_free = p_ready + 3;                  // [3] the weights are multiplied
    uint64_t* o_free = s_free + 3;                   // [2] the item's results are read, tile by tile
    uint64_t* drain = o_free + 2;                    // [2] the issuers' last MMAs
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drain + 2);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    unsigned int* s_ok = s_tmem + 2;                 // [kOkRing] boxes of a unit whose page is one
    long long* prefix = reinterpret_cast<long long*>(s_ok + F::kOkRing);                   // [warps] in front, then the run's first place
    Cursor<D>* found = reinterpret_cast<Cursor<D>*>(prefix + F::kThreads / 32 + 2);
    float* s_x = reinterpret_cast<float*>(found + 1);                                   // [group][row], one tile: what the two groups tell each other
    static_assert((2 * F::kSlots + 15) * 8 + 8 + F::kOkRing * 4 + (F::kThreads / 32 + 2) * 8 + sizeof(Cursor<D>) + 2 * kTile * 4 <= F::kControl, "control block");

    const AttentionArgs& a = p.a;
    const Batch& b = a.b;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < F::kSlots; ++i) { ptx::mbar_init(&full[i], 1); ptx::mbar_init(&empty[i], 1); }
        ptx::mbar_init(q_full, 1);
        ptx::mbar_init(q_empty, 1);
        for (int i = 0; i < 3; ++i) { ptx::mbar_init(&s_full[i], 1); ptx::mbar_init(&p_ready[i], 8 / F::kNT); ptx::mbar_init(&s_free[i], 1); }
        for (int i = 0; i < 2; ++i) { ptx::mbar_init(&o_free[i], 8 / F::kNT); ptx::mbar_init(&drain[i], 1); }
        *s_abort = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmq);
        ptx::prefetch_tensormap(&tmk);
        ptx::prefetch_tensormap(&tmv);
    }
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // ---- this block's run
    const int run = (b.sequences + F::kThreads - 1) / F::kThreads;
    const int s0 = min(tid * run, b.sequences), s1 = min(s0 + run, b.sequences);
    long long mine = 0;
    for (int s = s0; s < s1; ++s) {
        const Sequence q = sequence(b, s);
        const LongItems n = Cursor<D>::items(p, q);
        mine += long_places(q, n, n.tiles) * n.heads;
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
    for (int w = 0; w < F::kThreads / 32; ++w) {
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
        int s = s0;
        for (;; ++s) {
            const Sequence q = sequence(b, s);
            const LongItems n = Cursor<D>::items(p, q);
            const long long here = long_places(q, n, n.tiles) * n.heads;
            if (left < here) break;
            left -= here;
        }
        found->s = s;
        prefix[F::kThreads / 32] = left;
    }
    __syncthreads();
    if (warp == 0) {                                 // the tile, by cutting the range into 32 pieces at a time
        Cursor<D> x;
        x.s = found->s;
        x.q = sequence(b, x.s);
        x.n = Cursor<D>::items(p, x.q);
        const long long left = prefix[F::kThreads / 32];
        int lo = 0, hi = x.n.tiles;                  // places in front of tile lo <= left < those in front of tile hi
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, t = min(lo + (lane + 1) * step, hi);
            const unsigned int below = __ballot_sync(0xffffffffu, long_places(x.q, x.n, t) * x.n.heads <= left);
            const int k = __popc(below);             // the first k pieces end at or below
            const int from = lo;
            lo = min(from + k * step, hi);
            hi = min(from + (k + 1) * step, hi);
        }
        const long long at = long_places(x.q, x.n, lo) * x.n.heads;
        x.tile = lo;
        const int per = long_chunks(long_limit(x.q, x.n, lo)) + kLongCost;
        x.head = (int)((left - at) / per);
        x.at = c0 - (left - at) + (long long)x.head * per;
        x.set_item(c0, c1);
        __syncwarp();
        if (lane == 0) *found = x;
    }
    __syncwarp();
    if (warp == 2) umma::tmem_alloc_512(s_tmem);
    umma::tc_fence_before();
    __syncthreads();
    umma::tc_fence_after();
    const uint32_t tmem = *s_tmem;
    Cursor<D> at = *found;
    bool more = true;

    if (warp == 0) {
        // ------------------------------------------------------------------ producer
        int slot = 0, unit = 0;
        uint32_t phase = 0, q_phase = 0;
        const int boxes = kLongChunk / p.k_rows;
        // page and slot of the box of keys that is this lane's, in a unit
        auto look_up = [&](int chunk, int& page, int& place) {
            const int tok = chunk * kLongChunk + lane * p.k_rows;
            page = -1;
            place = 0;
            if (lane < boxes && tok < at.limit) {
                const int entry = divide(tok, b.div);
                place = tok - entry * b.page_size;
                page = b.table[(long long)at.s * b.table_stride + entry];
                if ((unsigned)page >= (unsigned)b.num_pages) {
                    atomicCAS(b.status, 0u, kStatusPlace);
                    page = -1;
                }
            }
        };
        auto next_slot = [&]() {
            if (++slot == F::kSlots) {
                slot = 0;
                phase ^= 1u;
            }
        };
        // lane = (64 elements, box of tokens)
        auto keys = [&](int page, int place) {
            const unsigned int ok = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) s_ok[unit % F::kOkRing] = ok;
            ++unit;
            const int box = lane % boxes, part = lane / boxes;
            const int pg = __shfl_sync(0xffffffffu, page, box), pl = __shfl_sync(0xffffffffu, place, box);
            const bool mine = part < F::kWidth / 64 && pg >= 0;
            for (int c = 0; c < F::kParts; ++c) {
                const bool go = ptx::mbar_wait(&empty[slot], phase ^ 1u, s_abort, b.status, 0xA20u);
                if (lane == 0 && go) ptx::mbar_arrive_expect_tx(&full[slot], (unsigned)(__popc(ok) * p.k_rows * F::kWidth * 2));
                __syncwarp();
                if (mine && go)
                    ptx::tma_load_5d(ring + slot * F::kSlotBytes + part * (kLongChunk * 128) + box * p.k_rows * 128, &tmk, &full[slot], 0, pl, c * (F::kWidth / 64) + part, at.head, pg);
                next_slot();
            }
        };
        auto values = [&](int page, int place) {
            constexpr int kAcross = D / 64;
            const int per = F::kVTokens / p.v_rows, part = lane % kAcross, box = lane / kAcross;
            for (int v = 0; v < F::kParts; ++v) {
                const int tok = v * F::kVTokens + min(box, per - 1) * p.v_rows, from = tok / p.k_rows;
                const int pg = __shfl_sync(0xffffffffu, page, from), pl = __shfl_sync(0xffffffffu, place, from) + tok - from * p.k_rows;
                const bool mine = box < per && pg >= 0;
                const unsigned int ok = __ballot_sync(0xffffffffu, mine);
                const bool go = ptx::mbar_wait(&empty[slot], phase ^ 1u, s_abort, b.status, 0xA21u);
                if (lane == 0 && go) ptx::mbar_arrive_expect_tx(&full[slot], (unsigned)(__popc(ok) * p.v_rows * 128));
                __syncwarp();
                if (mine && go)
                    ptx::tma_load_5d(ring + slot * F::kSlotBytes + part * (F::kVTokens * 128) + box * p.v_rows * 128, &tmv, &full[slot], 0, pl, part, at.head, pg);
                next_slot();
            }
        };
        while (more) {
            int page, place, page_before = -1, place_before = 0;
            look_up(at.chunk, page, place);
            const bool go = ptx::mbar_wait(q_empty, q_phase ^ 1u, s_abort, b.status, 0xA22u);
            q_phase ^= 1u;
            const int live = at.live(p);
            if (ptx::elect_one() && go) {
                ptx::mbar_arrive_expect_tx(q_full, (unsigned)(live * (D / 64) * p.tile_tokens * a.group * 128));
                for (int t = 0; t < live; ++t)
                    for (int c = 0; c < D / 64; ++c)
                        ptx::tma_load_3d(s_q + t * F::kQTile + c * (kTile * 128), &tmq, q_full, c * 64, at.head * a.group,
                                         at.q.q0 + at.tile * at.n.tile_tokens + t * p.tile_tokens);
            }
            __syncwarp();
            for (int j = at.chunk; j < at.to; ++j) {
                int page_next = -1, place_next = 0;
                if (j + 1 < at.to) look_up(j + 1, page_next, place_next);
                keys(page, place);
                if (F::kNT == 2) values(page, place);
                else if (j > at.chunk) values(page_before, place_before);
                page_before = page;
                place_before = place;
                page = page_next;
                place = place_next;
            }
            if (F::kNT == 1) values(page_before, place_before);
            more = at.next_item(p, c0, c1);
        }
        // nothing of this block's may still be on its way when it ends: every slot's last fill has been multiplied
        for (int i = 0; i < F::kSlots; ++i) {
            ptx::mbar_wait(&empty[slot], phase ^ 1u, s_abort, b.status, 0xA23u);
            next_slot();
        }
    } else if (warp <= 2) {
        // ------------------------------------------------------------------ MMA issuers
        const bool is_s = warp == 1;
        const uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(kTile >> 4) << 24 | (is_s ? (uint32_t)(kLongChunk >> 3) << 17 : 1u << 16 | (uint32_t)(D >> 3) << 17);
        // items and units so far; a second tile without rows does not count
        uint32_t item = 0, items_of[2] = {0, 0}, units_of[2] = {0, 0};
        unsigned int used = 0;                       // halves of units (keys or values) that the ring has seen
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int where) {
            ok = ptx::mbar_wait(bar, parity, s_abort, b.status, where) && ok;
            __syncwarp();
            ok = __all_sync(0xffffffffu, ok);
            umma::tc_fence_after();
        };
        while (more) {
            const int n = at.to - at.chunk, live = at.live(p);
            if (is_s) wait(q_full, item & 1u, 0xA32u);
            for (int j = 0; j < n; ++j) {
#pragma unroll
                for (int t = 0; t < F::kNT; ++t) {
                    if (t >= live) continue;
                    const uint32_t u = units_of[t] + j;
                    const int sb = F::kNT == 1 ? u % F::kBufs : t;
                    const bool release = t == live - 1;
                    // the unit's keys (values) come in this half of the ring's fills
                    const unsigned int half = used + (F::kNT == 2 ? 2 * j + !is_s : is_s ? (j ? 2 * j - 1 : 0) : (j < n - 1 ? 2 * j + 2 : 2 * n - 1));
                    if (is_s) {
                        // the buffer's weights before are multiplied
                        if (u >= F::kBufs) wait(&s_free[sb], u / F::kBufs - 1 & 1u, 0xA38u);
                    } else {
                        if (j == 0 && items_of[t] > 0) wait(&o_free[t], items_of[t] - 1 & 1u, 0xA34u);
                        wait(&p_ready[sb], u / F::kBufs & 1u, 0xA35u);
                    }
                    for (int c = 0; c < F::kParts; ++c) {
                        const unsigned int i = half * F::kParts + c;
                        const int s = (int)(i % F::kSlots);
                        if (t == 0) wait(&full[s], i / F::kSlots & 1u, is_s ? 0xA30u : 0xA31u);
                        if (!ok) continue;
                        const uint32_t from = ptx::smem_u32(ring + s * F::kSlotBytes);
                        if (is_s) {
#pragma unroll
                            for (int e = 0; e < F::kWidth / 64; ++e)
                                mma4_ss(tmem + sb * 128, umma::umma_desc_sw128(ptx::smem_u32(s_q + t * F::kQTile + (c * (F::kWidth / 64) + e) * (kTile * 128))),
                                        umma::umma_desc_sw128(from + e * (kLongChunk * 128)), idesc, c > 0 || e > 0);
                        } else {
#pragma unroll
                            for (int e = 0; e < F::kVTokens / 64; ++e)
                                mma4_ts(tmem + F::kOCol + t * F::kOStep, tmem + sb * 128 + (c * F::kVTokens + e * 64) / 2,
                                        values_desc(from, F::kVTokens) + e * 512, idesc, j > 0 || c > 0 || e > 0);
                        }
                        if (release) commit(&empty[s]);
                    }
                    if (ok) commit(is_s ? &s_full[sb] : &s_free[sb]);
                }
            }
            if (is_s && ok) commit(q_empty);
#pragma unroll
            for (int t = 0; t < F::kNT; ++t)
                if (t < live) {
                    units_of[t] += n;
                    ++items_of[t];
                }
            used += 2 * n;
            ++item;
            more = at.next_item(p, c0, c1);
        }
        commit(&drain[!is_s]);
        ptx::mbar_wait(&drain[!is_s], 0, s_abort, b.status, 0xA3Fu);
    } else {
        // ------------------------------------------------------------------ softmax: thread = row
        // Two tiles: a group of four warps each, thread = row.  One tile: the two groups share it, thread = row and 64 of the scores, half the result.
        constexpr bool kShared = F::kNT == 1;
        constexpr int kCols = kShared ? 64 : 128;
        const int g = (warp - 3) >> 2, t = kShared ? 0 : g, quarter = warp & 3, row = quarter * 32 + lane, s_col = kShared ? g * 64 : 0;
        const int col0 = kShared ? g * (D / 2) : 0, col1 = kShared ? col0 + D / 2 : D;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), o_addr = lanes + F::kOCol + t * F::kOStep;
        uint32_t unit = 0;                           // of this tile so far
        unsigned int used = 0;
        uint32_t units_seen = 0;                     // of the block, for the page masks
        // the other group's value of this row
        auto exchange = [&](float x) {
            s_x[g * kTile + row] = x;
            ptx::named_barrier_sync(1 + quarter, 64);
            const float y = s_x[(1 - g) * kTile + row];
            ptx::named_barrier_sync(1 + quarter, 64);
            return y;
        };
        while (more) {
            const int n = at.to - at.chunk;
            const bool live = t < at.live(p);
            const int tok = at.tile * at.n.tile_tokens + t * p.tile_tokens + row / a.group, hd = at.head * a.group + row % a.group;
            const bool there = row < p.tile_tokens * a.group && tok < at.q.q_len;
            const int see = there ? sees(at.q, tok) : 0x7fffffff;
            const bool whole = at.chunk == 0 && at.to == at.chunks;
            const int first = block_of(cost, blocks, at.at + kLongCost);
            if (!whole && first == (int)blockIdx.x && tid == 96)
                p.split[blockIdx.x] = LongSplit{block_of(cost, blocks, at.at + kLongCost + at.chunks - 1) - first + 1, at.q.q0, at.q.q_len, at.tile, at.head, {0, 0, 0}};
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; live && j < n; ++j, ++unit) {
                const int sb = F::kNT == 1 ? unit % F::kBufs : t;
                const uint32_t s_addr = lanes + sb * 128;
                ptx::mbar_wait(&s_full[sb], unit / F::kBufs & 1u, s_abort, b.status, 0xA40u);
                __syncwarp();
                umma::tc_fence_after();
                const int key0 = (at.chunk + j) * kLongChunk;
                const unsigned int ok = s_ok[(units_seen + j) % F::kOkRing], all = (1u << (kLongChunk / p.k_rows)) - 1u;
                if (key0 + kLongChunk > at.limit || ok != all) {
                    if (t == 0 && (!kShared || D > 64 || g == 0)) {
                        // values of keys that no row sees: whatever lies there, a weight of zero times it is to be zero
                        const int box = row / p.k_rows;
                        const bool none = key0 + row >= at.limit || !(ok >> box & 1u);
                        const unsigned int half = used + (F::kNT == 2 ? 2 * j + 1 : j < n - 1 ? 2 * j + 2 : 2 * n - 1);
                        const unsigned int i = half * F::kParts + row / F::kVTokens;
                        const int slot = (int)(i % F::kSlots);
                        ptx::mbar_wait(&full[slot], i / F::kSlots & 1u, s_abort, b.status, 0xA41u);
                        if (none) {
                            const uint32_t to = ptx::smem_u32(ring + slot * F::kSlotBytes) + row % F::kVTokens * 128;
#pragma unroll
                            for (int c = kShared && D > 64 ? g * (D / 128) : 0; c < (kShared && D > 64 ? (g + 1) * (D / 128) : D / 64); ++c)
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(to + c * (F::kVTokens * 128) + e * 16), "r"(0u) : "memory");
                        }
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                uint32_t s[kCols];
#pragma unroll
                for (int q = 0; q < kCols / 32; ++q) tmem_ld32(s_addr + s_col + q * 32, s + q * 32);
#pragma unroll
                for (int q = 0; q < kCols / 32; ++q) tmem_wait_ld32(s + q * 32);
                const int seen = see - key0 - s_col; // of this thread's columns those in front of this one
                const bool masked = __any_sync(0xffffffffu, there && seen < kCols) || ok != all;
                auto mask = [&](int q) {
                    const int box_log = 31 - __clz(p.k_rows);
                    unsigned int keep = seen >= q * 32 + 32 ? 0xffffffffu : seen <= q * 32 ? 0u : (1u << (seen - q * 32)) - 1u;
                    if (!(ok >> ((s_col + q * 32) >> box_log) & 1u)) keep &= 0xffff0000u;
                    if (!(ok >> ((s_col + q * 32 + 16) >> box_log) & 1u)) keep &= 0x0000ffffu;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(keep >> i & 1u)) s[q * 32 + i] = 0xff800000u;
                };
                if (masked) {
#pragma unroll
                    for (int q = 0; q < kCols / 32; ++q) mask(q);
                }
                float top[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) top[i] = fmaxf(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
#pragma unroll
                for (int i = 8; i < kCols; i += 2) top[i / 2 & 3] = max3(top[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                float now = max3(fmaxf(top[0], top[1]), top[2], top[3]) * p.scale_log2;
                if (kShared) now = fmaxf(now, exchange(now));
                if (__any_sync(0xffffffffu, there && now > m + 8.0f)) {
                    const float next = fmaxf(m, now), back = next == m ? 1.0f : ex2(m - next);
                    m = next;
                    l *= back;
                    if (j > 0) {                     // the results so far follow, once the product before is through
                        const uint32_t u = unit - 1;
                        ptx::mbar_wait(&s_free[F::kNT == 1 ? u % F::kBufs : t], u / F::kBufs & 1u, s_abort, b.status, 0xA42u);
                        __syncwarp();
                        umma::tc_fence_after();
#pragma unroll 1
                        for (int c = col0; c < col1; c += 32) {
                            uint32_t x[32];
                            tmem_ld32(o_addr + c, x);
                            tmem_wait_ld32(x);
#pragma unroll
                            for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * back);
                            tmem_st32(o_addr + c, x);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m;
                const uint64_t scale2 = pair(p.scale_log2, p.scale_log2), base2 = pair(-base, -base);
                uint64_t sum[2] = {0, 0};            // two sums each
#pragma unroll
                for (int q = 0; q < kCols / 32; ++q) {
                    uint32_t w[16];
                    if (q == 3) {
                        tmem_wait_ld32(s + q * 32);
                        if (masked) mask(q);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x, y;
                        unpair(fma2(pair_bits(s[q * 32 + 2 * i], s[q * 32 + 2 * i + 1]), scale2, base2), x, y);
                        x = ex2(x);
                        y = ex2(y);
                        sum[i & 1] = add2(sum[i & 1], pair(x, y));
                        w[i] = pack_bf16(x, y);
                    }
                    tmem_st16(s_addr + s_col / 2 + q * 16, w);         // over scores that are read
                    // 128 scores and the weights pass the 168 registers of 352 threads: the last 32 are read again rather than kept
                    if (kCols == 128 && q == 0) tmem_ld32(s_addr + 96, s + 96);
                }
                {
                    float x, y;
                    unpair(add2(sum[0], sum[1]), x, y);
                    l += x + y;
                }
                tmem_wait_st();
                umma::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&p_ready[sb]);
            }
            units_seen += n;
            used += 2 * n;
            // ---- the item, or this block's part of it
            if (live) {
                const uint32_t u = unit - 1;
                const long long tq = at.q.q0 + tok, out_at = tq * a.o_stride + (long long)hd * a.o_head, gate_at = tq * a.g_stride + (long long)hd * a.g_head;
                uint4 gates[2][4];                   // asked for 32 columns ahead
                ask_gates(a, there && whole, gate_at + col0, gates[0]);
                ptx::mbar_wait(&s_free[F::kNT == 1 ? u % F::kBufs : t], u / F::kBufs & 1u, s_abort, b.status, 0xA43u);
                __syncwarp();
                umma::tc_fence_after();
                if (kShared) {
                    const float other = exchange(l);
                    l = g == 0 ? l + other : other + l;
                }
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                float* part = p.parts + (size_t)part_slot(first, blockIdx.x) * kMaxPartFloats;
                const int prow = t * kTile + row;
#pragma unroll 2
                for (int c = col0; c < col1; c += 32) {
                    uint32_t x[32];
                    tmem_ld32(o_addr + c, x);
                    if (c + 32 < col1) ask_gates(a, there && whole, gate_at + c + 32, gates[((c - col0) / 32 + 1) & 1]);
                    tmem_wait_ld32(x);
                    if (whole) {
                        float y[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] = l == 0.0f ? 0.0f : __uint_as_float(x[i]) * inv;
                        if (there) write32(a, out_at + c, gates[(c - col0) / 32 & 1], y);
                        __syncwarp();
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            __stcg(reinterpret_cast<float4*>(part) + (c / 4 + i) * (F::kNT * kTile) + prow,
                                   make_float4(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1]), __uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3])));
                    }
                }
                if (!whole && col0 == 0) {
                    float* ml = part + F::kNT * kTile * D;
                    __stcg(ml + prow, m);
                    __stcg(ml + F::kNT * kTile + prow, l);
                }
                umma::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&o_free[t]);
            }
            more = at.next_item(p, c0, c1);
        }
    }
    umma::tc_fence_before();
    __syncthreads();
    umma::tc_fence_after();
    __syncwarp();
    if (warp == 2) umma::tmem_dealloc_512(tmem);
}

// Adds the parts of split items in the order of their blocks.  A warp takes 32 rows and 16 columns of an item; four parts are under way at once.
constexpr int kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads)
paged_prefill_join_kernel(const __grid_constant__ PrefillParams p, int blocks) {
    using F = Form<D>;
    constexpr int kRowGroups = F::kNT * kTile / 32, kPieces = kRowGroups * (D / 16);          // warps of an item
    __shared__ LongSplit s_item[kMaxBlocks];
    __shared__ int s_first[kMaxBlocks], s_count[kJoinThreads / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    static_assert(kMaxBlocks == kJoinThreads, "a thread looks at a block");
    LongSplit mine{};
    if (tid < blocks) {
        const int4 x = __ldcg(reinterpret_cast<const int4*>(p.split + tid));
        mine.count = x.x; mine.q0 = x.y; mine.q_len = x.z; mine.tile = x.w;
        mine.head = __ldcg(&p.split[tid].head);
    }
    const unsigned int vote = __ballot_sync(0xffffffffu, mine.count > 0);
    if (lane == 0) s_count[warp] = __popc(vote);
    __syncthreads();
    int items = 0, index = __popc(vote & ((1u << lane) - 1u));
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) {
        if (w < warp) index += s_count[w];
        items += s_count[w];
    }
    if (mine.count > 0) {
        s_item[index] = mine;
        s_first[index] = tid;
    }
    __syncthreads();
    for (int work = blockIdx.x * (kJoinThreads / 32) + warp; work < items * kPieces; work += gridDim.x * (kJoinThreads / 32)) {
        const LongSplit it = s_item[work / kPieces];
        const int first = s_first[work / kPieces], piece = work % kPieces, prow = piece % kRowGroups * 32 + lane, c0 = piece / kRowGroups * 16;
        const int t = prow / kTile, row = prow % kTile, rows = p.tile_tokens * p.a.group;
        const int tok = it.tile * (p.tile_tokens * F::kNT) + t * p.tile_tokens + row / p.a.group;
        const bool there = row < rows && tok < it.q_len;
        if (!__any_sync(0xffffffffu, there)) continue;
        float top = -INFINITY, den = 0.0f;
        float x[16] = {};
        for (int i0 = 0; i0 < it.count; i0 += 4) {
            float4 y[4][4];
            float m[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* part = p.parts + (size_t)part_slot(first, first + min(i0 + j, it.count - 1)) * kMaxPartFloats;
                m[j] = __ldcg(part + F::kNT * kTile * D + prow);
                l[j] = __ldcg(part + F::kNT * kTile * (D + 1) + prow);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[j][e] = __ldcg(reinterpret_cast<const float4*>(part) + (c0 / 4 + e) * (F::kNT * kTile) + prow);
            }
            float now = top;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i0 + j < it.count) now = fmaxf(now, m[j]);
            const float back = top == -INFINITY ? 0.0f : ex2(top - now);
            top = now;
            den *= back;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] *= back;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i0 + j >= it.count || m[j] == -INFINITY) continue;
                const float w = ex2(m[j] - now);
                den += w * l[j];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[4 * e] = fmaf(y[j][e].x, w, x[4 * e]);
                    x[4 * e + 1] = fmaf(y[j][e].y, w, x[4 * e + 1]);
                    x[4 * e + 2] = fmaf(y[j][e].z, w, x[4 * e + 2]);
                    x[4 * e + 3] = fmaf(y[j][e].w, w, x[4 * e + 3]);
                }
            }
        }
        if (!there) continue;
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        const AttentionArgs& a = p.a;
        const long long tq = it.q0 + tok, hd = it.head * a.group + row % a.group;
        const uint16_t* gate = a.gate ? a.gate + tq * a.g_stride + hd * a.g_head + c0 : nullptr;
        uint16_t* out = a.out + tq * a.o_stride + hd * a.o_head + c0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t w[4];
            const uint4 g4 = gate ? *reinterpret_cast<const uint4*>(gate + i * 8) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t g[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float u = x[i * 8 + 2 * e] * inv, v = x[i * 8 + 2 * e + 1] * inv;
                if (gate) {
                    u /= 1.0f + __expf(-__uint_as_float(g[e] << 16));
                    v /= 1.0f + __expf(-__uint_as_float(g[e] & 0xFFFF0000u));
                }
                w[e] = pack_bf16(u, v);
            }
            *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
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

int common_divisor(int a, int b) { return b ? common_divisor(b, a % b) : a; }

// q as [token][head][head_dim]: a box of a tile's tokens, a group's heads and 64 elements, rows of 128 bytes swizzled.
bool make_q_map(CUtensorMap* m, const AttentionArgs& a, int tile_tokens) {
    umma::EncodeFn enc = umma::get_encode();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a.b.head_dim, (cuuint64_t)a.q_heads, (cuuint64_t)a.b.tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)tile_tokens}, estr[3] = {1, 1, 1};
    for (const cuuint64_t x : strides)
        if (x >= 1ull << 40) return false;
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
bool make_maps(CUtensorMap (&maps)[3], PrefillParams& p) {
    using F = Form<D>;
    p.tile_tokens = kTile / p.a.group;
    p.k_rows = common_divisor(p.a.b.page_size, kLongChunk);
    p.v_rows = common_divisor(p.a.b.page_size, F::kVTokens);
    return make_q_map(&maps[0], p.a, p.tile_tokens) && make_cache_map(&maps[1], p.a.b, p.a.b.k, p.k_rows, 1) && make_cache_map(&maps[2], p.a.b, p.a.b.v, p.v_rows, 1);
}

template <int D>
bool launch(PrefillParams& p, const nvfp4_device_info& dev, cudaStream_t s, cudaError_t* e) {
    CUtensorMap maps[3];
    if (!make_maps<D>(maps, p)) return false;
    const int blocks = dev.sm_count < kMaxBlocks ? dev.sm_count : kMaxBlocks;
    *e = launch_behind(paged_prefill_kernel<D>, blocks, Form<D>::kThreads, Form<D>::kSmem, s, maps[0], maps[1], maps[2], p);
    if (*e == cudaSuccess) *e = launch_behind(paged_prefill_join_kernel<D>, 2 * blocks, kJoinThreads, 0, s, p, blocks);
    return true;
}

}  // namespace

size_t paged_prefill_scratch_bytes(int sm_count) {
    return kSplitBytes + (size_t)(sm_count < kMaxBlocks ? sm_count : kMaxBlocks) * 2 * kMaxPartFloats * sizeof(float);
}

cudaError_t configure_paged_prefill() {
    cudaError_t e = configure_large_smem(paged_prefill_kernel<64>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_prefill_kernel<128>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_prefill_kernel<256>, Form<256>::kSmem);
    return e;
}

// Whole boxes of 16 tokens, a group of heads that fits a tile, a maximum that grows with the products.
bool paged_prefill_supported(const paged::AttentionArgs& a) { return a.b.page_size % 16 == 0 && a.group <= kTile && a.scale > 0.0f; }

bool launch_paged_prefill(const paged::AttentionArgs& a, int above_rows, const nvfp4_device_info& dev, void* scratch, int* launches, cudaStream_t s, cudaError_t* e) {
    PrefillParams p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.above_rows = above_rows;
    p.min_cost = 4;
    p.split = static_cast<LongSplit*>(scratch);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + kSplitBytes);
    const bool done = a.b.head_dim == 64 ? launch<64>(p, dev, s, e) : a.b.head_dim == 128 ? launch<128>(p, dev, s, e) : launch<256>(p, dev, s, e);
    if (done) *launches = 2;
    return done;
}

}  // namespace nvfp4
