// Attention of many new tokens over the paged cache (prompts, chunks of prompts, batches that mix them with others): causal attention on the
// tensor cores, one pass over keys and values with a running maximum and sum.
//
//   S = Q K^T,   P = 2^(scale * log2(e) * S - m),   O = O * 2^(m_old - m) + P V,   l = l * 2^(m_old - m) + P 1,   out = O / l
//
// A tile is 128 rows of (new token, query head of the group): the group's heads share keys and values, so a short chunk of a prompt fills
// tiles too.  A pair of SMs (a cluster of two CTAs, tcgen05.mma.cta_group::2, M = 256) takes two tiles at once, or four with heads of up to 128
// (each CTA's tensor memory: results 256 columns, scores 2 x 128), that share every key and value: each CTA holds half of a unit's keys and half of
// its values' columns (heads of 64: all of them, the product's other half is left unread).  Alone on an SM the first product is bound by shared
// memory (128 bytes a clock for its two operands, beside the loads): 1800 clocks for 128 x 128 x 256 instead of 1024.  Keys come 128 at a time (a unit).
//   warp 0       of both: TMA producer: its tiles of q once per item; its halves of keys and values, one ring slot each, page by page.
//   warp 1       of the leader issues S = Q K^T: 256 x 128 x 16, both operands from shared memory.
//   warp 2       of the leader issues O += P V: 256 x D x 16, P from tensor memory over the scores it came from, V in shared memory as it lies in the
//                cache (its tokens are the operand's long way round).  A warp of its own: an MMA costs its issuer 50-60 clocks whatever its size,
//                a wait 130, a commit 75; one warp for both took 5000 clocks a unit whose products take 2048.
//   warps 3-10   of both: maximum, 2^x, sum, P: two groups of four warps share a tile, thread = row and 64 of the scores.  (A group of its own for each
//                tile ran in step with the other, both waiting for the tensor core and then for the one unit that does 2^x.)  The results follow the
//                maximum only when it grows by more than 8 (weights up to 2^8), which is rare behind the first units.
// Scores have two buffers, so that a unit's weights are formed while the tensor core multiplies the ones before and forms the next unit's scores.
//
// Work is shared as in the attention of few tokens: units of all (sequence, tiles, head) items in order, a prompt's later tiles with more of
// them, cut into equal runs, one persistent pair of blocks per pair of SMs; parts of split items (FP32 results, maxima, sums) are added by a second kernel.
// Keys behind the item's last one and those of pages out of bounds are masked, and their values zeroed in shared memory, whatever lies there.
//
// Measured, call after call under the power cap: a chunk of 256 tokens behind 16384 (24 heads over 2 of 256) 112-115 us at 1.7 GHz, 0.90 to 0.93 PFLOP/s; a prompt
// of 8192 815-841 us at 1.6 GHz, 0.98 to 1.01 PFLOP/s (747 us in the first calls behind a pause); 149 tokens 18 us, of which the products are 1; a prompt
// of 4096, 32 heads over 8 of 128, 175 us, 0.79 PFLOP/s, and of 64 148 us, 0.47.  A unit takes 2600 clocks with heads of 256 (products 2 x 1024, but the first one
// waits for shared memory, 1500, and the second for tensor memory's operand, 1490; the weights 1900, over two buffers), 4200 for four tiles of 128; an item
// several thousand for its way out (results from tensor memory, gates, rows written), which only the next item's loads and first scores overlap.
//
// The weights are rounded to BF16 for the second product, off by up to 2^-8 of each, which is the result's own rounding once more: 0.0018 to 0.0023 of the
// result's norm against 64 bits, where one rounding has 0.0017.  A second operand with the remainders, as with few tokens, would be half as many products again.
#include <cuda.h>
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

constexpr int kTile = 128;           // rows of a tile

template <int D>
struct Form {
    static constexpr int kNT = D == 256 ? 1 : 2;                 // tiles of a CTA
    static constexpr int kThreads = 96 + 256;
    static constexpr int kBufs = kNT == 2 ? 1 : 2;               // buffers of scores of a tile
    static constexpr int kVCols = D == 64 ? 64 : D / 2;          // columns of the values that a CTA holds
    static constexpr int kOCols = 2 * kVCols;                    // columns of the second product
    static constexpr int kKeys = kLongChunk / 2;                 // keys of a unit that a CTA holds
    static constexpr int kSlotBytes = kLongChunk * kVCols * 2;   // a CTA's values of a unit, or its keys (no more bytes)
    static constexpr int kQTile = kTile * D * 2;
    static constexpr int kSlots = (224 * 1024 - kNT * kQTile) / kSlotBytes;
    static constexpr int kOCol = 256;                            // scores in front: buffer or tile 0, 1
    static constexpr int kOkRing = 16;                           // units whose page masks are kept: more than the ring holds
    static constexpr int kControl = 3 * 1024;
    static constexpr int kSmem = kNT * kQTile + kSlots * kSlotBytes + kControl;
};
static_assert(Form<256>::kSmem <= 232448 && Form<128>::kSmem <= 232448 && Form<64>::kSmem <= 232448, "shared memory");
static_assert(Form<256>::kSlots >= 4 && Form<128>::kSlots >= 4 && Form<64>::kSlots / 2 < Form<64>::kOkRing, "ring");
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
    int box_rows, box_log;           // tokens of a box of keys or values (16, 32 or 64)
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
        return long_items_of(p.a.b, q, p.a.group, p.tile_tokens * Form<D>::kNT * 2, p.above_rows);
    }
    __device__ __forceinline__ void set_item(long long c0, long long c1) {
        limit = long_limit(q, n, tile);
        chunks = long_chunks(limit);
        const long long u = at + n.extra;
        chunk = (int)min(max(c0 - u, 0LL), (long long)chunks);
        to = (int)min(max(c1 - u, 0LL), (long long)chunks);
    }
    __device__ __forceinline__ bool next_item(const PrefillParams& p, long long c0, long long c1) {
        at += chunks + n.extra;
        if (at + n.extra >= c1) return false;
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
    // tiles of a CTA that have rows, in one of the two at least: the item's tiles go to (CTA 0, 1) and then to their second ones
    __device__ __forceinline__ int live(const PrefillParams& p) const {
        return Form<D>::kNT == 2 && q.q_len - tile * n.tile_tokens > 2 * p.tile_tokens ? 2 : 1;
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
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a3, b3, %3, t;\n\t}"
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
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [a2], b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [a3], b3, %3, t;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on this CTA's barrier and on the other's at the same address (`other` bytes on in the cluster's shared memory) once all MMAs issued so far
// have completed.
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t other) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b32 r;\n\tadd.u32 r, %0, %1;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [r];\n\t}" ::"r"(ptx::mapa_shared(ptx::smem_u32(bar), 0)), "r"(other) : "memory");
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

__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two values times the sigmoids of their BF16 gates, 1 / (1 + 2^(-log2(e) gate)).  2^x and 1 / x come from the same unit, four values a clock and scheduler; one
// reciprocal of (1 + u) (1 + v) for both is 1 us faster for a prompt's chunk (98.4 and 99.5) but fails for gates below -43.6 and carries a NaN over, and told
// apart by a branch it is not faster (100.3, and 19.0 instead of 18.2 for 149 tokens).
__device__ __forceinline__ uint32_t gated(float x, float y, uint32_t gate) {
    const float c = -1.4426950408889634f;
    return pack_bf16(x * reciprocal(1.0f + ex2(__uint_as_float(gate << 16) * c)), y * reciprocal(1.0f + ex2(__uint_as_float(gate & 0xFFFF0000u) * c)));
}
// 16 rows and 32 columns: register 4 i + 2 h + e of a lane is row lane / 4 + 8 h, column 8 i + 2 (lane % 4) + e.
__device__ __forceinline__ void tmem_ld16x32(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : NVFP4_R8(r, 0), NVFP4_R8(r, 8)
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {        // of all loads so far, r's among them
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 ::"memory");
}
// Among four lanes: word k of lane c becomes word c of lane k.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? w[i] : w[i + 1], 1);
        if (odd) w[i] = x; else w[i + 1] = x;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t x = __shfl_xor_sync(0xffffffffu, high ? w[i] : w[i + 2], 2);
        if (high) w[i] = x; else w[i + 2] = x;
    }
}

template <int D>
__global__ void __launch_bounds__(Form<D>::kThreads, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                     const __grid_constant__ PrefillParams p) {
    using F = Form<D>;
    extern __shared__ __align__(1024) unsigned char smem[];      // the swizzle's pattern repeats every 1024 bytes
    unsigned char* s_q = smem;
    unsigned char* ring = smem + F::kNT * F::kQTile;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + F::kSlots * F::kSlotBytes);            // [slots] the leader's: both halves are there
    uint64_t* empty = full + F::kSlots;              // [slots] each CTA its own, by commit
    uint64_t* q_full = empty + F::kSlots;            // the leader's
    uint64_t* q_empty = q_full + 1;                  // each CTA its own
    uint64_t* s_full = q_empty + 1;                  // [2] each its own: scores are there
    uint64_t* p_ready = s_full + 2;                  // [2] the leader's: weights are there, results scaled to them
    uint64_t* s_free = p_ready + 2;                  // [2] each its own: the weights are multiplied
    uint64_t* o_free = s_free + 2;                   // [2] the leader's: an item's results are read, tile by tile
    uint64_t* drain = o_free + 2;                    // [2] each its own: the issuers' last MMAs
    uint64_t* tail = drain + 2;                      // each its own: values that are zeroed in part before they count
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(tail + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    volatile unsigned int* s_ok = s_tmem + 2;        // [kOkRing] boxes of a unit whose page is one
    long long* prefix = reinterpret_cast<long long*>(s_tmem + 2 + F::kOkRing);          // [warps] in front, then the run's first place
    Cursor<D>* found = reinterpret_cast<Cursor<D>*>(prefix + F::kThreads / 32 + 2);
    float* s_x = reinterpret_cast<float*>(found + 1);                                   // [2 in turn][group][row]: what the two groups tell each other
    static_assert((2 * F::kSlots + 13) * 8 + 8 + F::kOkRing * 4 + (F::kThreads / 32 + 2) * 8 + sizeof(Cursor<D>) + 4 * kTile * 4 <= F::kControl, "control block");

    const AttentionArgs& a = p.a;
    const Batch& b = a.b;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)ptx::cluster_ctarank(), id = blockIdx.x >> 1;
    if (tid == 0) {
        for (int i = 0; i < F::kSlots; ++i) { ptx::mbar_init(&full[i], 2); ptx::mbar_init(&empty[i], 1); }
        ptx::mbar_init(q_full, 1);
        ptx::mbar_init(q_empty, 1);
        ptx::mbar_init(tail, 1);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_ready[i], 16);
            ptx::mbar_init(&s_free[i], 1);
            ptx::mbar_init(&o_free[i], 16);
            ptx::mbar_init(&drain[i], 1);
        }
        *s_abort = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmq);
        ptx::prefetch_tensormap(&tmk);
        ptx::prefetch_tensormap(&tmv);
    }
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // ---- this pair's run
    const int run = (b.sequences + F::kThreads - 1) / F::kThreads;
    const int s0 = min(tid * run, b.sequences), s1 = min(s0 + run, b.sequences);
    long long mine = 0;
    for (int s = s0; s < s1; ++s) {
        const Sequence q = sequence(b, s);
        const LongItems n = Cursor<D>::items(p, q);
        mine += long_places(q, n, n.tiles) * n.heads;
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
    for (int w = 0; w < F::kThreads / 32; ++w) {
        if (w < warp) before += prefix[w];
        cost += prefix[w];
    }
    upto += before;
    const int pairs = cost == 0 ? 0 : blocks_of(cost, gridDim.x >> 1, p.min_cost);
    if (tid == 0 && rank == 0) p.split[id].count = 0;
    if (id >= pairs) return;                         // both CTAs of a pair
    const long long c0 = run_begin(cost, pairs, id), c1 = run_begin(cost, pairs, id + 1);
    if (upto - mine <= c0 && c0 < upto) {            // exactly one thread
        long long left = c0 - (upto - mine);
        int s = s0;
        for (; run > 1; ++s) {                       // one sequence a thread: it is this one
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
    if (warp == 0) {                                 // the tiles, by cutting the range into 32 pieces at a time
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
        const int per = long_chunks(long_limit(x.q, x.n, lo)) + x.n.extra;
        x.head = (int)((left - at) / per);
        x.at = c0 - (left - at) + (long long)x.head * per;
        x.set_item(c0, c1);
        __syncwarp();
        if (lane == 0) *found = x;
    }
    __syncwarp();
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    umma::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();                             // both CTAs' barriers exist before anyone arrives on the other's
    umma::tc_fence_after();
    const uint32_t tmem = *s_tmem;
    Cursor<D> at = *found;
    bool more = true;

    if (warp == 0) {
        // ------------------------------------------------------------------ producer
        int slot = 0;
        unsigned int unit = 0, tails = 0, tail_ok = 0;
        int tail_slot = -1, tail_left = 0;
        uint32_t phase = 0, q_phase = 0;
        const int boxes = kLongChunk / p.box_rows, mine = boxes / 2;                     // of a unit; of its keys in this CTA
        const uint32_t full0 = ptx::mapa_shared(ptx::smem_u32(full), 0), q_full0 = ptx::mapa_shared(ptx::smem_u32(q_full), 0);
        // page and slot of the box that is this lane's, in a unit
        auto look_up = [&](int chunk, int& page, int& place) {
            const int tok = chunk * kLongChunk + lane * p.box_rows;
            page = -1;
            place = 0;
            if (lane < boxes && tok < at.limit) {
                const int entry = divide(tok, b.div);
                place = tok - entry * b.page_size;
                page = b.table[(long long)at.s * b.table_stride + entry];
                if ((unsigned)page >= (unsigned)b.num_pages) {
                    *b.places = kStatusPlace;
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
        // This CTA's part in a fill of the leader's: what it expects for both, or the other CTA's word that its loads are on their way.
        auto announce = [&](unsigned int bytes) {
            if (lane == 0) {
                if (rank == 0) ptx::mbar_arrive_expect_tx(&full[slot], bytes);
                else ptx::mbar_arrive_cluster(full0 + slot * 8);
            }
            __syncwarp();
        };
        // lane = (64 elements, box of tokens)
        auto keys = [&](int page, int place) {
            const unsigned int ok = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) s_ok[unit % F::kOkRing] = ok;
            ++unit;
            const int box = lane % mine, part = lane / mine;
            const int pg = __shfl_sync(0xffffffffu, page, rank * mine + box), pl = __shfl_sync(0xffffffffu, place, rank * mine + box);
            if (!ptx::mbar_wait(&empty[slot], phase ^ 1u, s_abort, b.status, 0xA20u)) return;
            announce((unsigned)(__popc(ok) * p.box_rows * D * 2));
            if (part < D / 64 && pg >= 0)
                ptx::tma_load_5d_pair(ring + slot * F::kSlotBytes + part * (F::kKeys * 128) + box * p.box_rows * 128, &tmk, full0 + slot * 8, 0, pl, part, at.head, pg);
            next_slot();
        };
        auto values = [&](int chunk, int page, int place) {
            constexpr int kAcross = F::kVCols / 64;
            const unsigned int ok = __ballot_sync(0xffffffffu, page >= 0);
            const int part = lane % kAcross, box = lane / kAcross;
            const int pg = __shfl_sync(0xffffffffu, page, box % boxes), pl = __shfl_sync(0xffffffffu, place, box % boxes);
            const int cols = (D == 64 ? 0 : rank * kAcross) + part;
            unsigned char* to = ring + slot * F::kSlotBytes;
            if (!ptx::mbar_wait(&empty[slot], phase ^ 1u, s_abort, b.status, 0xA21u)) return;
            const bool go = box < boxes && pg >= 0;
            const int left = at.limit - chunk * kLongChunk;                              // tokens that are seen
            if (left >= kLongChunk && ok == (1u << boxes) - 1u) {
                announce((unsigned)(2 * boxes * p.box_rows * F::kVCols * 2));
                if (go) ptx::tma_load_5d_pair(to + part * (kLongChunk * 128) + box * p.box_rows * 128, &tmv, full0 + slot * 8, 0, pl, cols, at.head, pg);
            } else {
                // values of keys that no row sees: whatever lies there, a weight of zero times it is to be zero
                if (lane == 0) ptx::mbar_arrive_expect_tx(tail, (unsigned)(__popc(ok) * p.box_rows * F::kVCols * 2));
                __syncwarp();
                if (go) ptx::tma_load_5d(to + part * (kLongChunk * 128) + box * p.box_rows * 128, &tmv, tail, 0, pl, cols, at.head, pg);
                tail_slot = slot;
                tail_left = left;
                tail_ok = ok;
            }
            next_slot();
        };
        // The values that a tail load brought are zeroed in part and then count; the next item's queries may be asked for in between.
        auto finish_tail = [&]() {
            if (tail_slot < 0) return;
            const bool there = ptx::mbar_wait(tail, tails & 1u, s_abort, b.status, 0xA24u);
            ++tails;
            unsigned char* to = ring + tail_slot * F::kSlotBytes;
            constexpr int kPer = F::kVCols / 8;                                          // 16-byte pieces of a token
            for (int i = lane; there && i < kLongChunk * kPer; i += 32) {
                const int tok = i / kPer, piece = i % kPer;
                if (tok >= tail_left || !(tail_ok >> (tok >> p.box_log) & 1u))
                    *reinterpret_cast<uint4*>(to + (piece >> 3) * (kLongChunk * 128) + tok * 128 + (piece & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster_release(full0 + tail_slot * 8);
            tail_slot = -1;
        };
        while (more) {
            int page, place, page_before = -1, place_before = 0;
            look_up(at.chunk, page, place);
            const bool go = ptx::mbar_wait(q_empty, q_phase ^ 1u, s_abort, b.status, 0xA22u);
            q_phase ^= 1u;
            const int live = at.live(p);
            if (ptx::elect_one() && go) {
                if (rank == 0) ptx::mbar_arrive_expect_tx(q_full, (unsigned)(2 * live * (D / 64) * p.tile_tokens * a.group * 128));
                for (int t = 0; t < live; ++t)
                    for (int c = 0; c < D / 64; ++c)
                        ptx::tma_load_3d_pair(s_q + t * F::kQTile + c * (kTile * 128), &tmq, q_full0, c * 64, at.head * a.group,
                                              at.q.q0 + at.tile * at.n.tile_tokens + (2 * t + rank) * p.tile_tokens);
            }
            __syncwarp();
            finish_tail();
            for (int j = at.chunk; j < at.to; ++j) {
                int page_next = -1, place_next = 0;
                if (j + 1 < at.to) look_up(j + 1, page_next, place_next);
                keys(page, place);
                if (F::kNT == 2) values(j, page, place);
                else if (j > at.chunk) values(j - 1, page_before, place_before);
                if (F::kNT == 1 || j + 1 < at.to) finish_tail();         // pages out of bounds in the middle; the last unit's waits for the next queries
                page_before = page;
                place_before = place;
                page = page_next;
                place = place_next;
            }
            if (F::kNT == 1) values(at.to - 1, page_before, place_before);
            more = at.next_item(p, c0, c1);
        }
        finish_tail();
        // nothing of this CTA's may still be on its way when it ends: every slot's last fill has been multiplied
        for (int i = 0; i < F::kSlots; ++i) {
            ptx::mbar_wait(&empty[slot], phase ^ 1u, s_abort, b.status, 0xA23u);
            next_slot();
        }
    } else if (warp <= 2) {
        // ------------------------------------------------------------------ MMA issuers (leader); the other CTA's two warps go to the end at once
        const bool is_s = warp == 1;
        const uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(2 * kTile >> 4) << 24 | (is_s ? (uint32_t)(kLongChunk >> 3) << 17 : 1u << 16 | (uint32_t)(F::kOCols >> 3) << 17);
        const uint32_t other = ptx::mapa_shared(ptx::smem_u32(full), 1) - ptx::mapa_shared(ptx::smem_u32(full), 0);
        // items and units so far; second tiles without rows do not count
        uint32_t item = 0, items_of[2] = {0, 0}, units_of[2] = {0, 0};
        unsigned int used = 0;                       // halves of units (keys or values) that the ring has seen
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int where) {
            ok = ptx::mbar_wait(bar, parity, s_abort, b.status, where) && ok;
            __syncwarp();
            ok = __all_sync(0xffffffffu, ok);
            umma::tc_fence_after();
        };
        while (rank == 0 && more) {
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
                        if (u >= F::kBufs) wait(&s_free[sb], u / F::kBufs - 1 & 1u, 0xA38u);           // the buffer's weights before are multiplied
                    } else {
                        if (j == 0 && items_of[t] > 0) wait(&o_free[t], items_of[t] - 1 & 1u, 0xA34u);
                        wait(&p_ready[sb], u / F::kBufs & 1u, 0xA35u);
                    }
                    const int s = (int)(half % F::kSlots);
                    if (t == 0) wait(&full[s], half / F::kSlots & 1u, is_s ? 0xA30u : 0xA31u);
                    if (!ok) continue;
                    const uint32_t from = ptx::smem_u32(ring + s * F::kSlotBytes);
                    if (is_s) {
#pragma unroll
                        for (int e = 0; e < D / 64; ++e)
                            mma4_ss(tmem + sb * 128, umma::umma_desc_sw128(ptx::smem_u32(s_q + t * F::kQTile + e * (kTile * 128))),
                                    umma::umma_desc_sw128(from + e * (F::kKeys * 128)), idesc, e > 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < kLongChunk / 64; ++e)
                            mma4_ts(tmem + F::kOCol + t * 128, tmem + sb * 128 + e * 32, values_desc(from, kLongChunk) + e * 512, idesc, j > 0 || e > 0);
                    }
                    if (release) commit(&empty[s], other);
                    commit(is_s ? &s_full[sb] : &s_free[sb], other);
                }
            }
            if (is_s && ok) commit(q_empty, other);
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
        if (rank == 0) commit(&drain[!is_s], other);
    } else {
        // ------------------------------------------------------------------ softmax: thread = row and 64 of the scores, half of the result
        const int g = (warp - 3) >> 2, quarter = warp & 3, row = quarter * 32 + lane, s_col = g * 64;
        constexpr int kCols = D / 2;                 // of the result
        const int col0 = g * kCols;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t p_ready0 = ptx::mapa_shared(ptx::smem_u32(p_ready), 0), o_free0 = ptx::mapa_shared(ptx::smem_u32(o_free), 0);
        const unsigned int all = (1u << (kLongChunk / p.box_rows)) - 1u;
        const int in_tile = row / a.group;           // token of the tile
        // rows lane / 4 + 8 r of the warp's 32: token of the tile and head of the group
        int out_tok[4], out_head[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            out_tok[r] = (quarter * 32 + r * 8 + (lane >> 2)) / a.group;
            out_head[r] = quarter * 32 + r * 8 + (lane >> 2) - out_tok[r] * a.group;
        }
        uint32_t units_of[2] = {0, 0};               // of a tile so far
        uint32_t units_seen = 0;                     // for the page masks
        int turn = 0;
        // the other group's value of this row; two places in turn, so that one barrier is enough
        auto exchange = [&](float x) {
            float* to = s_x + turn * (2 * kTile) + row;
            turn ^= 1;
            to[g * kTile] = x;
            ptx::named_barrier_sync(1 + quarter, 64);
            return to[(1 - g) * kTile];
        };
        while (more) {
            const int n = at.to - at.chunk, live = at.live(p);
            const bool whole = at.chunk == 0 && at.to == at.chunks;
            const int first = whole ? id : block_of(cost, pairs, at.at + at.n.extra);
            if (!whole && first == id && rank == 0 && tid == 96)
                p.split[id] = LongSplit{block_of(cost, pairs, at.at + at.n.extra + at.chunks - 1) - first + 1, at.q.q0, at.q.q_len, at.tile, at.head, {0, 0, 0}};
            int see[F::kNT];
            bool there[F::kNT];
            float m[F::kNT], l[F::kNT];
#pragma unroll
            for (int t = 0; t < F::kNT; ++t) {
                const int tok = at.tile * at.n.tile_tokens + (2 * t + rank) * p.tile_tokens + in_tile;
                there[t] = in_tile < p.tile_tokens && tok < at.q.q_len;
                see[t] = there[t] ? sees(at.q, tok) : 0x7fffffff;
                m[t] = -INFINITY;
                l[t] = 0.0f;
            }
            for (int j = 0; j < n; ++j) {
                const int key0 = (at.chunk + j) * kLongChunk;
#pragma unroll
                for (int t = 0; t < F::kNT; ++t) {
                    if (t >= live) continue;
                    const uint32_t u = units_of[t] + j;
                    const int sb = F::kNT == 1 ? u % F::kBufs : t;
                    const uint32_t s_addr = lanes + sb * 128, o_addr = lanes + F::kOCol + t * 128 + col0;
                    ptx::mbar_wait(&s_full[sb], u / F::kBufs & 1u, s_abort, b.status, 0xA40u);
                    __syncwarp();
                    umma::tc_fence_after();
                    const unsigned int ok = s_ok[(units_seen + j) % F::kOkRing];
                    uint32_t s[64];
                    tmem_ld32(s_addr + s_col, s);
                    tmem_ld32(s_addr + s_col + 32, s + 32);
                    tmem_wait_ld32(s);
                    tmem_wait_ld32(s + 32);
                    const int seen = see[t] - key0 - s_col;      // of this thread's columns those in front of this one
                    if (__any_sync(0xffffffffu, there[t] && seen < 64) || ok != all) {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            unsigned int keep = seen >= q * 32 + 32 ? 0xffffffffu : seen <= q * 32 ? 0u : (1u << (seen - q * 32)) - 1u;
                            if (!(ok >> ((s_col + q * 32) >> p.box_log) & 1u)) keep &= 0xffff0000u;
                            if (!(ok >> ((s_col + q * 32 + 16) >> p.box_log) & 1u)) keep &= 0x0000ffffu;
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(keep >> i & 1u)) s[q * 32 + i] = 0xff800000u;
                        }
                    }
                    float top[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) top[i] = fmaxf(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
#pragma unroll
                    for (int i = 8; i < 64; i += 2) top[i / 2 & 3] = max3(top[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                    float now = max3(fmaxf(top[0], top[1]), top[2], top[3]) * p.scale_log2;
                    now = fmaxf(now, exchange(now));             // behind it both groups hold their scores, which the weights may overwrite
                    if (__any_sync(0xffffffffu, there[t] && now > m[t] + 8.0f)) {
                        const float next = fmaxf(m[t], now), back = next == m[t] ? 1.0f : ex2(m[t] - next);
                        m[t] = next;
                        l[t] *= back;
                        if (j > 0) {                 // the results so far follow, once the product before is through
                            ptx::mbar_wait(&s_free[F::kNT == 1 ? (u - 1) % F::kBufs : t], (u - 1) / F::kBufs & 1u, s_abort, b.status, 0xA42u);
                            __syncwarp();
                            umma::tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < kCols; c += 32) {
                                uint32_t x[32];
                                tmem_ld32(o_addr + c, x);
                                tmem_wait_ld32(x);
#pragma unroll
                                for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * back);
                                tmem_st32(o_addr + c, x);
                            }
                        }
                    }
                    const float base = m[t] == -INFINITY ? 0.0f : m[t];
                    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2), base2 = pair(-base, -base);
                    uint64_t sum[2] = {0, 0};        // two sums each
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float x, y;
                        unpair(fma2(pair_bits(s[2 * i], s[2 * i + 1]), scale2, base2), x, y);
                        x = ex2(x);
                        y = ex2(y);
                        sum[i & 1] = add2(sum[i & 1], pair(x, y));
                        w[i] = pack_bf16(x, y);
                    }
                    tmem_st32(s_addr + s_col / 2, w);
                    {
                        float x, y;
                        unpair(add2(sum[0], sum[1]), x, y);
                        l[t] += x + y;
                    }
                    tmem_wait_st();
                    umma::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_cluster(p_ready0 + sb * 8);
                }
            }
            units_seen += n;
            // ---- the item, or this pair's part of it
#pragma unroll
            for (int t = 0; t < F::kNT; ++t) {
                if (t >= live) continue;
                units_of[t] += n;
                const uint32_t u = units_of[t] - 1, o_addr = lanes + F::kOCol + t * 128 + col0;
                // A thread's row is 32 lines away from its neighbours': for the way out four lanes take a row instead (row lane / 4 and further ones 8,
                // 16, 24 on), 16 bytes each, with the row's factor from the thread whose row it is.
                const int span = at.tile * at.n.tile_tokens + (2 * t + rank) * p.tile_tokens;          // the tile's first token
                auto goes = [&](int r) { return whole && out_tok[r] < p.tile_tokens && span + out_tok[r] < at.q.q_len; };
                auto place_of = [&](int r, long long stride, long long head_stride) {
                    return (long long)(at.q.q0 + span + out_tok[r]) * stride + (long long)(at.head * a.group + out_head[r]) * head_stride + col0 + (lane & 3) * 8;
                };
                uint4 gates[kCols / 32][2];          // of two of the four rows, asked for while the last product runs
                auto ask_gates = [&](int h) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const bool go = a.gate && goes(2 * h + r);
                        const uint16_t* from = a.gate + (go ? place_of(2 * h + r, a.g_stride, a.g_head) : 0);
#pragma unroll
                        for (int c = 0; c < kCols / 32; ++c) gates[c][r] = go ? *reinterpret_cast<const uint4*>(from + c * 32) : make_uint4(0u, 0u, 0u, 0u);
                    }
                };
                ask_gates(0);
                const float mine_l = l[t], other_l = exchange(mine_l), sum = g == 0 ? mine_l + other_l : other_l + mine_l;
                ptx::mbar_wait(&s_free[F::kNT == 1 ? u % F::kBufs : t], u / F::kBufs & 1u, s_abort, b.status, 0xA43u);
                __syncwarp();
                umma::tc_fence_after();
                float* part = p.parts + (size_t)(part_slot(first, id) * 2 + rank) * kMaxPartFloats;
                if (whole) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float inv_r[2] = {__shfl_sync(0xffffffffu, inv, h * 16 + (lane >> 2)), __shfl_sync(0xffffffffu, inv, h * 16 + 8 + (lane >> 2))};
                        uint32_t x[kCols / 32][16];
#pragma unroll
                        for (int c = 0; c < kCols / 32; ++c) tmem_ld16x32(o_addr + ((uint32_t)(h * 16) << 16) + c * 32, x[c]);
#pragma unroll
                        for (int c = 0; c < kCols / 32; ++c) tmem_wait_ld16(x[c]);
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const bool go = goes(2 * h + r);
                            uint16_t* out = a.out + (go ? place_of(2 * h + r, a.o_stride, a.o_head) : 0);
#pragma unroll
                            for (int c = 0; c < kCols / 32; ++c) {
                                uint32_t gate[4] = {gates[c][r].x, gates[c][r].y, gates[c][r].z, gates[c][r].w}, w[4];
                                if (a.gate) transpose4(gate);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    // rows without a key: zero, whatever the product holds
                                    const float y = inv_r[r] == 0.0f ? 0.0f : __uint_as_float(x[c][4 * i + 2 * r]) * inv_r[r];
                                    const float z = inv_r[r] == 0.0f ? 0.0f : __uint_as_float(x[c][4 * i + 2 * r + 1]) * inv_r[r];
                                    w[i] = a.gate ? gated(y, z, gate[i]) : pack_bf16(y, z);
                                }
                                transpose4(w);
                                if (go) *reinterpret_cast<uint4*>(out + c * 32) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                        if (h == 0) ask_gates(1);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kCols; c += 32) {
                        uint32_t x[32];
                        tmem_ld32(o_addr + c, x);
                        tmem_wait_ld32(x);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            __stcg(reinterpret_cast<float4*>(part) + (t * (D / 4) + (col0 + c) / 4 + i) * kTile + row,
                                   make_float4(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1]), __uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3])));
                    }
                }
                if (!whole && g == 0) {
                    float* ml = part + F::kNT * kTile * D + t * (2 * kTile);
                    __stcg(ml + row, m[t]);
                    __stcg(ml + kTile + row, sum);
                }
                umma::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_cluster(o_free0 + t * 8);
            }
            more = at.next_item(p, c0, c1);
        }
    }
    __syncwarp();
    umma::tc_fence_before();
    __syncthreads();
    // The issuers' last MMAs, in both CTAs.  A wait's limit is about a second and a run may take longer, so no wait spans the run: behind the barrier the
    // softmax warps have read the last item's results, and what is left is the arrival.
    if (warp == 1 || warp == 2) ptx::mbar_wait(&drain[warp == 2], 0, s_abort, b.status, 0xA3Fu);
    __syncthreads();
    if (*s_abort) {                                  // a wait ran out: nobody issues any more; give what is in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
    ptx::cluster_sync();                             // neither CTA leaves, or frees its tensor memory, while the other may still reach it
    if (warp == 2) {
        umma::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Adds the parts of split items in the order of their pairs.  A warp takes 32 rows and 8 columns of an item, eight parts under way at once.
constexpr int kJoinThreads = 256, kJoinAhead = 8;
template <int D>
__global__ void __launch_bounds__(kJoinThreads)
paged_prefill_join_kernel(const __grid_constant__ PrefillParams p, int pairs) {
    using F = Form<D>;
    constexpr int kRowGroups = 2 * F::kNT * 4, kPieces = kRowGroups * (D / 8);           // warps of an item
    __shared__ LongSplit s_item[kMaxBlocks];
    __shared__ int s_first[kMaxBlocks], s_count[kJoinThreads / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    static_assert(kMaxBlocks == kJoinThreads, "a thread looks at a pair");
    LongSplit mine{};
    if (tid < pairs) {
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
        const int first = s_first[work / kPieces], piece = work % kPieces, group = piece / (D / 8), c0 = piece % (D / 8) * 8;
        const int tile = group >> 2, row = (group & 3) * 32 + lane, in_tile = row / p.a.group;         // tile = 2 t + rank
        const int tok = it.tile * (p.tile_tokens * F::kNT * 2) + tile * p.tile_tokens + in_tile;
        const bool there = in_tile < p.tile_tokens && tok < it.q_len;
        if (!__any_sync(0xffffffffu, there)) continue;
        const AttentionArgs& a = p.a;
        const long long tq = it.q0 + tok, hd = it.head * a.group + row - in_tile * a.group;
        const uint4 gate = a.gate && there ? *reinterpret_cast<const uint4*>(a.gate + tq * a.g_stride + hd * a.g_head + c0) : make_uint4(0u, 0u, 0u, 0u);
        float top = -INFINITY, den = 0.0f;
        float x[8] = {};
        for (int i0 = 0; i0 < it.count; i0 += kJoinAhead) {
            float4 y[kJoinAhead][2];
            float m[kJoinAhead], l[kJoinAhead];
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                const bool is = i0 + j < it.count;
                const float* part = p.parts + (size_t)(part_slot(first, first + i0 + j) * 2 + (tile & 1)) * kMaxPartFloats;
                const float* ml = part + F::kNT * kTile * D + (tile >> 1) * (2 * kTile) + row;
                const float4* from = reinterpret_cast<const float4*>(part) + ((tile >> 1) * (D / 4) + c0 / 4) * kTile + row;
                y[j][0] = ptx::ldcg_if(is, from);
                y[j][1] = ptx::ldcg_if(is, from + kTile);
                m[j] = ptx::ldcg_if(is, ml, -INFINITY);
                l[j] = ptx::ldcg_if(is, ml + kTile, 0.0f);
            }
            float now = top;
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) now = fmaxf(now, m[j]);
            const float back = top == -INFINITY ? 0.0f : ex2(top - now);
            top = now;
            den *= back;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= back;
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                const float w = m[j] == -INFINITY ? 0.0f : ex2(m[j] - now);         // a sum of NaN stays one
                den += w * l[j];
                x[0] = fmaf(y[j][0].x, w, x[0]); x[1] = fmaf(y[j][0].y, w, x[1]); x[2] = fmaf(y[j][0].z, w, x[2]); x[3] = fmaf(y[j][0].w, w, x[3]);
                x[4] = fmaf(y[j][1].x, w, x[4]); x[5] = fmaf(y[j][1].y, w, x[5]); x[6] = fmaf(y[j][1].z, w, x[6]); x[7] = fmaf(y[j][1].w, w, x[7]);
            }
        }
        if (!there) continue;
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        const uint32_t g[4] = {gate.x, gate.y, gate.z, gate.w};
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float u = x[2 * e] * inv, v = x[2 * e + 1] * inv;
            w[e] = a.gate ? gated(u, v, g[e]) : pack_bf16(u, v);
        }
        *reinterpret_cast<uint4*>(a.out + tq * a.o_stride + hd * a.o_head + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <class... P, class... A>
cudaError_t launch_behind(void (*kernel)(P...), int grid, int threads, int smem, int cluster, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int pairs_of(const nvfp4_device_info& dev) {
    const int pairs = dev.sm_count / 2 < kMaxBlocks ? dev.sm_count / 2 : kMaxBlocks;
    return dev.max_pairs > 0 && dev.max_pairs < pairs ? dev.max_pairs : pairs;
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
bool launch(PrefillParams& p, const nvfp4_device_info& dev, cudaStream_t s, cudaError_t* e) {
    CUtensorMap maps[3];
    p.tile_tokens = kTile / p.a.group;
    p.box_rows = common_divisor(p.a.b.page_size, Form<D>::kKeys);
    p.box_log = p.box_rows == 64 ? 6 : p.box_rows == 32 ? 5 : 4;
    if (!make_q_map(&maps[0], p.a, p.tile_tokens) || !make_cache_map(&maps[1], p.a.b, p.a.b.k, p.box_rows, 1) || !make_cache_map(&maps[2], p.a.b, p.a.b.v, p.box_rows, 1))
        return false;
    const int pairs = pairs_of(dev);
    *e = launch_behind(paged_prefill_kernel<D>, 2 * pairs, Form<D>::kThreads, Form<D>::kSmem, 2, s, maps[0], maps[1], maps[2], p);
    if (*e == cudaSuccess) *e = launch_behind(paged_prefill_join_kernel<D>, 4 * pairs, kJoinThreads, 0, 1, s, p, pairs);
    return true;
}

}  // namespace

size_t paged_prefill_scratch_bytes(int sm_count) {
    return kSplitBytes + (size_t)(sm_count / 2 < kMaxBlocks ? sm_count / 2 : kMaxBlocks) * 4 * kMaxPartFloats * sizeof(float);
}

cudaError_t configure_paged_prefill() {
    cudaError_t e = configure_large_smem(paged_prefill_kernel<64>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_prefill_kernel<128>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_prefill_kernel<256>, Form<256>::kSmem);
    return e;
}

// Whole boxes of 16 tokens, a group of heads that fits a tile, a maximum that grows with the products (and a scale that is none of the numbers
// taken for zero, which would make NaN of a hidden score).
bool paged_prefill_supported(const paged::AttentionArgs& a) { return a.b.page_size % 16 == 0 && a.group <= kTile && a.scale >= 1e-30f; }

bool launch_paged_prefill(const paged::AttentionArgs& a, int above_rows, const nvfp4_device_info& dev, void* scratch, int* launches, cudaStream_t s, cudaError_t* e) {
    PrefillParams p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.above_rows = above_rows;
    p.min_cost = long_cost(a.b.head_dim) + 1;
    p.split = static_cast<LongSplit*>(scratch);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + kSplitBytes);
    const bool done = a.b.head_dim == 64 ? launch<64>(p, dev, s, e) : a.b.head_dim == 128 ? launch<128>(p, dev, s, e) : launch<256>(p, dev, s, e);
    if (done) *launches = 2;
    return done;
}

}  // namespace nvfp4
