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

namespace nvfp4 {
namespace {

using namespace paged;

constexpr int kGroup = 16;           // tokens of a unit and warp

template <int D>
struct Form {
    static constexpr int kWarps = D == 256 ? 4 : 8;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kChunk = kWarps * kGroup;                     // tokens of a unit
    static constexpr int kStageBytes = 2 * kGroup * D * 2;             // a warp's keys and values of one unit
    static constexpr int kStages = 192 * 1024 / (kWarps * kStageBytes);
    static constexpr int kTiles = D / 8;                               // 8-column tiles of the result
    static constexpr int kRounds = D == 64 ? 1 : 2;                    // rounds in which the warps' results are added
    static constexpr int kRoundTiles = kTiles / kRounds, kWarpTiles = kRoundTiles / kWarps;
    static constexpr int kMergeBytes = kWarps * kRoundTiles * 512;
    static constexpr int kSmem = kWarps * kStages * kStageBytes + kMergeBytes + kWarps * kRows * 8 + kWarps * kStages * 4 + 64;
};
static_assert(Form<256>::kSmem <= 232448 && Form<128>::kSmem <= 232448 && Form<64>::kSmem <= 232448, "shared memory");
static_assert(Form<256>::kStages == 3 && Form<128>::kStages == 3 && Form<64>::kStages == 6, "ring");

// Scratch of the handle: one counter per block, then two part slots per block: results [16 rows, D] in the layout of the registers,
// maxima and sums.
constexpr int kPartFloats = kRows * 256 + 2 * kRows;
constexpr size_t kCounterBytes = 4096;

struct DecodeParams {
    AttentionArgs a;
    float scale_log2;
    int min_units;           // units that a block takes at least, where there are fewer than blocks times this
    int most_rows;           // sequences with more rows (new tokens x group) belong to another kernel
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

// A walk over consecutive units.
template <int D>
struct Cursor {
    static __device__ __forceinline__ Items items(const DecodeParams& p, const Sequence& q) {
        return items_of(p.a.b, q, p.a.group, Form<D>::kChunk, p.most_rows);
    }
    Sequence q;
    Items n;
    int s, item, chunk;
    __device__ __forceinline__ void enter(const DecodeParams& p, int seq) {
        s = seq;
        q = sequence(p.a.b, s);
        n = items(p, q);
    }
    // To the next unit; the caller knows that there is one.
    __device__ __forceinline__ void advance(const DecodeParams& p) {
        if (++chunk < n.chunks) return;
        chunk = 0;
        if (++item < n.items) return;
        item = 0;
        do enter(p, s + 1); while (n.items == 0 && s + 1 < p.a.b.sequences);
    }
    // Tokens that some row of the item's tile sees.
    __device__ __forceinline__ int limit(const DecodeParams& p) const {
        return sees(q, (min((item % n.tiles + 1) * kRows, q.q_len * p.a.group) - 1) / p.a.group);
    }
};

template <int D>
__global__ void __launch_bounds__(Form<D>::kThreads, 1)
paged_decode_kernel(const __grid_constant__ DecodeParams p) {
    using F = Form<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    const AttentionArgs& a = p.a;
    const Batch& b = a.b;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* ring = smem + warp * F::kStages * F::kStageBytes;
    float4* merge = reinterpret_cast<float4*>(smem + F::kWarps * F::kStages * F::kStageBytes);
    float* s_max = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(merge) + F::kMergeBytes);   // [warp][row]
    float* s_sum = s_max + F::kWarps * kRows;
    unsigned int* s_ok = reinterpret_cast<unsigned int*>(s_sum + F::kWarps * kRows);                     // [warp][stage]: tokens whose page is one
    int* s_word = reinterpret_cast<int*>(s_ok + F::kWarps * F::kStages);

    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // ---- this block's units: prefix sums over the sequences, a run of them per thread
    long long* prefix = reinterpret_cast<long long*>(merge);
    const int run = (b.sequences + F::kThreads - 1) / F::kThreads;
    const int s0 = min(tid * run, b.sequences), s1 = min(s0 + run, b.sequences);
    long long mine = 0;
    for (int s = s0; s < s1; ++s) {
        const Items n = Cursor<D>::items(p, sequence(b, s));
        mine += (long long)n.items * n.chunks;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) prefix[warp] = upto;
    __syncthreads();
    long long units = 0, before = 0;
#pragma unroll
    for (int w = 0; w < F::kWarps; ++w) {
        if (w < warp) before += prefix[w];
        units += prefix[w];
    }
    upto += before;
    if (units == 0) return;
    const int blocks = blocks_of(units, gridDim.x, p.min_units);
    if ((int)blockIdx.x >= blocks) return;
    const long long u0 = run_begin(units, blocks, blockIdx.x), u1 = run_begin(units, blocks, blockIdx.x + 1);
    __syncthreads();
    if (upto - mine <= u0 && u0 < upto) {            // exactly one thread
        long long left = u0 - (upto - mine);
        int s = s0;
        for (;; ++s) {
            const Items n = Cursor<D>::items(p, sequence(b, s));
            const long long here = (long long)n.items * n.chunks;
            if (left < here) break;
            left -= here;
        }
        s_word[0] = s;
        *reinterpret_cast<long long*>(s_word + 2) = left;
    }
    __syncthreads();
    Cursor<D> at;
    at.enter(p, s_word[0]);
    {
        const long long off = *reinterpret_cast<const long long*>(s_word + 2);
        at.item = (int)(off / at.n.chunks);
        at.chunk = (int)(off % at.n.chunks);
    }
    Cursor<D> ld = at;                               // where the loads are
    long long ld_left = u1 - u0;

    // ---- loads: the page number of this lane's token (lanes 0..15) is asked for one unit ahead
    int page_ahead = -1, slot_ahead = 0;
    bool seen_ahead = false;
    auto look_up = [&]() {
        const int tok = ld.chunk * F::kChunk + warp * kGroup + (lane & 15);
        seen_ahead = ld_left > 0 && tok < ld.limit(p);
        page_ahead = -1;
        if (seen_ahead) {
            const int entry = divide(tok, b.div);
            slot_ahead = tok - entry * b.page_size;
            page_ahead = b.table[(long long)ld.s * b.table_stride + entry];
        }
    };
    auto load = [&](int stage) {
        if (ld_left > 0) {
            const bool there = seen_ahead && (unsigned)page_ahead < (unsigned)b.num_pages;
            if (seen_ahead && !there) atomicCAS(b.status, 0u, kStatusPlace);
            const unsigned int ok = __ballot_sync(0xffffffffu, there) & 0xFFFFu;
            if (lane == 0) s_ok[warp * F::kStages + stage] = ok;
            const long long head = (long long)(ld.item / ld.n.tiles) * b.head_stride;
            const long long off = there ? (long long)page_ahead * b.page_stride + (long long)slot_ahead * b.token_stride + head : 0;
            if (__any_sync(0xffffffffu, seen_ahead)) {
                constexpr int kPer = D / 8;                  // 16-byte pieces of a token
                unsigned char* ks = ring + stage * F::kStageBytes;
                unsigned char* vs = ks + kGroup * D * 2;
#pragma unroll
                for (int i = 0; i < kGroup * kPer / 32; ++i) {
                    const int tok = (i * 32 + lane) / kPer, piece = (i * 32 + lane) % kPer;
                    const long long o = __shfl_sync(0xffffffffu, off, tok);
                    const uint32_t bytes = (ok >> tok) & 1u ? 16u : 0u;
                    const int to = tok * D * 2 + ((piece ^ (tok & 7)) << 4);
                    ptx::cp_async_16(ks + to, b.k + o + piece * 8, bytes);
                    ptx::cp_async_16(vs + to, b.v + o + piece * 8, bytes);
                }
            }
            if (--ld_left > 0) ld.advance(p);
            look_up();
        }
        cp_async_commit();
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < F::kStages - 1; ++i) load(i);

    // ---- units
    uint32_t qf[D / 16][4];
    float o[F::kTiles][4];
    float m0 = 0, m1 = 0, l0 = 0, l1 = 0;            // of rows lane / 4 and lane / 4 + 8
    int see0 = 0, see1 = 0, limit = 0, head = 0;
    bool fresh = true;
    int stage = 0, next = F::kStages - 1;
    const int row = lane >> 2;
    for (long long u = u0; u < u1; ++u) {
        if (fresh) {                                 // a new item: its rows of q
            fresh = false;
            head = at.item / at.n.tiles;
            limit = at.limit(p);
            const int r0 = (at.item % at.n.tiles) * kRows + row, rows = at.q.q_len * a.group;
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
            for (int k = 0; k < D / 16; ++k) {
                const int c = k * 16 + (lane & 3) * 2;
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
        cp_async_wait<F::kStages - 2>();
        __syncwarp();
        load(next);
        next = next + 1 == F::kStages ? 0 : next + 1;
        const int tok0 = at.chunk * F::kChunk + warp * kGroup;
        if (tok0 < limit) {
            const uint32_t ks = ptx::smem_u32(ring + stage * F::kStageBytes), vs = ks + kGroup * D * 2;
            const unsigned int ok = s_ok[warp * F::kStages + stage];
            float sc[2][2][4] = {};                  // [even / odd step][8 tokens][element]
            {
                const int tok = ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t r[4];
                    ldmatrix_x4(r, ks + tok * D * 2 + (((k * 2 + ((lane >> 3) & 1)) ^ (tok & 7)) << 4));
                    ptx::mma_bf16_16x8x16(sc[k & 1][0], qf[k], r[0], r[1]);
                    ptx::mma_bf16_16x8x16(sc[k & 1][1], qf[k], r[2], r[3]);
                }
            }
            float t[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[n][e] = (sc[0][n][e] + sc[1][n][e]) * p.scale_log2;
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
            const float u0f = m0 == -INFINITY ? 0.0f : m0, u1f = m1 == -INFINITY ? 0.0f : m1;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                t[n][0] = ex2(t[n][0] - u0f);
                t[n][1] = ex2(t[n][1] - u0f);
                t[n][2] = ex2(t[n][2] - u1f);
                t[n][3] = ex2(t[n][3] - u1f);
                l0 += t[n][0] + t[n][1];
                l1 += t[n][2] + t[n][3];
            }
            const uint32_t pf[4] = {pack_bf16(t[0][0], t[0][1]), pack_bf16(t[0][2], t[0][3]), pack_bf16(t[1][0], t[1][1]), pack_bf16(t[1][2], t[1][3])};
            const int tok = lane & 15;
#pragma unroll
            for (int c = 0; c < F::kTiles; c += 2) {
                uint32_t r[4];
                ldmatrix_x4_trans(r, vs + tok * D * 2 + (((c + (lane >> 4)) ^ (tok & 7)) << 4));
                ptx::mma_bf16_16x8x16(o[c], pf, r[0], r[1]);
                ptx::mma_bf16_16x8x16(o[c + 1], pf, r[2], r[3]);
            }
        }
        stage = stage + 1 == F::kStages ? 0 : stage + 1;
        if (at.chunk + 1 < at.n.chunks && u + 1 < u1) {
            ++at.chunk;
            continue;
        }

        // ---- the item (or this block's part of it) is through
        fresh = true;
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        __syncthreads();                             // the item before is out of the shared arrays
        if ((lane & 3) == 0) {
            s_max[warp * kRows + row] = m0;
            s_max[warp * kRows + row + 8] = m1;
            s_sum[warp * kRows + row] = l0;
            s_sum[warp * kRows + row + 8] = l1;
        }
        __syncthreads();
        float top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int w = 0; w < F::kWarps; ++w) {
            top0 = fmaxf(top0, s_max[w * kRows + row]);
            top1 = fmaxf(top1, s_max[w * kRows + row + 8]);
        }
#pragma unroll
        for (int w = 0; w < F::kWarps; ++w) {
            const float a0 = s_max[w * kRows + row], a1 = s_max[w * kRows + row + 8];
            sum0 += a0 == -INFINITY ? 0.0f : s_sum[w * kRows + row] * ex2(a0 - top0);
            sum1 += a1 == -INFINITY ? 0.0f : s_sum[w * kRows + row + 8] * ex2(a1 - top1);
        }
        const float f0 = m0 == -INFINITY ? 0.0f : ex2(m0 - top0), f1 = m1 == -INFINITY ? 0.0f : ex2(m1 - top1);

        // the item's units and the blocks that share it
        const long long item_u0 = u - at.chunk, item_u1 = item_u0 + at.n.chunks;
        const bool whole = item_u0 >= u0 && item_u1 <= u1;
        const int first = block_of(units, blocks, item_u0);
        const int count = whole ? 1 : block_of(units, blocks, item_u1 - 1) - first + 1;
        float* part = p.parts + (size_t)(blockIdx.x * 2 + (first == (int)blockIdx.x ? 1 : 0)) * kPartFloats;

        // one row pair's two columns of the result, normalised, gated, rounded once
        const int r_first = (at.item % at.n.tiles) * kRows + row, rows = at.q.q_len * a.group;
        auto write_row = [&](int r, int tile, float x, float y) {
            if (r >= rows) return;
            const int t = r / a.group, hd = head * a.group + r - t * a.group;
            const long long tq = at.q.q0 + t;
            const int c = tile * 8 + (lane & 3) * 2;
            if (a.gate) {
                const uint32_t g = *reinterpret_cast<const uint32_t*>(a.gate + tq * a.g_stride + (long long)hd * a.g_head + c);
                x /= 1.0f + __expf(-__uint_as_float(g << 16));
                y /= 1.0f + __expf(-__uint_as_float(g & 0xFFFF0000u));
            }
            *reinterpret_cast<uint32_t*>(a.out + tq * a.o_stride + (long long)hd * a.o_head + c) = pack_bf16(x, y);
        };
        const float inv0 = sum0 == 0.0f ? 0.0f : 1.0f / sum0, inv1 = sum1 == 0.0f ? 0.0f : 1.0f / sum1;
#pragma unroll
        for (int rd = 0; rd < F::kRounds; ++rd) {
            if (rd) __syncthreads();
#pragma unroll
            for (int i = 0; i < F::kRoundTiles; ++i) {
                const float(&x)[4] = o[rd * F::kRoundTiles + i];
                merge[(warp * F::kRoundTiles + i) * 32 + lane] = make_float4(x[0] * f0, x[1] * f0, x[2] * f1, x[3] * f1);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < F::kWarpTiles; ++i) {
                const int tile = i * F::kWarps + warp;
                float4 x = merge[tile * 32 + lane];
#pragma unroll
                for (int w = 1; w < F::kWarps; ++w) {
                    const float4 y = merge[(w * F::kRoundTiles + tile) * 32 + lane];
                    x.x += y.x;
                    x.y += y.y;
                    x.z += y.z;
                    x.w += y.w;
                }
                const int nt = rd * F::kRoundTiles + tile;
                if (whole) {
                    write_row(r_first, nt, x.x * inv0, x.y * inv0);
                    write_row(r_first + 8, nt, x.z * inv1, x.w * inv1);
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
            __threadfence();
            __syncthreads();
            if (tid == 0) s_word[0] = atomicAdd(&p.counters[first], 1u) == (unsigned)(count - 1);
            __syncthreads();
            if (s_word[0]) {                         // every part is there: add them in block order
                __threadfence();
                auto part_of = [&](int i) { return p.parts + (size_t)((first + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats; };
                float* weight = reinterpret_cast<float*>(merge);        // [part][row], then the rows' 1 / sum behind them
                if (warp == 0) {
                    const int r = lane & 15;
                    float top = -INFINITY, sum = 0.0f;
                    for (int i = lane >> 4; i < count; i += 2) top = fmaxf(top, __ldcg(part_of(i) + kRows * D + r));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    for (int i = lane >> 4; i < count; i += 2) {
                        const float mi = __ldcg(part_of(i) + kRows * D + r);
                        const float f = mi == -INFINITY ? 0.0f : ex2(mi - top);
                        weight[i * kRows + r] = f;
                        sum += f * __ldcg(part_of(i) + kRows * D + kRows + r);
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    if (lane < 16) weight[count * kRows + r] = sum == 0.0f ? 0.0f : 1.0f / sum;
                }
                __syncthreads();
                for (int nt = warp; nt < F::kTiles; nt += F::kWarps) {
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int i = 0; i < count; ++i) {
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(part_of(i)) + nt * 32 + lane);
                        const float w0 = weight[i * kRows + row], w1 = weight[i * kRows + row + 8];
                        x.x = fmaf(y.x, w0, x.x);
                        x.y = fmaf(y.y, w0, x.y);
                        x.z = fmaf(y.z, w1, x.z);
                        x.w = fmaf(y.w, w1, x.w);
                    }
                    const float w0 = weight[count * kRows + row], w1 = weight[count * kRows + row + 8];
                    write_row(r_first, nt, x.x * w0, x.y * w0);
                    write_row(r_first + 8, nt, x.z * w1, x.w * w1);
                }
                if (tid == 0) p.counters[first] = 0u;
            }
        }
        if (u + 1 < u1) at.advance(p);
    }
    cp_async_wait<0>();
}

template <int D>
cudaError_t launch(const DecodeParams& p, int blocks, cudaStream_t s) {
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
    return cudaLaunchKernelEx(&cfg, paged_decode_kernel<D>, p);
}

}  // namespace

size_t paged_scratch_bytes(int sm_count) { return kCounterBytes + (size_t)sm_count * 2 * kPartFloats * sizeof(float); }

cudaError_t configure_paged_decode() {
    cudaError_t e = configure_large_smem(paged_decode_kernel<64>, Form<64>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<128>, Form<128>::kSmem);
    if (e == cudaSuccess) e = configure_large_smem(paged_decode_kernel<256>, Form<256>::kSmem);
    return e;
}

cudaError_t launch_paged_decode(const paged::AttentionArgs& a, const nvfp4_device_info& dev, void* scratch, int* launches, cudaStream_t s) {
    DecodeParams p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.min_units = 1;
    p.most_rows = 0x7fffffff;
    p.counters = static_cast<unsigned int*>(scratch);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + kCounterBytes);
    const int blocks = dev.sm_count;
    *launches = 1;
    return a.b.head_dim == 64 ? launch<64>(p, blocks, s) : a.b.head_dim == 128 ? launch<128>(p, blocks, s) : launch<256>(p, blocks, s);
}

}  // namespace nvfp4
