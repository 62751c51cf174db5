// New tokens into the paged cache: norms of queries and keys for each head, rotation by the position, and the writes of keys and
// values to their places, in one pass (the reference's fused qk-norm-rope and KV-write kernels, src/engine/light_ops.cu).
//
// Every value is read once and written once; the arithmetic (an FMA per value for the norm, a product with cos and sin for the
// rotated part) is nothing beside it.  A head is spread over head_dim / 8 lanes of a warp, 16 bytes a lane, so a norm is a reduction
// over those lanes and the partner i + rot_dim / 2 of element i lies rot_dim / 16 lanes away, a shuffle.  The angles are the same
// for all heads of a token: the block's threads compute them once, in shared memory, while the loads are under way.
// position * inv_freq is formed and reduced to [-pi, pi] in FP64 (a float of 2^17 has steps of 1/64: the angle itself would be lost),
// the reduced angle is rounded to FP32 (1.2e-7) for sincosf.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "nvfp4_internal.h"
#include "paged_plan.h"
#include "ptx.cuh"

namespace nvfp4 {
namespace {

using namespace paged;

constexpr int kThreads = 256;
constexpr double kTwoPi = 6.283185307179586476925286766559;

__device__ __forceinline__ void unpack8(const uint4& x, float (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// One block per token and run of `per` heads: head x of the token's q_heads + 2 kv_heads (queries, keys, values).
template <int D, int UNROLL>
__global__ void __launch_bounds__(kThreads)
kv_append_kernel(AppendArgs a, int per) {
    constexpr int kLanes = D / 8, kHeads = kThreads / kLanes;      // lanes per head, heads per step of the block
    __shared__ float2 s_turn[D / 2];
    const int tid = threadIdx.x, t = blockIdx.x, lane = tid % kLanes;
    const Batch& b = a.b;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();                              // rows, lengths and table may come from the kernel in front
    int seq, pos;
    if (!find_row(b, t, seq, pos)) return;            // the same in the whole block
    const int total = a.q_heads + 2 * b.kv_heads, end = min(total, (int)(blockIdx.y + 1) * per);
    const int half = a.rot_dim / 2;
    if (tid < half) {
        const int p = a.positions ? a.positions[t] : pos;
        double angle = (double)p * (double)a.inv_freq[tid];
        angle = fma(-rint(angle * (1.0 / kTwoPi)), kTwoPi, angle);
        float sn, cs;
        sincosf((float)angle, &sn, &cs);
        s_turn[tid] = make_float2(cs, sn);
    }
    long long at = -1;
    if (pos < b.max_kv) at = place(b, seq, pos);
    if (at < 0 && tid == 0 && blockIdx.y == 0) atomicCAS(b.status, 0u, kStatusPlace);
    __syncthreads();
    const int reach = half / 8;                       // lanes between an element and its partner
    for (int base = blockIdx.y * per + tid / kLanes; base - tid / kLanes < end; base += kHeads * UNROLL) {
        uint4 x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int head = base + u * kHeads;
            const uint16_t* from = nullptr;
            if (head < end) {
                if (head < a.q_heads) from = a.q + (long long)t * a.q_stride + (long long)head * a.q_head;
                else if (head < a.q_heads + b.kv_heads) from = a.k + (long long)t * a.k_stride + (long long)(head - a.q_heads) * a.k_head;
                else from = a.v + (long long)t * a.v_stride + (long long)(head - a.q_heads - b.kv_heads) * a.v_head;
            }
            x[u] = from ? *reinterpret_cast<const uint4*>(from + lane * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int head = base + u * kHeads;
            const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + b.kv_heads;
            const uint16_t* weight = is_q ? a.q_norm : a.k_norm;
            uint4 out = x[u];
            if (__any_sync(0xffffffffu, !is_v)) {
                float v[8];
                unpack8(x[u], v);
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (weight) {
                    const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
                    float w[8];
                    unpack8(*reinterpret_cast<const uint4*>(weight + lane * 8), w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * (1.0f + w[i]);
                }
                // lanes 0 .. reach-1 hold the first halves of the pairs, the next `reach` lanes the second ones
                const bool first = lane < reach, turns = lane < 2 * reach;
                const int partner = (tid & 31) + (first ? reach : turns ? -reach : 0);
                const float2* turn = s_turn + (first ? lane : turns ? lane - reach : 0) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float other = __shfl_sync(0xffffffffu, v[i], partner);
                    if (turns) {
                        const float2 cs = turn[i];
                        v[i] = first ? v[i] * cs.x - other * cs.y : v[i] * cs.x + other * cs.y;
                    }
                }
                if (!is_v) out = pack8(v);
            }
            if (head >= end) continue;
            uint16_t* to = nullptr;
            if (is_q) to = a.q_out + (long long)t * a.o_stride + (long long)head * a.o_head;
            else if (at >= 0) to = (is_v ? b.v + (long long)(head - a.q_heads - b.kv_heads) * b.head_stride : b.k + (long long)(head - a.q_heads) * b.head_stride) + at;
            if (to) *reinterpret_cast<uint4*>(to + lane * 8) = out;
        }
    }
}

template <int D>
cudaError_t launch(const AppendArgs& a, const nvfp4_device_info& dev, cudaStream_t s) {
    constexpr int kHeads = kThreads / (D / 8);
    const int total = a.q_heads + 2 * a.b.kv_heads, steps = (total + kHeads - 1) / kHeads;
    // Few tokens: a block for each step of a token's heads.  Many: one block per token, which shares its angles and keeps
    // more loads in flight.
    const bool spread = (long long)a.b.tokens * steps <= 8LL * dev.sm_count;
    const int per = spread ? kHeads : steps * kHeads;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.b.tokens, spread ? steps : 1);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return spread ? cudaLaunchKernelEx(&cfg, kv_append_kernel<D, 1>, a, per) : cudaLaunchKernelEx(&cfg, kv_append_kernel<D, 2>, a, per);
}

}  // namespace

cudaError_t launch_kv_append(const paged::AppendArgs& a, const nvfp4_device_info& dev, int* launches, cudaStream_t s) {
    *launches = 1;
    return a.b.head_dim == 64 ? launch<64>(a, dev, s) : a.b.head_dim == 128 ? launch<128>(a, dev, s) : launch<256>(a, dev, s);
}

}  // namespace nvfp4
