// New tokens into the paged cache: norms of queries and keys for each head, rotation by the position, and the writes of keys and
// values to their places, in one pass (the reference's fused qk-norm-rope and KV-write kernels, src/engine/light_ops.cu).
//
// Every value is read once and written once, and the bound should be that.  With a thread for eight neighbours, partners exchanged by shuffles and addresses
// formed for every head of every token 6534 tokens of 28 heads of 256 took 61-79 us.  Now a head is spread over head_dim / 8 lanes; a lane of the part that
// turns holds four elements and their partners i + rot_dim / 2, and goes through four tokens with the same head: 46 us, 0.62 of the copy rate, with 67 % of
// the issue slots used and DRAM at 36 %: neither is the bound, but a block begins with its chain of look-ups and a barrier, and 1634 blocks, four an SM, are 2.8
// rounds of them.  One token of one sequence takes 2.6 us from a graph, 5.5 to 6.5 called, which is the host's.  A norm is a reduction over the head's
// lanes.  The angles are the same for all heads of a token and computed once, in shared memory, while the loads are under way.
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

// The sequence of row t, by a whole warp: the last s with cu_q[s] <= t, the range cut into 32 pieces at a time.
__device__ __forceinline__ bool find_row(const Batch& b, int t, int& seq, int& pos) {
    if (!b.cu_q) {
        seq = t;
        return t < b.sequences && row_position(b, t, t, t + 1, t, pos);
    }
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = b.sequences;                     // lo <= s < hi
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, s = lo + lane * step;
        const unsigned int below = __ballot_sync(0xffffffffu, s < hi && b.cu_q[s] <= t);
        const int k = below ? 31 - __clz(below) : 0;
        hi = min(lo + (k + 1) * step, hi);
        lo = lo + k * step;
    }
    seq = lo;
    return row_position(b, lo, b.cu_q[lo], b.cu_q[lo + 1], t, pos);
}

// One block per TOKENS tokens and run of `per` heads: head x of a token's q_heads + 2 kv_heads (queries, keys, values).  A head's lanes keep it for
// UNROLL tokens at a time.  The first values are asked for at once; which sequence, length and page a token belongs to, a chain of three loads, and its
// angles are a warp's work for each token beside them.
template <int D, int TOKENS, int UNROLL>
__global__ void __launch_bounds__(kThreads)
kv_append_kernel(AppendArgs a, int per) {
    constexpr int kLanes = D / 8, kHeads = kThreads / kLanes;      // lanes per head, heads per step of the block
    static_assert(TOKENS <= kThreads / 32, "a warp looks a token up");
    __shared__ float4 s_turn[TOKENS][D / 4];          // cos and sin of two pairs each
    __shared__ long long s_at[TOKENS];                // place in the cache; -1: none; -2: the row is left out
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid % kLanes, t0 = blockIdx.x * TOKENS;
    const Batch& b = a.b;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();                              // rows, lengths and table may come from the kernel in front
    const int h0 = blockIdx.y * per, end = min(a.q_heads + 2 * b.kv_heads, h0 + per), tokens = min(TOKENS, b.tokens - t0);
    // this lane's elements: four and their partners where the head turns, eight in a row behind that
    const int half = a.rot_dim / 2;
    const bool turns = lane * 8 < a.rot_dim;
    const int e0 = turns ? lane * 4 : lane * 8, e1 = turns ? half + lane * 4 : lane * 8 + 4;
    int h = h0 + tid / kLanes;
    const uint16_t* from = nullptr;
    long long stride = 0;
    auto begin_head = [&]() {
        if (h < a.q_heads) { from = a.q + (long long)h * a.q_head; stride = a.q_stride; }
        else if (h < a.q_heads + b.kv_heads) { from = a.k + (long long)(h - a.q_heads) * a.k_head; stride = a.k_stride; }
        else { from = a.v + (long long)(h - a.q_heads - b.kv_heads) * a.v_head; stride = a.v_stride; }
        from += (long long)t0 * stride;
    };
    uint2 x[UNROLL][2];
    auto ask = [&](int tk) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const bool go = h < end && tk + u < tokens;
            const uint16_t* at = from + (tk + u) * stride;
            x[u][0] = go ? *reinterpret_cast<const uint2*>(at + e0) : make_uint2(0u, 0u);
            x[u][1] = go ? *reinterpret_cast<const uint2*>(at + e1) : make_uint2(0u, 0u);
        }
    };
    begin_head();
    ask(0);
    // cu_q ascends: its ends tell whether rows outside [0, tokens] are left out
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == kThreads - 1 && b.cu_q && (b.cu_q[0] < 0 || b.cu_q[b.sequences] > b.tokens)) *b.places = kStatusPlace;
    if (warp < tokens) {
        int seq, pos = 0;
        const bool there = find_row(b, t0 + warp, seq, pos);
        const int p = a.positions ? a.positions[t0 + warp] : pos;
        long long at = there ? -1 : -2;
        if (there && pos < b.max_kv) at = place(b, seq, pos);
        if ((tid & 31) == 0) {
            s_at[warp] = at;
            if (at == -1) *b.places = kStatusPlace;
        }
        for (int i = tid & 31; i < half; i += 32) {
            double angle = (double)p * (double)a.inv_freq[i];
            angle = fma(-rint(angle * (1.0 / kTwoPi)), kTwoPi, angle);
            float sn, cs;
            sincosf((float)angle, &sn, &cs);
            reinterpret_cast<float2*>(s_turn[warp])[i] = make_float2(cs, sn);
        }
    }
    __syncthreads();
    for (int base = h0; base < end; base += kHeads) {
        if (base != h0) {
            h = base + tid / kLanes;
            begin_head();
            ask(0);
        }
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + b.kv_heads;
        const uint16_t* weight = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
        float w[8];                                   // 1 + weight
        if (weight && h < end) {
            const uint2 w0 = *reinterpret_cast<const uint2*>(weight + e0), w1 = *reinterpret_cast<const uint2*>(weight + e1);
            unpack8(make_uint4(w0.x, w0.y, w1.x, w1.y), w);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] += 1.0f;
        }
        // the head's place in a token's row of q_out or of the cache
        uint16_t* const to = is_q ? a.q_out + (long long)h * a.o_head : is_v ? b.v + (long long)(h - a.q_heads - b.kv_heads) * b.head_stride : b.k + (long long)(h - a.q_heads) * b.head_stride;
        for (int tk = 0; tk < tokens; tk += UNROLL) {
            if (tk) ask(tk);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                uint4 out = make_uint4(x[u][0].x, x[u][0].y, x[u][1].x, x[u][1].y);
                const bool go = h < end && tk + u < tokens;
                if (!is_v) {
                    float v[8];
                    unpack8(out, v);
                    if (weight) {
                        float ss = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
                        // the lanes of a head take the branches together
                        const unsigned int group = kLanes == 32 ? 0xffffffffu : ((1u << (kLanes & 31)) - 1u) << ((tid & 31) / kLanes * kLanes);
#pragma unroll
                        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
                        const float inv = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
                    }
                    if (turns && go) {
                        const float4 c0 = s_turn[tk + u][lane * 2], c1 = s_turn[tk + u][lane * 2 + 1];
                        const float cs[4] = {c0.x, c0.z, c1.x, c1.z}, sn[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float lo = v[i], hi = v[i + 4];
                            v[i] = lo * cs[i] - hi * sn[i];
                            v[i + 4] = hi * cs[i] + lo * sn[i];
                        }
                    }
                    out = pack8(v);
                }
                if (!go) continue;
                const long long at = s_at[tk + u];
                if (is_q ? at == -2 : at < 0) continue;
                uint16_t* row = to + (is_q ? (long long)(t0 + tk + u) * a.o_stride : at);
                *reinterpret_cast<uint2*>(row + e0) = make_uint2(out.x, out.y);
                *reinterpret_cast<uint2*>(row + e1) = make_uint2(out.z, out.w);
            }
        }
    }
}

template <int D>
cudaError_t launch(const AppendArgs& a, const nvfp4_device_info& dev, cudaStream_t s) {
    constexpr int kHeads = kThreads / (D / 8), kTokens = 4;
    const int total = a.q_heads + 2 * a.b.kv_heads, steps = (total + kHeads - 1) / kHeads;
    // Few tokens: a block for each step of a token's heads.  Many: a block for four tokens, whose look-ups run side by side (6534 tokens of 28 heads of 256:
    // 46.8 us; eight tokens, four or two at a time 52.9 and 59.7, two 47.5).
    const bool spread = (long long)a.b.tokens * steps <= 8LL * dev.sm_count;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(spread ? a.b.tokens : (a.b.tokens + kTokens - 1) / kTokens, spread ? steps : 1);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return spread ? cudaLaunchKernelEx(&cfg, kv_append_kernel<D, 1, 1>, a, kHeads) : cudaLaunchKernelEx(&cfg, kv_append_kernel<D, kTokens, kTokens>, a, total);
}

}  // namespace

cudaError_t launch_kv_append(const paged::AppendArgs& a, const nvfp4_device_info& dev, int* launches, cudaStream_t s) {
    *launches = 1;
    return a.b.head_dim == 64 ? launch<64>(a, dev, s) : a.b.head_dim == 128 ? launch<128>(a, dev, s) : launch<256>(a, dev, s);
}

}  // namespace nvfp4
