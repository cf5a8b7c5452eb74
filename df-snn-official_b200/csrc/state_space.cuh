// state_space.cuh -- shared device helpers of the state-space kernels (selective scan, short
// causal convolution, and their single-token forms).
#pragma once
#include <atomic>
#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/dfsnn_b200.h"

namespace dfsnn {

constexpr float kLog2e = 1.44269504088896340736f;

// element type <-> float (one rounding to nearest on the way out)
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename IO> __device__ __forceinline__ IO from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// 2^x by the hardware approximation (2 ulp; results below the normal range become 0)
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / x by the hardware approximation (1 ulp); x = inf gives 0
__device__ __forceinline__ float rcp_ftz(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float sigmoid_f(float x) {
    return rcp_ftz(1.0f + exp2_approx(-kLog2e * x));
}

__device__ __forceinline__ float2 sigmoid_f(float2 x) {
    const float2 y = __fmul2_rn(x, make_float2(-kLog2e, -kLog2e));
    const float2 d = __fadd2_rn(make_float2(exp2_approx(y.x), exp2_approx(y.y)), make_float2(1.0f, 1.0f));
    return make_float2(rcp_ftz(d.x), rcp_ftz(d.y));
}

// log(1 + e^x) = max(x, 0) + log(1 + v), v = e^-|x|, which loses nothing at either end.  The
// logarithm by its series log(1 + v) = 2 atanh(s), s = v / (2 + v) <= 1/3: an odd polynomial in s,
// fitted at Chebyshev nodes in s^2 (0.07 units of 2^-24 off), in a third of log1pf's instructions.
__device__ __forceinline__ float2 softplus_f(float2 x) {
    auto two = [](float c) { return make_float2(c, c); };
    const float2 v = make_float2(exp2_approx(-kLog2e * fabsf(x.x)), exp2_approx(-kLog2e * fabsf(x.y)));
    const float2 d = __fadd2_rn(v, two(2.0f));
    const float2 s = __fmul2_rn(v, make_float2(rcp_ftz(d.x), rcp_ftz(d.y))), w = __fmul2_rn(s, s);
    float2 q = __ffma2_rn(w, two(0.2817465727f), two(0.2796141883f));
    q = __ffma2_rn(w, q, two(0.4002485372f));
    q = __ffma2_rn(w, q, two(0.6666631594f));
    q = __ffma2_rn(w, q, two(2.0f));
    return __ffma2_rn(s, q, make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}
__device__ __forceinline__ float softplus_f(float x) { return softplus_f(make_float2(x, x)).x; }

// 2^x for |x| < 2^-4, two at a time: 1 + x p(x), fitted at Chebyshev nodes (0.64 units of 2^-24
// off).  Near 1 the hardware's approximation is off by up to 2^-22, and a state that decays by
// little each step adds those errors up over all the steps that it remembers.
constexpr float kExp2Near = 0.0625f;
__device__ __forceinline__ float2 exp2_near1(float2 x) {
    const float2 one = make_float2(1.0f, 1.0f);
    float2 q = __ffma2_rn(x, make_float2(0.0555093173f, 0.0555093173f), make_float2(0.2402546865f, 0.2402546865f));
    q = __ffma2_rn(x, q, make_float2(0.693147178f, 0.693147178f));
    return __ffma2_rn(x, q, one);
}

// A log2 e, as the scans keep it.  An infinite product becomes the largest number: a step behind the
// end has d = 0 and leaves the state alone (0 times infinity would not), and any other d still gives
// the decay 0 (or infinity).
__device__ __forceinline__ float log2_rate(float a) {
    a *= kLog2e;
    return isinf(a) ? copysignf(FLT_MAX, a) : a;
}

// 2^(2 x) h + end, where 2^(2 x) is the decay over a whole part of a sequence.  Step by step a growing
// state stays finite as long as it is; the power alone need not (nor is 0 times its infinity 0), so it
// is taken as two factors.  (A NaN in x is one in `end` too.)
__device__ __forceinline__ float carry_over(float x, float h, float end) {
    const float f = exp2_approx(fminf(x, 127.5f));              // any state overflows by 2^255
    return fmaf(f * h, f, end);
}

// sequence length of row b: lengths[b] clamped to [0, T]; T without lengths
__device__ __forceinline__ int seq_length(const void* lengths, int wide, long long b, int T) {
    if (lengths == nullptr) return T;
    const long long n = wide ? static_cast<const long long*>(lengths)[b]
                             : static_cast<const int*>(lengths)[b];
    return n < 0 ? 0 : (n > T ? T : (int)n);
}

// Sums each of CNT values over W lanes (lane = any + STRIDE * w, w = 0 .. W-1) by exchanging
// halves: a stage sends the half of the values that the partner keeps, so W lanes need
// CNT * (1 - 1/W) shuffles instead of CNT * log2 W.  Afterwards lane w holds, in
// v[0 .. max(1, CNT / W) - 1], the sums of the values first(w) + i.
template <int CNT, int W, int STRIDE>
struct LaneSums {
    static constexpr int kHeld = CNT >= W ? CNT / W : 1;
    static __device__ __forceinline__ int first(int w) { return CNT >= W ? w * (CNT / W) : w / (W / CNT); }
    // whether lane w is the one that stores (lanes share a sum when there are more lanes than values)
    static __device__ __forceinline__ bool stores(int w) { return CNT >= W || w % (W >= CNT ? W / CNT : 1) == 0; }
    static __device__ __forceinline__ void run(float (&v)[CNT], int w) {
        int cnt = CNT;
#pragma unroll
        for (int m = W / 2; m >= 1; m >>= 1) {
            if (cnt > 1) {
                const int half = cnt / 2;
                const bool up = (w & m) != 0;
#pragma unroll
                for (int i = 0; i < CNT / 2; ++i) {
                    if (i < half) {
                        const float send = up ? v[i] : v[i + half];
                        const float keep = up ? v[i + half] : v[i];
                        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m * STRIDE);
                    }
                }
                cnt = half;
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * STRIDE);
            }
        }
    }
};

// Slot of row b of a step call: its index; kIdle for a negative one, kBad behind the last slot.
// taken_before: whether an earlier row has the same slot (two rows of one call cannot both advance
// it, so the later one is refused).  It is found out while the state is on its way: reading a slot
// harms nobody.  All threads of the block call it together.
constexpr long long kIdle = -1, kBad = -2;
__device__ __forceinline__ long long index_at(const void* index, int wide, long long b) {
    return wide ? static_cast<const long long*>(index)[b]
                : (long long)static_cast<const int*>(index)[b];
}
__device__ __forceinline__ long long step_slot(const void* index, int wide, long long b, long long slots) {
    if (index == nullptr) return b;
    const long long slot = index_at(index, wide, b);
    return slot < 0 ? kIdle : slot >= slots ? kBad : slot;
}
__device__ __forceinline__ bool taken_before(const void* index, int wide, long long b, long long slot) {
    if (index == nullptr) return false;
    bool taken = false;
    for (long long r = threadIdx.x; r < b; r += blockDim.x) taken |= index_at(index, wide, r) == slot;
    return __syncthreads_or(taken);
}

// Lets Kernel use `bytes` of dynamic shared memory on the current device: the driver is asked once
// for each device.
template <auto Kernel>
inline cudaError_t allow_shared(size_t bytes) {
    static std::atomic<unsigned long long> done{0};
    if (bytes <= 48 * 1024) return cudaSuccess;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

}  // namespace dfsnn
