// dropout.cu -- y = keep ? T(x * 1 / (1 - p)) : 0 with the mask of
// tk_philox.cuh, recomputed wherever it is needed and never stored; the
// backward pass is the same call on the gradient.
//
// The generator bounds it: ten Philox rounds of four elements are 18 wide
// multiplies, which issue at a quarter of the rate of an add (75 % of the
// multiplier's cycles busy at 36 % of HBM's, fp16); the loads are in flight
// meanwhile.
#include <cuda_fp16.h>

#include "tk_internal.h"
#include "tk_philox.cuh"

namespace tk {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // octets of elements in flight per thread

template <typename T>
struct Octet {  // 8 elements as one (fp16) or two (fp32) 16-byte vectors
    static constexpr int N = sizeof(T) / 2;
    uint4 v[N];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < N; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, v[i]);
    }
};

// Scales the octet's values whose word reaches the threshold, zeroes the rest.
__device__ __forceinline__ uint32_t scale2(uint32_t pair, float s, uint32_t w0, uint32_t w1, uint32_t threshold) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    const __half2 h = __floats2half2_rn(w0 >= threshold ? f.x * s : 0.0f, w1 >= threshold ? f.y * s : 0.0f);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void apply(Octet<__half>& o, float s, const uint32_t (&a)[4], const uint32_t (&b)[4], uint32_t threshold) {
    o.v[0].x = scale2(o.v[0].x, s, a[0], a[1], threshold);
    o.v[0].y = scale2(o.v[0].y, s, a[2], a[3], threshold);
    o.v[0].z = scale2(o.v[0].z, s, b[0], b[1], threshold);
    o.v[0].w = scale2(o.v[0].w, s, b[2], b[3], threshold);
}

__device__ __forceinline__ uint32_t scale1(uint32_t bits, float s, uint32_t w, uint32_t threshold) {
    return w >= threshold ? __float_as_uint(__uint_as_float(bits) * s) : 0u;
}

__device__ __forceinline__ void apply(Octet<float>& o, float s, const uint32_t (&a)[4], const uint32_t (&b)[4], uint32_t threshold) {
    o.v[0] = make_uint4(scale1(o.v[0].x, s, a[0], threshold), scale1(o.v[0].y, s, a[1], threshold),
                        scale1(o.v[0].z, s, a[2], threshold), scale1(o.v[0].w, s, a[3], threshold));
    o.v[1] = make_uint4(scale1(o.v[1].x, s, b[0], threshold), scale1(o.v[1].y, s, b[1], threshold),
                        scale1(o.v[1].z, s, b[2], threshold), scale1(o.v[1].w, s, b[3], threshold));
}

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }

// n elements, 16-byte aligned pointers: octets by vectors, the last n % 8
// elements one thread each.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const T* x, T* y, int64_t n,
                                                           const DropoutParams d) {
    const int64_t octets = n / 8;
    // a block's 1024 Philox blocks share the counter's high word
    static_assert((2 * kThreads * kUnroll & (2 * kThreads * kUnroll - 1)) == 0, "a power of two");
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads * kUnroll, base = first + threadIdx.x;
    const uint32_t hi = static_cast<uint32_t>(2 * first >> 32);
    Octet<T> o[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = base + u * kThreads;
        if (i < octets) o[u].load(x + 8 * i);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = base + u * kThreads;
        if (i < octets) {
            uint32_t a[4], b[4];
            const uint32_t lo = static_cast<uint32_t>(2 * first) + 2 * (threadIdx.x + u * kThreads);
            philox4x32_10(lo, hi, d.offset, d.seed, a);
            philox4x32_10(lo + 1, hi, d.offset, d.seed, b);
            apply(o[u], d.scale, a, b, d.threshold);
            o[u].store(y + 8 * i);
        }
    }
    const int64_t tail = octets * 8 + threadIdx.x;
    if (blockIdx.x == gridDim.x - 1 && tail < n) {
        uint32_t w[4];
        philox4x32_10(static_cast<uint32_t>(tail >> 2), static_cast<uint32_t>(tail >> 34), d.offset, d.seed, w);
        const uint32_t lane = static_cast<uint32_t>(tail) & 3u;
        const uint32_t v = lane == 0 ? w[0] : lane == 1 ? w[1] : lane == 2 ? w[2] : w[3];
        from_f(v >= d.threshold ? to_f(x[tail]) * d.scale : 0.0f, y[tail]);
    }
}

// Pointers off a 16-byte boundary: one block of four elements per thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_any_kernel(const T* x, T* y, int64_t n,
                                                               const DropoutParams d) {
    const int64_t b = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (4 * b >= n) return;
    uint32_t w[4];
    philox4x32_10(static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32), d.offset, d.seed, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t i = 4 * b + j;
        if (i < n) from_f(w[j] >= d.threshold ? to_f(x[i]) * d.scale : 0.0f, y[i]);
    }
}

template <typename T>
int dropout_launch(const void* x, void* y, int64_t n, const DropoutParams& d, cudaStream_t s) {
    const T* xp = static_cast<const T*>(x);
    T* yp = static_cast<T*>(y);
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0) {
        const int64_t blocks = std::max<int64_t>(1, ceil_div(n / 8, kThreads * kUnroll));
        TK_CHECK_ARG(blocks <= 0x7FFFFFFF, "tk_dropout: too many elements");
        dropout_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(xp, yp, n, d);
    } else {
        const int64_t blocks = ceil_div(ceil_div(n, 4), kThreads);
        TK_CHECK_ARG(blocks <= 0x7FFFFFFF, "tk_dropout: too many elements");
        dropout_any_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(xp, yp, n, d);
    }
    return launch_status("dropout");
}

}  // namespace
}  // namespace tk

extern "C" int tk_dropout(tk_dtype_t dtype, const void* x, void* y, int64_t n, double p, uint64_t seed,
                          uint64_t offset, void* stream) {
    TK_CHECK_ARG(dtype == TK_DTYPE_F16 || dtype == TK_DTYPE_F32, "tk_dropout: bad dtype %d",
                 static_cast<int>(dtype));
    TK_CHECK_ARG(n >= 0, "tk_dropout: n must not be negative");
    TK_CHECK_ARG(p >= 0.0 && p <= 1.0, "tk_dropout: p must be in [0, 1], got %g", p);
    if (n == 0) return TK_OK;
    TK_CHECK_ARG(x != nullptr && y != nullptr, "tk_dropout: NULL pointer");
    const tk::DropoutParams d = tk::dropout_params(p, seed, offset);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d.none_kept) {
        TK_CHECK_ARG(n <= INT64_MAX / 4, "tk_dropout: too many elements");
        TK_CUDA_TRY(cudaMemsetAsync(y, 0, static_cast<size_t>(n) * tk::dtype_size(dtype), s));
        return TK_OK;
    }
    return dtype == TK_DTYPE_F16 ? tk::dropout_launch<__half>(x, y, n, d, s)
                                 : tk::dropout_launch<float>(x, y, n, d, s);
}
