// residual_norm.cu -- the norms behind and before a transformer block with
// the block's dropout, gate and residual scale, in one pass over the rows:
//
//   u     = post ? Norm(f) * post_weight + post_bias : f
//   d     = dropout(u)                         (mask of tk_philox.cuh)
//   x_new = a * x + gate * d
//   h     = Norm(x_new) * weight + bias
//
// Norm is (v - mean) * rstd (layer) or v * rstd with the mean square (rms).
// Arithmetic is fp32, each output is rounded once; h is computed from the
// unrounded x_new.  With n = Norm(x_new), q = Norm(f) and the gradients gx of
// x_new and gh of h, the backward pass is
//
//   t = gh * weight;   g = gx + rstd * (t - mean(t) - n * mean(t * n))
//   dx = a * g;        dgate = g * d
//   gu = gate * g * keep / (1 - p);   t' = gu * post_weight
//   df = post ? rstd' * (t' - mean(t') - q * mean(t' * q)) : gu
//   dweight = sum gh * n, dbias = sum gh, dpost_weight = sum gu * q,
//   dpost_bias = sum gu over the rows
//
// (an rms norm has no mean(t) terms).  x_new stands for x there, so neither x
// nor h is read again.
//
// HBM bounds both directions: 4 tensors forward, 6 backward (5 without a post
// norm and a gate, which need f).  A group of W warps holds a row in
// registers, 8 * NV columns per thread; a CTA runs several groups when rows
// are short, and a cluster of CTAs shares a row past 8192 (fp16) or 4096
// (fp32) columns, its sums exchanged through distributed shared memory.  Each
// thread copies its own columns of the next rows into its own shared-memory
// slots (cp.async), so loads stay in flight without registers or barriers.
// CTAs own contiguous rows; column sums stay in registers until a CTA's rows
// end, and a second kernel adds the CTAs' partial sums in a fixed order, so
// no gradient depends on timing.
#include <cuda_fp16.h>

#include <algorithm>

#include "tk_internal.h"
#include "tk_philox.cuh"
#include "tk_ptx.cuh"

namespace tk {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxCols = 32768;

struct RnParams {
    const void *x, *f, *weight, *bias, *post_weight, *post_bias, *gate;
    void *x_new, *h;
    const void *gx, *gh;  // backward: gradients of x_new and h
    void *dx, *df, *dgate;
    float4* stats;   // per row: mean and rstd of f (post), mean and rstd of x_new
    float* partial;  // backward: [4][units][cols], then the gate's [2 * units][cols]
    int64_t rows, cols, gate_period;  // row r uses gate row r / gate_period
    int units;                        // row ranges: clusters of `cluster` CTAs
    int cluster, warps, groups, stages;
    float a, eps, inv_cols;
    bool layer, drop;
    DropoutParams dropout;
};

__host__ __device__ __forceinline__ int64_t unit_begin(int64_t unit, int64_t rows, int64_t units) {
    return unit * rows / units;
}
// The unit whose range holds row r.
__device__ __forceinline__ int64_t unit_of(int64_t r, int64_t rows, int64_t units) {
    return ((r + 1) * units - 1) / rows;
}

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }

__device__ __forceinline__ void unpack8(const uint4 (&u)[1], float* o) {
    const __half2* h = reinterpret_cast<const __half2*>(&u[0]);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const float2 f = __half22float2(h[t]);
        o[2 * t] = f.x;
        o[2 * t + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack8(const uint4 (&u)[2], float* o) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        o[4 * t] = __uint_as_float(u[t].x);
        o[4 * t + 1] = __uint_as_float(u[t].y);
        o[4 * t + 2] = __uint_as_float(u[t].z);
        o[4 * t + 3] = __uint_as_float(u[t].w);
    }
}
__device__ __forceinline__ void store8(__half* p, const float* v) {
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int t = 0; t < 4; ++t) h[t] = __floats2half2_rn(v[2 * t], v[2 * t + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `pending` of this thread's copy groups are in flight.
__device__ __forceinline__ void cp_async_wait(int pending) {
    if (pending <= 0) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (pending == 1) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
        asm volatile("cp.async.wait_group 2;" ::: "memory");
    }
}

// One thread's share of a row: which columns it holds, its shared-memory
// slots, and the sums over the threads that hold the rest of the row.
//
// VEC: octets of 8 consecutive columns, 16-byte accesses (every pointer
// 16-byte aligned, cols a multiple of 8).  Otherwise single columns, one
// row's width of threads apart.
template <typename T, int NV, bool VEC>
struct Lane {
    static constexpr int E = 8 * NV;
    static constexpr int PARTS = sizeof(T) / 2;  // 16-byte vectors of an octet
    int t, lane, warp, group, gthreads, rank;
    int64_t col0;  // first column of the CTA's slice
    uint32_t ring;
    float2* red;
    int red_stride, red_n, parity;
    const RnParams& p;

    __device__ Lane(const RnParams& pr, uint8_t* smem) : p(pr) {
        gthreads = p.warps * 32;
        group = threadIdx.x / gthreads;
        t = threadIdx.x - group * gthreads;
        lane = threadIdx.x & 31;
        warp = t >> 5;
        rank = p.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
        col0 = static_cast<int64_t>(rank) * gthreads * E;
        red = reinterpret_cast<float2*>(smem);
        red_n = p.warps * p.cluster;
        red_stride = red_n * p.groups;
        parity = 0;
        ring = smem_u32(smem + 2 * sizeof(float2) * ((red_stride + 1) & ~1)) + threadIdx.x * 16;
        if (p.cluster > 1) cluster_sync_all();  // every CTA runs before its memory is written
    }
    __device__ __forceinline__ int64_t col(int e) const {
        return VEC ? col0 + (static_cast<int64_t>(e / 8) * gthreads + t) * 8 + e % 8
                   : col0 + static_cast<int64_t>(e) * gthreads + t;
    }
    __device__ __forceinline__ bool has(int e) const { return col(e) < p.cols; }

    // Begins the copy of tensor `k` (of `tensors`) of a row into `stage`.
    __device__ __forceinline__ void fetch(const void* base, int64_t row, int stage, int k, int tensors) const {
        if constexpr (VEC) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!has(8 * v)) continue;
                const T* src = static_cast<const T*>(base) + row * p.cols + col(8 * v);
                const uint32_t slot = ring + static_cast<uint32_t>(((stage * tensors + k) * NV + v) * PARTS) * blockDim.x * 16;
#pragma unroll
                for (int i = 0; i < PARTS; ++i) cp_async16(slot + i * blockDim.x * 16, reinterpret_cast<const uint4*>(src) + i);
            }
        }
    }
    __device__ __forceinline__ void row_values(const void* base, int64_t row, int stage, int k, int tensors, float (&o)[E]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                uint4 u[PARTS];
                const uint32_t slot = ring + static_cast<uint32_t>(((stage * tensors + k) * NV + v) * PARTS) * blockDim.x * 16;
#pragma unroll
                for (int i = 0; i < PARTS; ++i) {
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(u[i].x), "=r"(u[i].y), "=r"(u[i].z), "=r"(u[i].w)
                                 : "r"(slot + i * blockDim.x * 16)
                                 : "memory");
                }
                unpack8(u, &o[8 * v]);
                if (!has(8 * v)) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[8 * v + j] = 0.0f;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = has(e) ? to_f(static_cast<const T*>(base)[row * p.cols + col(e)]) : 0.0f;
        }
    }
    // This thread's columns of a [cols] vector, `absent` where it is NULL.
    __device__ __forceinline__ void vector(const void* base, float absent, float (&o)[E]) const {
        const T* b = static_cast<const T*>(base);
        if constexpr (VEC) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (b != nullptr && has(8 * v)) {
                    uint4 u[PARTS];
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(b + col(8 * v)) + i);
                    unpack8(u, &o[8 * v]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[8 * v + j] = absent;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = b != nullptr && has(e) ? to_f(b[col(e)]) : absent;
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t row, const float (&v)[E]) const {
        T* b = static_cast<T*>(base) + row * p.cols;
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (has(8 * k)) store8(b + col(8 * k), &v[8 * k]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (has(e)) b[col(e)] = from_f<T>(v[e]);
        }
    }
    // Keep bits of this thread's columns of a row (bit e).
    __device__ __forceinline__ uint32_t keep(int64_t row) const {
        uint32_t m = 0;
        if constexpr (VEC) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                m |= dropout_keep8(p.dropout, static_cast<uint64_t>(row * p.cols + col(8 * v)) / 8) << (8 * v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) m |= (dropout_keep1(p.dropout, row * p.cols + col(e)) ? 1u : 0u) << e;
        }
        return m;
    }
    // Sums of a and b over the row's threads; every thread gets the same bits.
    // One exchange buffer is read while the next sum fills the other, so one
    // barrier per sum is enough.
    __device__ __forceinline__ void row_sum(float& a, float& b) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            a += __shfl_xor_sync(0xFFFFFFFFu, a, m);
            b += __shfl_xor_sync(0xFFFFFFFFu, b, m);
        }
        if (red_n == 1) return;
        float2* buf = red + parity * red_stride + group * red_n;
        parity ^= 1;
        const int slot = rank * p.warps + warp;
        if (p.cluster == 1) {
            if (lane == 0) buf[slot] = make_float2(a, b);
            named_barrier_sync(1 + group, gthreads);
        } else {
            if (lane < p.cluster) {
                const uint32_t to = mapa_shared(smem_u32(buf + slot), lane);
                st_shared_cluster_u32(to, __float_as_uint(a));
                st_shared_cluster_u32(to + 4, __float_as_uint(b));
            }
            __syncwarp();
            cluster_sync_all();
        }
        a = 0.0f;
        b = 0.0f;
        if (red_n <= 4) {
            for (int i = 0; i < red_n; ++i) {
                a += buf[i].x;
                b += buf[i].y;
            }
        } else {
            for (int i = lane; i < red_n; i += 32) {
                a += buf[i].x;
                b += buf[i].y;
            }
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) {
                a += __shfl_xor_sync(0xFFFFFFFFu, a, m);
                b += __shfl_xor_sync(0xFFFFFFFFu, b, m);
            }
        }
    }
    // mean and rstd of v over the row (mean 0 for an rms norm); the mean
    // square is taken about the mean, as values held in registers.
    __device__ __forceinline__ void moments(const float (&v)[E], float& mean, float& rstd) {
        mean = 0.0f;
        float unused = 0.0f;
        if (p.layer) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) s += v[e];
            row_sum(s, unused);
            mean = s * p.inv_cols;
        }
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float c = v[e] - mean;
            if (has(e)) q += c * c;
        }
        unused = 0.0f;
        row_sum(q, unused);
        rstd = rsqrtf(q * p.inv_cols + p.eps);
    }
};

template <typename T, int NV, bool VEC, bool POST>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_kernel(const RnParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    using L = Lane<T, NV, VEC>;
    constexpr int E = L::E;
    L ln(p, smem);
    const int64_t unit = blockIdx.x / p.cluster;
    const int64_t end = unit_begin(unit + 1, p.rows, p.units);
    const int64_t begin = unit_begin(unit, p.rows, p.units) + ln.group;
    const int ahead = VEC ? p.stages - 1 : 0;
    if constexpr (VEC) {
        for (int i = 0; i < ahead; ++i) {
            const int64_t r = begin + static_cast<int64_t>(i) * p.groups;
            if (r < end) {
                ln.fetch(p.x, r, i, 0, 2);
                ln.fetch(p.f, r, i, 1, 2);
            }
            cp_async_commit();
        }
    }
    int stage = 0;
    for (int64_t r = begin; r < end; r += p.groups) {
        if constexpr (VEC) {
            const int64_t next = r + static_cast<int64_t>(ahead) * p.groups;
            int ns = stage + ahead;
            if (ns >= p.stages) ns -= p.stages;
            if (next < end) {
                ln.fetch(p.x, next, ns, 0, 2);
                ln.fetch(p.f, next, ns, 1, 2);
            }
            cp_async_commit();
        }
        const uint32_t keep = p.drop ? ln.keep(r) : 0u;
        if constexpr (VEC) cp_async_wait(ahead);
        float u[E], v[E];
        ln.row_values(p.f, r, stage, 1, 2, u);
        float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
        if constexpr (POST) {
            ln.moments(u, st.x, st.y);
            ln.vector(p.post_weight, 1.0f, v);
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] = (u[e] - st.x) * st.y * v[e];
            if (p.post_bias != nullptr) {
                ln.vector(p.post_bias, 0.0f, v);
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] += v[e];
            }
        }
        if (p.drop) {
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] = (keep >> e) & 1u ? u[e] * p.dropout.scale : 0.0f;
        }
        if (p.gate != nullptr) {
            ln.vector(static_cast<const T*>(p.gate) + r / p.gate_period * p.cols, 0.0f, v);
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] *= v[e];
        }
        ln.row_values(p.x, r, stage, 0, 2, v);
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = fmaf(p.a, v[e], u[e]);
        if constexpr (POST) {  // a vector's columns past the row hold its bias there
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!ln.has(e)) u[e] = 0.0f;
        }
        ln.store(p.x_new, r, u);
        ln.moments(u, st.z, st.w);
        ln.vector(p.weight, 1.0f, v);
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = (u[e] - st.z) * st.w * v[e];
        if (p.bias != nullptr) {
            ln.vector(p.bias, 0.0f, v);
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] += v[e];
        }
        ln.store(p.h, r, u);
        if (p.stats != nullptr && ln.t == 0 && ln.rank == 0) p.stats[r] = st;
        if (++stage == p.stages) stage = 0;
    }
}

// Adds `acc` over the CTA's groups and writes the CTA's columns, as fp32
// partial sums or (to_final) as the finished gradient.  Every thread of the
// CTA takes part; `buf` is the ring's memory, idle at this point.
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void flush_columns(const Lane<T, NV, VEC>& ln, float* buf, const float (&acc)[8 * NV],
                                              float* partial, T* final_row) {
    const RnParams& p = ln.p;
    const int width = ln.gthreads * 8 * NV;
    if (p.groups > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8 * NV; ++e) buf[ln.group * width + (ln.col(e) - ln.col0)] = acc[e];
        __syncthreads();
        for (int c = threadIdx.x; c < width && ln.col0 + c < p.cols; c += blockDim.x) {
            float s = 0.0f;
            for (int g = 0; g < p.groups; ++g) s += buf[g * width + c];
            if (final_row != nullptr) {
                final_row[ln.col0 + c] = from_f<T>(s);
            } else {
                partial[ln.col0 + c] = s;
            }
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int e = 0; e < 8 * NV; ++e) {
            if (!ln.has(e)) continue;
            if (final_row != nullptr) {
                final_row[ln.col(e)] = from_f<T>(acc[e]);
            } else {
                partial[ln.col(e)] = acc[e];
            }
        }
    }
}

template <typename T, int NV, bool VEC, bool POST, bool GATE>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_backward_kernel(const RnParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    using L = Lane<T, NV, VEC>;
    constexpr int E = L::E;
    constexpr bool NEED_F = POST || GATE;
    constexpr int TENSORS = NEED_F ? 4 : 3;
    L ln(p, smem);
    float* const buf = reinterpret_cast<float*>(smem + 2 * sizeof(float2) * ((ln.red_stride + 1) & ~1));
    const int64_t unit = blockIdx.x / p.cluster;
    const int64_t unit_lo = unit_begin(unit, p.rows, p.units), unit_hi = unit_begin(unit + 1, p.rows, p.units);
    const int ahead = VEC ? p.stages - 1 : 0;
    const bool gate_sums = GATE && p.gate_period > 1;  // else each row writes its own gradient
    float dw[E], db[E], dpw[POST ? E : 1], dpb[POST ? E : 1], dgt[GATE ? E : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        dw[e] = 0.0f;
        db[e] = 0.0f;
        if constexpr (POST) dpw[e] = dpb[e] = 0.0f;
    }
    auto fetch = [&](int64_t r, int stage) {
        if (p.gx != nullptr) ln.fetch(p.gx, r, stage, 0, TENSORS);
        if (p.gh != nullptr) ln.fetch(p.gh, r, stage, 1, TENSORS);
        ln.fetch(p.x_new, r, stage, 2, TENSORS);
        if constexpr (NEED_F) ln.fetch(p.f, r, stage, 3, TENSORS);
    };
    // a segment: the rows of this unit that share a gate row (all of them
    // where no sum of the gate's gradient is kept)
    int64_t seg_lo = unit_lo;
    while (seg_lo < unit_hi) {
        const int64_t gate_row = gate_sums ? seg_lo / p.gate_period : 0;
        const int64_t seg_hi = gate_sums ? min(unit_hi, (gate_row + 1) * p.gate_period) : unit_hi;
        if constexpr (GATE) {
#pragma unroll
            for (int e = 0; e < E; ++e) dgt[e] = 0.0f;
        }
        const int64_t begin = seg_lo + ln.group;
        if constexpr (VEC) {
            for (int i = 0; i < ahead; ++i) {
                const int64_t r = begin + static_cast<int64_t>(i) * p.groups;
                if (r < seg_hi) fetch(r, i);
                cp_async_commit();
            }
        }
        int stage = 0;
        for (int64_t r = begin; r < seg_hi; r += p.groups) {
            if constexpr (VEC) {
                const int64_t next = r + static_cast<int64_t>(ahead) * p.groups;
                int ns = stage + ahead;
                if (ns >= p.stages) ns -= p.stages;
                if (next < seg_hi) fetch(next, ns);
                cp_async_commit();
            }
            const float4 st = p.stats[r];
            const uint32_t keep = p.drop ? ln.keep(r) : 0u;
            if constexpr (VEC) cp_async_wait(ahead);
            float g[E], n[E], t[E];
            if (p.gh != nullptr) {
                float wv[E];
                ln.row_values(p.x_new, r, stage, 2, TENSORS, n);
                ln.row_values(p.gh, r, stage, 1, TENSORS, t);
                ln.vector(p.weight, 1.0f, wv);
                float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    n[e] = ln.has(e) ? (n[e] - st.z) * st.w : 0.0f;
                    dw[e] += t[e] * n[e];
                    db[e] += t[e];
                    t[e] *= wv[e];
                    c1 += t[e];
                    c2 += t[e] * n[e];
                }
                ln.row_sum(c1, c2);
                c1 = p.layer ? c1 * p.inv_cols : 0.0f;
                c2 *= p.inv_cols;
                if (p.gx != nullptr) {
                    ln.row_values(p.gx, r, stage, 0, TENSORS, g);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) g[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < E; ++e) g[e] += st.w * (t[e] - c1 - n[e] * c2);
            } else {
                ln.row_values(p.gx, r, stage, 0, TENSORS, g);
            }
            if (p.dx != nullptr) {
#pragma unroll
                for (int e = 0; e < E; ++e) t[e] = p.a * g[e];
                ln.store(p.dx, r, t);
            }
            if constexpr (NEED_F) {  // n: q = Norm(f) with a post norm, else f
                ln.row_values(p.f, r, stage, 3, TENSORS, n);
                if constexpr (POST) {
#pragma unroll
                    for (int e = 0; e < E; ++e) n[e] = ln.has(e) ? (n[e] - st.x) * st.y : 0.0f;
                }
            }
            if constexpr (GATE) {
                float u[E];
                if constexpr (POST) {
                    ln.vector(p.post_weight, 1.0f, u);
#pragma unroll
                    for (int e = 0; e < E; ++e) u[e] *= n[e];
                    if (p.post_bias != nullptr) {
                        ln.vector(p.post_bias, 0.0f, t);
#pragma unroll
                        for (int e = 0; e < E; ++e) u[e] += t[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) u[e] = n[e];
                }
                if (p.drop) {
#pragma unroll
                    for (int e = 0; e < E; ++e) u[e] = (keep >> e) & 1u ? u[e] * p.dropout.scale : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] *= g[e];
                if (gate_sums) {
#pragma unroll
                    for (int e = 0; e < E; ++e) dgt[e] += u[e];
                } else if (p.dgate != nullptr) {
                    ln.store(p.dgate, r, u);
                }
                ln.vector(static_cast<const T*>(p.gate) + r / p.gate_period * p.cols, 0.0f, u);
#pragma unroll
                for (int e = 0; e < E; ++e) g[e] *= u[e];
            }
            if (p.drop) {
#pragma unroll
                for (int e = 0; e < E; ++e) g[e] = (keep >> e) & 1u ? g[e] * p.dropout.scale : 0.0f;
            }
            if constexpr (POST) {
                ln.vector(p.post_weight, 1.0f, t);
                float c3 = 0.0f, c4 = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!ln.has(e)) g[e] = 0.0f;
                    dpw[e] += g[e] * n[e];
                    dpb[e] += g[e];
                    g[e] *= t[e];
                    c3 += g[e];
                    c4 += g[e] * n[e];
                }
                ln.row_sum(c3, c4);
                c3 = p.layer ? c3 * p.inv_cols : 0.0f;
                c4 *= p.inv_cols;
#pragma unroll
                for (int e = 0; e < E; ++e) g[e] = st.y * (g[e] - c3 - n[e] * c4);
            }
            if (p.df != nullptr) ln.store(p.df, r, g);
            if (++stage == p.stages) stage = 0;
        }
        if constexpr (VEC) cp_async_wait(0);
        if constexpr (GATE) {
            if (gate_sums && p.dgate != nullptr) {
                // whole segments are finished here; one that other units share
                // goes to the unit's first or last slot
                const bool whole = seg_lo == gate_row * p.gate_period && seg_hi == (gate_row + 1) * p.gate_period;
                float* slot = p.partial + (4 * static_cast<int64_t>(p.units) + 2 * unit + (seg_lo == unit_lo ? 0 : 1)) * p.cols;
                flush_columns<T, NV, VEC>(ln, buf, dgt, slot, whole ? static_cast<T*>(p.dgate) + gate_row * p.cols : nullptr);
            }
        }
        seg_lo = seg_hi;
    }
    const int64_t plane = static_cast<int64_t>(p.units) * p.cols;
    flush_columns<T, NV, VEC>(ln, buf, dw, p.partial + unit * p.cols, nullptr);
    flush_columns<T, NV, VEC>(ln, buf, db, p.partial + plane + unit * p.cols, nullptr);
    if constexpr (POST) {
        flush_columns<T, NV, VEC>(ln, buf, dpw, p.partial + 2 * plane + unit * p.cols, nullptr);
        flush_columns<T, NV, VEC>(ln, buf, dpb, p.partial + 3 * plane + unit * p.cols, nullptr);
    }
}

constexpr int kColLanes = 32, kColRows = 16;

// The units' partial sums added in their order, rounded once.  Items 0..3 are
// the parameter vectors; item 4 + c finishes the gate row that unit c ends
// and unit c + 1 (and more) continues.
template <typename T>
__global__ void __launch_bounds__(kColLanes* kColRows)
residual_norm_columns_kernel(const RnParams p, T* d0, T* d1, T* d2, T* d3, int col_blocks) {
    pdl_wait();
    __shared__ float part[kColRows][kColLanes + 1];
    const int item = static_cast<int>(blockIdx.x) / col_blocks;
    const int64_t c = static_cast<int64_t>(blockIdx.x - item * col_blocks) * kColLanes + threadIdx.x;
    float s = 0.0f;
    T* out;
    if (item < 4) {
        out = item == 0 ? d0 : item == 1 ? d1 : item == 2 ? d2 : d3;
        if (out == nullptr) return;
        if (c < p.cols) {
            const float* src = p.partial + static_cast<int64_t>(item) * p.units * p.cols + c;
            for (int u = threadIdx.y; u < p.units; u += kColRows) s += src[static_cast<int64_t>(u) * p.cols];
        }
    } else {
        const int64_t next = item - 4 + 1;  // a unit whose start may cut a gate row
        const int64_t start = unit_begin(next, p.rows, p.units);
        const int64_t row = start / p.gate_period;
        if (start % p.gate_period == 0 || unit_of(row * p.gate_period, p.rows, p.units) != next - 1) return;
        const int64_t last = unit_of((row + 1) * p.gate_period - 1, p.rows, p.units);
        out = static_cast<T*>(p.dgate) + row * p.cols;
        if (c < p.cols) {
            const float* src = p.partial + 4 * static_cast<int64_t>(p.units) * p.cols + c;
            for (int64_t u = next - 1 + threadIdx.y; u <= last; u += kColRows) {
                const int64_t slot = 2 * u + (unit_begin(u, p.rows, p.units) / p.gate_period == row ? 0 : 1);
                s += src[slot * p.cols];
            }
        }
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < p.cols) {
        s = 0.0f;
        for (int i = 0; i < kColRows; ++i) s += part[i][threadIdx.x];
        out[c] = from_f<T>(s);
    }
}

// ---- host ----------------------------------------------------------------------

// NV octets per thread, W warps per row and CTA, CTAs per row: the cover of
// the row with the least idle columns, more octets per thread where equal
// (fewer warps to sum over).  NV 3 holds 768 columns in one warp; the
// backward pass with a post norm or a gate keeps up to five sums per column
// in registers and stays at 2.  fp32 doubles the bytes of a slot and takes 1.
struct Geometry {
    int nv, warps, cluster, groups;
};

Geometry geometry(const RnParams& p, bool f16, bool vec, bool sums5) {
    Geometry best = {1, 1, 1, 1};
    int64_t best_cover = INT64_MAX;
    const int nv_max = f16 ? (sums5 || !vec ? 2 : 3) : 1;
    for (int nv = nv_max; nv >= 1; --nv) {
        const int64_t per_warp = 256 * nv;
        const int max_warps = nv == 3 ? 8 : kMaxThreads / 32;
        const int64_t need = ceil_div(p.cols, per_warp);
        int cluster = 1;
        while (cluster * max_warps < need && cluster < kMaxCluster) cluster *= 2;
        const int64_t warps = ceil_div(need, cluster);
        if (warps > max_warps) continue;
        const int64_t cover = warps * cluster * per_warp;
        if (cover * (cluster > 1 ? 2 : 1) < best_cover) {
            best_cover = cover * (cluster > 1 ? 2 : 1);
            best = {nv, static_cast<int>(warps), cluster, 1};
        }
    }
    best.groups = best.cluster > 1 ? 1 : std::max(1, 8 / best.warps);
    return best;
}

using Kernel = void (*)(RnParams);

template <typename T, bool VEC>
Kernel forward_kernel(int nv, bool post) {
    if constexpr (VEC && sizeof(T) == 2) {
        if (nv == 3) return post ? residual_norm_kernel<T, 3, VEC, true> : residual_norm_kernel<T, 3, VEC, false>;
    }
    if constexpr (sizeof(T) == 2) {
        if (nv == 2) return post ? residual_norm_kernel<T, 2, VEC, true> : residual_norm_kernel<T, 2, VEC, false>;
    }
    return post ? residual_norm_kernel<T, 1, VEC, true> : residual_norm_kernel<T, 1, VEC, false>;
}

template <typename T, int NV, bool VEC>
Kernel backward_kernel_nv(bool post, bool gate) {
    if (post) return gate ? residual_norm_backward_kernel<T, NV, VEC, true, true> : residual_norm_backward_kernel<T, NV, VEC, true, false>;
    return gate ? residual_norm_backward_kernel<T, NV, VEC, false, true> : residual_norm_backward_kernel<T, NV, VEC, false, false>;
}

template <typename T, bool VEC>
Kernel backward_kernel(int nv, bool post, bool gate) {
    if constexpr (VEC && sizeof(T) == 2) {
        if (nv == 3) return residual_norm_backward_kernel<T, 3, VEC, false, false>;
    }
    if constexpr (sizeof(T) == 2) {
        if (nv == 2) return backward_kernel_nv<T, 2, VEC>(post, gate);
    }
    return backward_kernel_nv<T, 1, VEC>(post, gate);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const char* who, const tk_residual_norm_desc_t& d) {
    TK_CHECK_ARG(d.dtype == TK_DTYPE_F16 || d.dtype == TK_DTYPE_F32, "%s: bad dtype %d", who, static_cast<int>(d.dtype));
    TK_CHECK_ARG(d.norm == TK_NORM_LAYER || d.norm == TK_NORM_RMS, "%s: bad norm %d", who, static_cast<int>(d.norm));
    TK_CHECK_ARG(d.rows >= 0 && d.cols >= 1, "%s: rows must not be negative and cols must be positive", who);
    if (d.cols > kMaxCols) TK_FAIL(TK_ERR_UNSUPPORTED, "%s: at most %lld columns, got %lld", who, static_cast<long long>(kMaxCols), static_cast<long long>(d.cols));
    TK_CHECK_ARG(d.rows <= INT64_MAX / 8 / d.cols, "%s: too many elements", who);
    TK_CHECK_ARG(d.p >= 0.0 && d.p <= 1.0, "%s: p must be in [0, 1], got %g", who, d.p);
    TK_CHECK_ARG(d.post_norm || (d.post_weight == nullptr && d.post_bias == nullptr), "%s: post_weight and post_bias need post_norm", who);
    TK_CHECK_ARG(d.gate == nullptr || (d.gate_rows >= 1 && d.rows % d.gate_rows == 0), "%s: gate_rows must divide rows", who);
    return TK_OK;
}

RnParams params(const tk_residual_norm_desc_t& d) {
    RnParams p = {};
    p.x = d.x;
    p.f = d.f;
    p.weight = d.weight;
    p.bias = d.bias;
    p.post_weight = d.post_weight;
    p.post_bias = d.post_bias;
    p.gate = d.gate;
    p.x_new = d.x_new;
    p.h = d.h;
    p.stats = reinterpret_cast<float4*>(d.stats);
    p.rows = d.rows;
    p.cols = d.cols;
    p.gate_period = d.gate != nullptr ? d.rows / d.gate_rows : 1;
    p.a = d.residual_scale;
    p.eps = d.eps;
    p.inv_cols = static_cast<float>(1.0 / static_cast<double>(d.cols));
    p.layer = d.norm == TK_NORM_LAYER;
    p.dropout = dropout_params(d.p, d.seed, d.offset);
    p.drop = d.p > 0.0;
    return p;
}

bool vectorised(const RnParams& p) {
    for (const void* q : {p.x, p.f, p.weight, p.bias, p.post_weight, p.post_bias, p.gate, static_cast<const void*>(p.x_new),
                          static_cast<const void*>(p.h), p.gx, p.gh, static_cast<const void*>(p.dx), static_cast<const void*>(p.df),
                          static_cast<const void*>(p.dgate)})
        if (!aligned16(q)) return false;
    return p.cols % 8 == 0;
}

size_t red_bytes(const Geometry& g) {
    return 2 * sizeof(float2) * ((static_cast<size_t>(g.warps) * g.cluster * g.groups + 1) & ~static_cast<size_t>(1));
}

// Row ranges for the launch: one per resident cluster or CTA, at most one per
// `groups` rows.  `most` bounds them where a workspace was sized for it.
int max_units(int device, int64_t rows, const Geometry& g, int per_sm) {
    const int64_t resident = std::max<int64_t>(1, static_cast<int64_t>(sm_count(device)) * per_sm / g.cluster);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(resident, ceil_div(rows, g.groups))));
}

constexpr size_t kSmemPerSm = 220 * 1024;

size_t stage_bytes(const Geometry& g, bool f16, int tensors) {
    return static_cast<size_t>(g.warps) * 32 * g.groups * g.nv * (f16 ? 16 : 32) * tensors;
}

// The launch's shape and its dynamic shared memory: a ring of three rows per
// group (two in flight while one is used) where that leaves room for the CTAs
// that the registers admit, fewer rows otherwise.
size_t configure(RnParams& p, const Geometry& g, bool f16, bool vec, int tensors, bool backward) {
    p.cluster = g.cluster;
    p.warps = g.warps;
    p.groups = g.groups;
    const size_t one = stage_bytes(g, f16, tensors);
    const size_t fold = backward && g.groups > 1 ? static_cast<size_t>(g.warps) * 32 * g.groups * 8 * g.nv * sizeof(float) : 0;
    const int resident = std::max(1, 512 / (g.warps * 32 * g.groups));  // CTAs that registers admit
    p.stages = 1;
    if (vec) {
        p.stages = 3;
        while (p.stages > 1 && (red_bytes(g) + p.stages * one + 1024) * resident > kSmemPerSm) --p.stages;
    }
    return red_bytes(g) + std::max(vec ? p.stages * one : size_t(0), fold);
}

int launch(Kernel k, const RnParams& p, size_t smem, cudaStream_t s, const char* what) {
    TK_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.units) * p.cluster);
    cfg.blockDim = dim3(p.warps * 32 * p.groups);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, k, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        TK_FAIL(TK_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    }
    return launch_status(what);
}

int resident_ctas(Kernel k, const RnParams& p, size_t smem, int& per_sm) {
    TK_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    TK_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, reinterpret_cast<const void*>(k), p.warps * 32 * p.groups, smem));
    if (per_sm < 1) TK_FAIL(TK_ERR_CUDA, "residual norm: the kernel does not fit an SM");
    return TK_OK;
}

// CTAs per SM the backward pass may use: its partial sums are sized by it.
constexpr int kBackwardPerSm = 2;

template <typename T>
int columns(const RnParams& p, const tk_residual_norm_grad_desc_t& g, bool gate_items, cudaStream_t s) {
    const int col_blocks = static_cast<int>(ceil_div(p.cols, kColLanes));
    const int items = 4 + (gate_items ? p.units - 1 : 0);
    cudaError_t e = launch_pdl(residual_norm_columns_kernel<T>, dim3(static_cast<unsigned>(items) * col_blocks), dim3(kColLanes, kColRows), 0, s,
                               p, static_cast<T*>(g.dweight), static_cast<T*>(g.dbias), static_cast<T*>(g.dpost_weight),
                               static_cast<T*>(g.dpost_bias), col_blocks);
    if (e != cudaSuccess) {
        cudaGetLastError();
        TK_FAIL(TK_ERR_CUDA, "residual norm columns launch failed: %s", cudaGetErrorString(e));
    }
    return launch_status("residual_norm_columns");
}

}  // namespace
}  // namespace tk

extern "C" {

int tk_residual_norm(const tk_residual_norm_desc_t* desc, void* stream) {
    using namespace tk;
    TK_CHECK_ARG(desc != nullptr, "tk_residual_norm: NULL descriptor");
    const tk_residual_norm_desc_t& d = *desc;
    if (int rc = check("tk_residual_norm", d)) return rc;
    if (d.rows == 0) return TK_OK;
    TK_CHECK_ARG(d.x && d.f && d.x_new && d.h, "tk_residual_norm: NULL pointer");
    TK_CHECK_ARG(aligned16(d.stats), "tk_residual_norm: stats must be 16-byte aligned");
    RnParams p = params(d);
    const bool f16 = d.dtype == TK_DTYPE_F16, vec = vectorised(p);
    const Geometry g = geometry(p, f16, vec, false);
    const size_t smem = configure(p, g, f16, vec, 2, false);
    const Kernel k = f16 ? (vec ? forward_kernel<__half, true>(g.nv, d.post_norm) : forward_kernel<__half, false>(g.nv, d.post_norm))
                         : (vec ? forward_kernel<float, true>(g.nv, d.post_norm) : forward_kernel<float, false>(g.nv, d.post_norm));
    int per_sm = 0;
    if (int rc = resident_ctas(k, p, smem, per_sm)) return rc;
    p.units = max_units(current_device(), p.rows, g, per_sm);
    return launch(k, p, smem, static_cast<cudaStream_t>(stream), "residual_norm");
}

size_t tk_residual_norm_backward_workspace_size(const tk_residual_norm_grad_desc_t* desc) {
    using namespace tk;
    if (desc == nullptr || check("tk_residual_norm_backward", desc->fwd) != TK_OK) return 0;
    // [4 + 2][units][cols] fp32 partial sums, `units` at its largest
    const int64_t units = std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(sm_count(current_device())) * kBackwardPerSm, desc->fwd.rows));
    return static_cast<size_t>(6 * units * desc->fwd.cols) * sizeof(float) + 256;
}

int tk_residual_norm_backward(const tk_residual_norm_grad_desc_t* desc, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace tk;
    TK_CHECK_ARG(desc != nullptr, "tk_residual_norm_backward: NULL descriptor");
    const tk_residual_norm_desc_t& d = desc->fwd;
    if (int rc = check("tk_residual_norm_backward", d)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f16 = d.dtype == TK_DTYPE_F16;
    if (d.rows == 0) {  // sums over no rows
        const size_t row = static_cast<size_t>(d.cols) * dtype_size(d.dtype);
        for (void* q : {desc->dweight, desc->dbias, desc->dpost_weight, desc->dpost_bias})
            if (q != nullptr) TK_CUDA_TRY(cudaMemsetAsync(q, 0, row, s));
        if (desc->dgate != nullptr && d.gate != nullptr) TK_CUDA_TRY(cudaMemsetAsync(desc->dgate, 0, row * d.gate_rows, s));
        return TK_OK;
    }
    TK_CHECK_ARG(d.x_new && d.stats && aligned16(d.stats), "tk_residual_norm_backward: x_new and 16-byte aligned stats are needed");
    TK_CHECK_ARG(desc->grad_x_new || desc->grad_h, "tk_residual_norm_backward: no incoming gradient");
    TK_CHECK_ARG(d.f || !(d.post_norm || d.gate), "tk_residual_norm_backward: f is needed with a post norm or a gate");
    RnParams p = params(d);
    p.x = nullptr;
    p.h = nullptr;
    p.bias = nullptr;
    p.gx = desc->grad_x_new;
    p.gh = desc->grad_h;
    p.dx = desc->dx;
    p.df = desc->df;
    p.dgate = d.gate != nullptr ? desc->dgate : nullptr;
    const bool gate = d.gate != nullptr, post = d.post_norm != 0;
    if (!gate && !post) p.f = nullptr;
    const bool vec = vectorised(p);
    const Geometry g = geometry(p, f16, vec, gate || post);
    const size_t smem = configure(p, g, f16, vec, gate || post ? 4 : 3, true);
    const Kernel k = f16 ? (vec ? backward_kernel<__half, true>(g.nv, post, gate) : backward_kernel<__half, false>(g.nv, post, gate))
                         : (vec ? backward_kernel<float, true>(g.nv, post, gate) : backward_kernel<float, false>(g.nv, post, gate));
    int per_sm = 0;
    if (int rc = resident_ctas(k, p, smem, per_sm)) return rc;
    p.units = max_units(current_device(), p.rows, g, std::min(per_sm, kBackwardPerSm));
    const size_t need = static_cast<size_t>(6) * p.units * p.cols * sizeof(float);
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
        TK_FAIL(TK_ERR_WORKSPACE, "tk_residual_norm_backward: 16-byte aligned workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    p.partial = static_cast<float*>(workspace);
    if (int rc = launch(k, p, smem, s, "residual_norm_backward")) return rc;
    const bool gate_items = p.dgate != nullptr && p.gate_period > 1;
    if (!desc->dweight && !desc->dbias && !desc->dpost_weight && !desc->dpost_bias && !gate_items) return TK_OK;
    return f16 ? columns<__half>(p, *desc, gate_items, s) : columns<float>(p, *desc, gate_items, s);
}

}  // extern "C"
