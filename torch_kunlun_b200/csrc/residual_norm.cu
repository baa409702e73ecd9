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
// (an rms norm has no mean(t) terms).  x_new is formed again from x and f, as
// the forward pass had it before it was rounded: from the rounded x_new the
// binary16 gradient of weight came out up to 1.5 times as far off.
//
// HBM bounds both directions: 4 tensors forward, 6 backward.  A group of W
// warps (or some lanes of a warp, where rows are narrow) holds a row in
// registers, 8 * NV columns per thread, as pairs for the two-wide binary32
// instructions (one per element made the kernels issue-bound: 8192 x 4096 with
// both norms took 93 us forward, 2.4 TB/s, at 63 % issue); a CTA runs several
// groups when rows are short, and a cluster of CTAs shares a row that one CTA
// cannot hold, its sums exchanged through distributed shared memory.  The next
// rows are copied to shared memory (cp.async) while a row is worked on: each
// thread its own columns where rows are 16-byte aligned, which needs no
// barrier, otherwise the group the 16-byte vectors that cover the row.  CTAs
// own contiguous rows; column sums stay in registers until a CTA's rows end,
// and a second kernel adds the CTAs' partial sums in a fixed order, so no
// gradient depends on timing.  Where a CTA cannot hold a row's columns and
// their sums, a pass of its own adds the columns, from the row statistics and
// the two row means that the first pass leaves.
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
    float2* means;   // backward of wide rows: mean(t), mean(t * n) per row
    float* partial;  // backward: [4][units][cols], then the gate's [2 * units][cols]
    int64_t rows, cols, gate_period;  // row r uses gate row r / gate_period
    int units;                        // row ranges: clusters of `cluster` CTAs
    int cluster, warps, lanes, groups, stages;  // a row has warps * lanes threads of a CTA
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

template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }

// Two-wide binary32 arithmetic (one instruction for a pair).
union Pair {
    float2 f;
    unsigned long long u;
};
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    Pair x{a}, y{b}, z{c}, r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(x.u), "l"(y.u), "l"(z.u));
    return r.f;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    Pair x{a}, y{b}, r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(x.u), "l"(y.u));
    return r.f;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    Pair x{a}, y{b}, r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(x.u), "l"(y.u));
    return r.f;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The first `bytes` of a 16-byte vector, zeros after them.
__device__ __forceinline__ void cp_async16_part(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// E values of type T in registers, as stored (two binary16 to a word).
template <typename T, int E>
struct Raw {
    uint32_t r[E * sizeof(T) / 4];
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (sizeof(T) == 2) {
            return __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
        } else {
            return make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        }
    }
    __device__ __forceinline__ void set(int e, T v) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t b = __half_as_ushort(v);
            r[e / 2] = e % 2 ? (r[e / 2] & 0xFFFFu) | b << 16 : b;
        } else {
            r[e] = __float_as_uint(v);
        }
    }
    __device__ __forceinline__ void vec(int i, uint4 v) { r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w; }
};

// The W words that start `bytes` (0 to 15, even) into u, in u[0..W).
template <int W>
__device__ __forceinline__ void shift_words(uint32_t (&u)[W + 5], uint32_t bytes) {
    u[W + 4] = 0;
    if (bytes & 8u) {
#pragma unroll
        for (int i = 0; i < W + 2; ++i) u[i] = u[i + 2];
    }
    if (bytes & 4u) {
#pragma unroll
        for (int i = 0; i < W + 1; ++i) u[i] = u[i + 1];
    }
    if (bytes & 2u) {
#pragma unroll
        for (int i = 0; i < W; ++i) u[i] = __funnelshift_r(u[i], u[i + 1], 16);
    }
}

constexpr int kTailPad = 32;  // bytes of a row's copy beyond the row: both 16-byte roundings

// One thread's share of a row: which columns it holds, the copies of the rows
// to come, and the sums over the threads that hold the rest of the row.
//
// A thread holds octets of 8 consecutive columns.  VEC: every row is 16-byte
// aligned (pointers and cols * size), octets are 16-byte accesses.  Otherwise a
// row starts anywhere in a 16-byte vector: its copy in shared memory keeps that
// offset, an octet is shifted out of the vectors that cover it, and a lane
// stores the whole vector that its octet and its neighbour's fill (the warp's
// outer lanes and the row's end store element by element).
//
// NARROW (NV 1): a row has p.lanes threads, a power of two below 32, and a warp
// several rows, whose lanes name only one another in shuffles and barriers: the
// rows of a warp need not end together.
template <typename T, int NV, bool VEC, bool NARROW = false>
struct Lane {
    static_assert(!NARROW || NV == 1, "a narrow row is one octet to a lane");
    static constexpr int E = 8 * NV, P = E / 2;
    [[maybe_unused]] static constexpr int PARTS = sizeof(T) / 2;  // 16-byte vectors of an octet
    int t, lane, lanes, warp, group, gthreads, rank, tensors;  // lane, lanes: of the warp, or of the narrow row
    unsigned mask;   // those lanes
    int col0, cols;  // first column of the CTA's slice, columns of a row
    uint32_t ring;   // this thread's (VEC) or this group's copies
    uint32_t image;  // bytes of one row's copy (not VEC)
    float2* red;
    int red_stride, red_n, red_width, parity;  // red_width: red_n up to a power of two, at most 32
    bool full;       // every column of the slice is in the row
    const RnParams& p;

    __device__ Lane(const RnParams& pr, uint8_t* smem, int tensors_) : tensors(tensors_), p(pr) {
        gthreads = NARROW ? p.lanes : p.warps * 32;
        group = threadIdx.x / gthreads;
        t = threadIdx.x - group * gthreads;
        lanes = NARROW ? p.lanes : 32;
        lane = threadIdx.x & (lanes - 1);
        mask = NARROW ? ((1u << lanes) - 1u) << ((threadIdx.x & 31) - lane) : 0xFFFFFFFFu;
        warp = t >> 5;
        rank = p.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
        col0 = rank * gthreads * E;
        cols = static_cast<int>(p.cols);
        full = col0 + gthreads * E <= cols;
        red = reinterpret_cast<float2*>(smem);
        red_n = p.warps * p.cluster;
        red_stride = red_n * p.groups;
        red_width = red_n >= 32 ? 32 : red_n <= 1 ? 1 : 1 << (32 - __clz(red_n - 1));
        parity = 0;
        ring = smem_u32(smem + 2 * sizeof(float2) * ((red_stride + 1) & ~1));
        image = static_cast<uint32_t>(gthreads * E * sizeof(T) + kTailPad);
        if constexpr (VEC) {
            ring += threadIdx.x * 16;
        } else {
            ring += static_cast<uint32_t>(group * p.stages * tensors) * image;
        }
        if (p.cluster > 1) cluster_sync_all();  // every CTA runs before its memory is written
    }
    __device__ __forceinline__ int col(int e) const { return col0 + (e / 8 * gthreads + t) * 8 + e % 8; }
    __device__ __forceinline__ bool has(int e) const { return full || col(VEC ? e & ~7 : e) < cols; }
    // All of octet v is in the row (VEC: or none of it).
    __device__ __forceinline__ bool whole(int v) const { return full || col(8 * v) + (VEC ? 0 : 7) < cols; }

    // Begins the copy of tensor k's row into `stage`; `row` is the element at
    // which the row starts.
    __device__ __forceinline__ void fetch(const void* tensor, int64_t row, int stage, int k) const {
        if constexpr (VEC) {
            const T* src = static_cast<const T*>(tensor) + row;
            const uint32_t slot = ring + static_cast<uint32_t>((stage * tensors + k) * NV * PARTS) * blockDim.x * 16;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!has(8 * v)) continue;
#pragma unroll
                for (int i = 0; i < PARTS; ++i) cp_async16(slot + (v * PARTS + i) * blockDim.x * 16, reinterpret_cast<const uint4*>(src + col(8 * v)) + i);
            }
        } else {
            const int width = min(cols - col0, gthreads * E);
            if (width <= 0) return;
            const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<const T*>(tensor) + row + col0);
            const uintptr_t from = at & ~static_cast<uintptr_t>(15);
            const uintptr_t end = reinterpret_cast<uintptr_t>(static_cast<const T*>(tensor) + p.rows * p.cols);
            const uint32_t slot = ring + static_cast<uint32_t>(stage * tensors + k) * image;
            const int vectors = static_cast<int>((at + width * sizeof(T) - from + 15) / 16);
            for (int i = t; i < vectors; i += gthreads) {
                const uintptr_t v = from + 16 * static_cast<uintptr_t>(i);
                if (v >= reinterpret_cast<uintptr_t>(tensor)) {
                    cp_async16_part(slot + 16 * i, reinterpret_cast<const void*>(v), static_cast<int>(min(static_cast<uintptr_t>(16), end - v)));
                } else {  // the tensor begins inside this vector
                    for (uintptr_t a = reinterpret_cast<uintptr_t>(tensor); a < v + 16 && a < end; a += 2)
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(slot + static_cast<uint32_t>(a - from)), "h"(*reinterpret_cast<const uint16_t*>(a)) : "memory");
                }
            }
        }
    }
    // Threads of the group wait for one another.
    __device__ __forceinline__ void group_sync() const {
        if (NARROW || p.warps == 1) {
            __syncwarp(mask);
        } else {
            named_barrier_sync(1 + group, gthreads);
        }
    }
    __device__ __forceinline__ void row_values(const void* tensor, int64_t row, int stage, int k, float2 (&o)[P]) const {
        Raw<T, E> w;
        if constexpr (VEC) {
            const uint32_t slot = ring + static_cast<uint32_t>((stage * tensors + k) * NV * PARTS) * blockDim.x * 16;
#pragma unroll
            for (int v = 0; v < NV * PARTS; ++v) {
                uint4 u;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(slot + v * blockDim.x * 16) : "memory");
                w.vec(v, u);
            }
            if (!full) {  // octets past the row were not copied
#pragma unroll
                for (int v = 0; v < NV * PARTS; ++v)
                    if (!has(8 * (v / PARTS))) w.vec(v, make_uint4(0, 0, 0, 0));
            }
        } else {
            const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(static_cast<const T*>(tensor) + row + col0)) & 15u;
            const uint32_t slot = ring + static_cast<uint32_t>(stage * tensors + k) * image;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                constexpr int W = 4 * PARTS;  // words of an octet
                uint32_t u[W + 5];
#pragma unroll
                for (int i = 0; i <= PARTS; ++i)
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(u[4 * i]), "=r"(u[4 * i + 1]), "=r"(u[4 * i + 2]), "=r"(u[4 * i + 3])
                                 : "r"(slot + static_cast<uint32_t>((v * gthreads + t) * PARTS + i) * 16)
                                 : "memory");
                shift_words<W>(u, at);
                if (!whole(v)) {  // what lies past the row reads as zero
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (has(8 * v + e)) continue;
                        if constexpr (sizeof(T) == 2) {
                            u[e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                        } else {
                            u[e] = 0;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < W; ++i) w.r[v * W + i] = u[i];
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) o[i] = w.pair(i);
    }
    // This thread's columns of a [cols] vector: `absent` where it is NULL, 0
    // past the row.
    __device__ __forceinline__ void vector(const void* base, float absent, Raw<T, E>& w) const {
        const T* b = static_cast<const T*>(base);
        const bool vec = VEC || (reinterpret_cast<uintptr_t>(b) & 15) == 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (b != nullptr && vec && whole(v) && has(8 * v)) {
#pragma unroll
                for (int i = 0; i < PARTS; ++i) w.vec(v * PARTS + i, __ldg(reinterpret_cast<const uint4*>(b + col(8 * v)) + i));
            } else {
#pragma unroll
                for (int e = 8 * v; e < 8 * v + 8; ++e) w.set(e, !has(e) ? from_f<T>(0.0f) : b != nullptr ? b[col(e)] : from_f<T>(absent));
            }
        }
    }
    __device__ __forceinline__ void store(void* tensor, int64_t row, const float2 (&v)[P]) const {
        T* b = static_cast<T*>(tensor) + row;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            constexpr int W = 4 * PARTS;
            uint32_t o[W];
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __half2 h = __float22half2_rn(v[4 * k + i]);
                    o[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(i % 2 ? v[4 * k + i / 2].y : v[4 * k + i / 2].x);
            }
            T* to = b + col(8 * k);
            if constexpr (VEC) {
                if (!has(8 * k)) continue;
#pragma unroll
                for (int i = 0; i < PARTS; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            } else {
                // `off` bytes of the octet's first vector belong to the octet before
                const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to)) & 15u;
                uint32_t u[W + 5];
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = __shfl_up_sync(mask, o[W - 4 + i], 1, lanes);
#pragma unroll
                for (int i = 0; i < W; ++i) u[4 + i] = o[i];
                if (off == 0) {
#pragma unroll
                    for (int i = 0; i < W; ++i) u[i] = o[i];
                } else {
                    shift_words<W>(u, 16u - off);
                }
                const bool me = whole(k) && has(8 * k);
                if (me && (lane > 0 || off == 0)) {
                    uint4* q = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(to) - off);
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) q[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
                }
                // what no whole store covers: the head of a first or partial
                // octet, the tail where the next lane stores no whole vector
                const bool next = lane < lanes - 1 && (full || col(8 * k) + 15 < cols);
                const int count = full ? 8 : min(8, max(0, cols - col(8 * k)));        // elements of the octet in the row
                const int split = static_cast<int>((16u * PARTS - off) / sizeof(T));  // elements in its own vectors
                const uint32_t head = (1u << min(split, 8)) - 1u;
                uint32_t need = me && (lane > 0 || off == 0) ? 0u : head;
                if (off != 0 && !next) need |= ~head;
                need &= (1u << count) - 1u;
                if (need != 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if constexpr (sizeof(T) == 2) {
                            if ((need >> e) & 1u) reinterpret_cast<uint16_t*>(to)[e] = static_cast<uint16_t>(e % 2 ? o[e / 2] >> 16 : o[e / 2]);
                        } else {
                            if ((need >> e) & 1u) reinterpret_cast<uint32_t*>(to)[e] = o[e];
                        }
                    }
                }
            }
        }
    }
    // Keep bits of this thread's columns of the row that starts at an element.
    __device__ __forceinline__ uint32_t keep(int64_t row) const {
        uint32_t m = 0;
        if constexpr (VEC) {
#pragma unroll
            for (int v = 0; v < NV; ++v) m |= dropout_keep8(p.dropout, static_cast<uint32_t>((row + col(8 * v)) / 8)) << (8 * v);
        } else {
            // the octet's elements begin `shift` into a block of four
            const uint32_t shift = static_cast<uint32_t>(row) & 3u;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const uint32_t block = static_cast<uint32_t>((row + col(8 * v)) / 4);
                const uint32_t bits = dropout_keep4(p.dropout, block) | dropout_keep4(p.dropout, block + 1) << 4 | dropout_keep4(p.dropout, block + 2) << 8;
                m |= ((bits >> shift) & 0xFFu) << (8 * v);
            }
        }
        return m;
    }
    // Sums over the row's threads of N values; every thread gets the same bits.
    // One exchange buffer is read while the next sum fills the other, so one
    // barrier per sum is enough.
    template <int N>
    __device__ __forceinline__ float2 row_sum(float2 s) {
        if constexpr (NARROW) {
#pragma unroll
            for (int m = 8; m > 0; m >>= 1)
                if (m < lanes) s = lanes_add<N>(s, m, mask);
            return s;
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s = lanes_add<N>(s, m);
        if (red_n == 1) return s;
        float2* buf = red + parity * red_stride + group * red_n;
        parity ^= 1;
        const int slot = rank * p.warps + warp;
        if (p.cluster == 1) {
            if (lane == 0) buf[slot] = s;
            named_barrier_sync(1 + group, gthreads);
        } else {
            if (lane < p.cluster) {
                const uint32_t to = mapa_shared(smem_u32(buf + slot), lane);
                st_shared_cluster_u32(to, __float_as_uint(s.x));
                st_shared_cluster_u32(to + 4, __float_as_uint(s.y));
            }
            __syncwarp();
            cluster_sync_all();
        }
        const int at = lane & (red_width - 1);
        s = at < red_n ? buf[at] : make_float2(0.0f, 0.0f);
        for (int i = at + 32; i < red_n; i += 32) s = add2(s, buf[i]);
        for (int m = red_width / 2; m > 0; m >>= 1) s = lanes_add<N>(s, m);
        return s;
    }
    template <int N>
    static __device__ __forceinline__ float2 lanes_add(float2 s, int m, unsigned mask = 0xFFFFFFFFu) {
        const float x = __shfl_xor_sync(mask, s.x, m);
        if (N == 1) return make_float2(s.x + x, 0.0f);
        return add2(s, make_float2(x, __shfl_xor_sync(mask, s.y, m)));
    }
    // mean and rstd of v over the row (mean 0 for an rms norm); the mean
    // square is taken about the mean, of values held in registers.
    __device__ __forceinline__ void moments(const float2 (&v)[P], float& mean, float& rstd) {
        mean = 0.0f;
        if (p.layer) {
            float2 s = v[0];
#pragma unroll
            for (int i = 1; i < P; ++i) s = add2(s, v[i]);
            mean = row_sum<1>(make_float2(s.x + s.y, 0.0f)).x * p.inv_cols;
        }
        const float2 shift = both(-mean);
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int o = 0; o < NV; ++o) {
            if (VEC ? has(8 * o) : whole(o)) {
#pragma unroll
                for (int i = 4 * o; i < 4 * o + 4; ++i) {
                    const float2 c = add2(v[i], shift);
                    s = fma2(c, c, s);
                }
            } else if constexpr (!VEC) {
#pragma unroll
                for (int i = 4 * o; i < 4 * o + 4; ++i) {
                    const float2 c = add2(v[i], shift);
                    if (has(2 * i)) s.x = fmaf(c.x, c.x, s.x);
                    if (has(2 * i + 1)) s.y = fmaf(c.y, c.y, s.y);
                }
            }
        }
        rstd = rsqrtf(row_sum<1>(make_float2(s.x + s.y, 0.0f)).x * p.inv_cols + p.eps);
    }
    __device__ __forceinline__ void drop(uint32_t keep, float2 (&v)[P]) const {
        const float2 s = both(p.dropout.scale);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            v[i] = mul2(v[i], s);
            if (!((keep >> (2 * i)) & 1u)) v[i].x = 0.0f;
            if (!((keep >> (2 * i + 1)) & 1u)) v[i].y = 0.0f;
        }
    }
    // The same straight from the generator's words, where no mask is needed.
    __device__ __forceinline__ void drop_row(int64_t row, float2 (&v)[P]) const {
        if constexpr (VEC) {
            const float2 s = both(p.dropout.scale);
            const uint32_t t32 = p.dropout.threshold;
#pragma unroll
            for (int o = 0; o < E / 4; ++o) {
                uint32_t w[4];
                philox4x32_10(static_cast<uint32_t>((row + col(4 * o)) / 4), 0, p.dropout.offset, p.dropout.seed, w);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 m = mul2(v[2 * o + i], s);
                    v[2 * o + i] = make_float2(w[2 * i] >= t32 ? m.x : 0.0f, w[2 * i + 1] >= t32 ? m.y : 0.0f);
                }
            }
            if (p.dropout.none_kept) {
#pragma unroll
                for (int i = 0; i < P; ++i) v[i] = make_float2(0.0f, 0.0f);
            }
        } else {
            drop(keep(row), v);
        }
    }
    // The group's walk over rows: a step of `groups` apart, or (OWN) whole gate
    // rows of gate_period rows, a step of `groups` gate rows apart.
    template <bool OWN>
    struct Walk {
        int64_t row;
        int left;  // OWN: rows of this gate row from here on
        __device__ __forceinline__ void next(const RnParams& p) {
            if constexpr (OWN) {
                ++row;
                if (--left == 0) {
                    left = static_cast<int>(p.gate_period);
                    row += static_cast<int64_t>(p.groups - 1) * p.gate_period;
                }
            } else {
                row += p.groups;
            }
        }
    };
    // Runs f(walk, stage) over the group's rows from `begin` to below `end`, with
    // the copies of the rows ahead under way.
    template <bool OWN, typename Fetch, typename F>
    __device__ __forceinline__ void rows(int64_t begin, int64_t end, Fetch fetch_row, F f) const {
        const int ahead = p.stages - 1;
        Walk<OWN> at = {begin, OWN ? static_cast<int>(p.gate_period) : 0}, next = at;
        for (int i = 0; i < ahead; ++i) {
            if (next.row < end) fetch_row(next.row, i);
            cp_async_commit();
            next.next(p);
        }
        int stage = 0;
        for (; at.row < end; at.next(p)) {
            int ns = stage + ahead;
            if (ns >= p.stages) ns -= p.stages;
            if constexpr (VEC) {
                if (next.row < end) fetch_row(next.row, ns);
                cp_async_commit();
                cp_async_wait(ahead);
            } else {
                // the group's copies of this row are in, and its last row's
                // are read, before that stage is filled again (stages >= 2)
                cp_async_wait(ahead - 1);
                group_sync();
                if (next.row < end) fetch_row(next.row, ns);
                cp_async_commit();
            }
            next.next(p);
            f(at, stage);
            if (++stage == p.stages) stage = 0;
        }
        cp_async_wait(0);
    }
};

// Parameter vectors stay in registers for up to 24 columns per thread; wider
// shares read them again for each row (from L1).
template <typename T, int NV, bool VEC, bool POST, bool NARROW = false>
__global__ void __launch_bounds__(kMaxThreads, 1) residual_norm_kernel(const RnParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    using L = Lane<T, NV, VEC, NARROW>;
    constexpr int P = L::P;
    constexpr bool KEPT = NV <= 3;
    L ln(p, smem, 2);
    const int64_t unit = blockIdx.x / p.cluster;
    const int64_t end = unit_begin(unit + 1, p.rows, p.units);
    const int64_t begin = unit_begin(unit, p.rows, p.units) + ln.group;
    Raw<T, L::E> w, b, pw, pb, gate;
    int64_t gate_row = -1;
    if constexpr (KEPT) {
        ln.vector(p.weight, 1.0f, w);
        if (p.bias != nullptr) ln.vector(p.bias, 0.0f, b);
        if constexpr (POST) {
            ln.vector(p.post_weight, 1.0f, pw);
            if (p.post_bias != nullptr) ln.vector(p.post_bias, 0.0f, pb);
        }
    }
    ln.template rows<false>(
        begin, end,
        [&](int64_t r, int stage) {
            const int64_t at = r * p.cols;
            ln.fetch(p.x, at, stage, 0);
            ln.fetch(p.f, at, stage, 1);
        },
        [&](const auto& walk, int stage) {
            const int64_t r = walk.row, at = r * p.cols;
            float2 u[P], x[P];
            ln.row_values(p.f, at, stage, 1, u);
            float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
            if constexpr (POST) {
                ln.moments(u, st.x, st.y);
                if constexpr (!KEPT) ln.vector(p.post_weight, 1.0f, pw);
                const float2 s = both(st.y), c = both(-st.x);
#pragma unroll
                for (int i = 0; i < P; ++i) u[i] = mul2(mul2(add2(u[i], c), s), pw.pair(i));
                if (p.post_bias != nullptr) {
                    if constexpr (!KEPT) ln.vector(p.post_bias, 0.0f, pb);
#pragma unroll
                    for (int i = 0; i < P; ++i) u[i] = add2(u[i], pb.pair(i));
                }
            }
            if (p.drop) ln.drop_row(at, u);
            if (p.gate != nullptr) {
                const int64_t g = p.gate_period == p.rows ? 0 : r / p.gate_period;
                if (!KEPT || g != gate_row) ln.vector(static_cast<const T*>(p.gate) + g * p.cols, 0.0f, gate);
                gate_row = g;
#pragma unroll
                for (int i = 0; i < P; ++i) u[i] = mul2(u[i], gate.pair(i));
            }
            ln.row_values(p.x, at, stage, 0, x);
            const float2 a = both(p.a);
#pragma unroll
            for (int i = 0; i < P; ++i) u[i] = fma2(a, x[i], u[i]);
            ln.store(p.x_new, at, u);
            ln.moments(u, st.z, st.w);
            if constexpr (!KEPT) ln.vector(p.weight, 1.0f, w);
            const float2 s = both(st.w), c = both(-st.z);
#pragma unroll
            for (int i = 0; i < P; ++i) u[i] = mul2(mul2(add2(u[i], c), s), w.pair(i));
            if (p.bias != nullptr) {
                if constexpr (!KEPT) ln.vector(p.bias, 0.0f, b);
#pragma unroll
                for (int i = 0; i < P; ++i) u[i] = add2(u[i], b.pair(i));
            }
            ln.store(p.h, at, u);
            if (p.stats != nullptr && ln.t == 0 && ln.rank == 0) p.stats[r] = st;
        });
}

// Adds `acc` over the CTA's groups and writes the CTA's columns, as fp32
// partial sums or (to_final) as the finished gradient.  Every thread of the
// CTA takes part; `buf` is the ring's memory, idle at this point.
template <typename T, int NV, bool VEC, bool NARROW>
__device__ __forceinline__ void flush_columns(const Lane<T, NV, VEC, NARROW>& ln, float* buf, const float2 (&acc)[4 * NV],
                                              float* partial, T* final_row) {
    const RnParams& p = ln.p;
    const int width = ln.gthreads * 8 * NV;
    if (p.groups > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8 * NV; ++e) buf[ln.group * width + (ln.col(e) - ln.col0)] = e % 2 ? acc[e / 2].y : acc[e / 2].x;
        __syncthreads();
        for (int c = threadIdx.x; c < width && ln.col0 + c < p.cols; c += blockDim.x) {
            float s = 0.0f;
#pragma unroll 8
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
            const float v = e % 2 ? acc[e / 2].y : acc[e / 2].x;
            if (final_row != nullptr) {
                final_row[ln.col(e)] = from_f<T>(v);
            } else {
                partial[ln.col(e)] = v;
            }
        }
    }
}

// SUMS: keeps the column sums; otherwise leaves p.means for the column pass.
// kGateOwn: groups take whole gate rows and finish their gradients alone.
enum Gate { kNoGate, kGate, kGateOwn };

template <typename T, int NV, bool VEC, bool POST, Gate GATED, bool SUMS, bool NARROW = false>
__global__ void __launch_bounds__(kMaxThreads, 1) residual_norm_backward_kernel(const RnParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    using L = Lane<T, NV, VEC, NARROW>;
    constexpr int P = L::P;
    constexpr bool GATE = GATED != kNoGate, OWN = GATED == kGateOwn;
    L ln(p, smem, 4);
    float* const buf = reinterpret_cast<float*>(smem + 2 * sizeof(float2) * ((ln.red_stride + 1) & ~1));
    const int64_t unit = blockIdx.x / p.cluster;
    // a unit is a range of rows, or of gate rows
    const int64_t each = OWN ? p.gate_period : 1;
    const int64_t unit_lo = unit_begin(unit, p.rows / each, p.units) * each, unit_hi = unit_begin(unit + 1, p.rows / each, p.units) * each;
    const bool gate_sums = GATE && SUMS && p.gate_period > 1;  // else each row writes its own gradient
    Raw<T, L::E> w, pw, gate;
    ln.vector(p.weight, 1.0f, w);
    if constexpr (POST) ln.vector(p.post_weight, 1.0f, pw);
    float2 dw[SUMS ? P : 1], db[SUMS ? P : 1], dpw[POST && SUMS ? P : 1], dpb[POST && SUMS ? P : 1], dgt[GATE && SUMS ? P : 1];
    if constexpr (SUMS) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            dw[i] = db[i] = make_float2(0.0f, 0.0f);
            if constexpr (POST) dpw[i] = dpb[i] = make_float2(0.0f, 0.0f);
        }
    }
    int64_t gate_row = -1;
    // a segment: the rows of this unit that share a gate row (all of them
    // where the CTA's groups do not add up a gate's gradient together)
    int64_t seg_lo = unit_lo;
    while (seg_lo < unit_hi) {
        const int64_t seg_gate = gate_sums && !OWN ? seg_lo / p.gate_period : 0;
        const int64_t seg_hi = gate_sums && !OWN ? min(unit_hi, (seg_gate + 1) * p.gate_period) : unit_hi;
        if constexpr (GATE && SUMS) {
#pragma unroll
            for (int i = 0; i < P; ++i) dgt[i] = make_float2(0.0f, 0.0f);
        }
        float4 next_st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // read a row ahead
        const int64_t first = seg_lo + ln.group * each;
        if (first < seg_hi) next_st = p.stats[first];
        ln.template rows<OWN>(
            first, seg_hi,
            [&](int64_t r, int stage) {
                const int64_t at = r * p.cols;
                if (p.gx != nullptr) ln.fetch(p.gx, at, stage, 0);
                if (p.gh != nullptr) {
                    ln.fetch(p.gh, at, stage, 1);
                    ln.fetch(p.x, at, stage, 2);
                }
                ln.fetch(p.f, at, stage, 3);
            },
            [&](const auto& walk, int stage) {
                const int64_t r = walk.row, at = r * p.cols;
                const float4 st = next_st;
                auto after = walk;
                after.next(p);
                if (after.row < seg_hi) next_st = p.stats[after.row];
                const uint32_t keep = p.drop ? ln.keep(at) : 0u;
                if constexpr (GATE) {
                    const int64_t k = p.gate_period == p.rows ? 0 : r / p.gate_period;
                    if (k != gate_row) ln.vector(static_cast<const T*>(p.gate) + k * p.cols, 0.0f, gate);
                    gate_row = k;
                }
                float2 u[P];  // the block's dropped output
                ln.row_values(p.f, at, stage, 3, u);
                if constexpr (POST) {
                    const float2 s = both(st.y), c = both(-st.x);
#pragma unroll
                    for (int i = 0; i < P; ++i) u[i] = mul2(mul2(add2(u[i], c), s), pw.pair(i));
                    if (p.post_bias != nullptr) {
                        Raw<T, L::E> pb;
                        ln.vector(p.post_bias, 0.0f, pb);
#pragma unroll
                        for (int i = 0; i < P; ++i) u[i] = add2(u[i], pb.pair(i));
                    }
                }
                if (p.drop) ln.drop(keep, u);
                float2 g[P];
                if (p.gh != nullptr) {
                    float2 n[P], h[P];
                    ln.row_values(p.x, at, stage, 2, n);
                    ln.row_values(p.gh, at, stage, 1, h);
                    const float2 a = both(p.a);
#pragma unroll
                    for (int i = 0; i < P; ++i) n[i] = GATE ? fma2(a, n[i], mul2(u[i], gate.pair(i))) : fma2(a, n[i], u[i]);
                    const float2 s = both(st.w), c = both(-st.z);
                    float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        n[i] = mul2(add2(n[i], c), s);
                        if constexpr (SUMS) {
                            dw[i] = fma2(h[i], n[i], dw[i]);
                            db[i] = add2(db[i], h[i]);
                        }
                        h[i] = mul2(h[i], w.pair(i));  // 0 past the row
                        s1 = add2(s1, h[i]);
                        s2 = fma2(h[i], n[i], s2);
                    }
                    s1 = ln.template row_sum<2>(make_float2(s1.x + s1.y, s2.x + s2.y));
                    const float2 m1 = both(p.layer ? -s1.x * p.inv_cols : 0.0f), m2 = both(-s1.y * p.inv_cols);
                    if (!SUMS && ln.t == 0 && ln.rank == 0) p.means[r] = make_float2(-m1.x, -m2.x);
#pragma unroll
                    for (int i = 0; i < P; ++i) h[i] = add2(fma2(n[i], m2, h[i]), m1);
                    if (p.gx != nullptr) {
                        ln.row_values(p.gx, at, stage, 0, g);
#pragma unroll
                        for (int i = 0; i < P; ++i) g[i] = fma2(h[i], s, g[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < P; ++i) g[i] = mul2(h[i], s);
                    }
                } else {
                    ln.row_values(p.gx, at, stage, 0, g);
                }
                if (p.dx != nullptr) {
                    float2 o[P];
                    const float2 a = both(p.a);
#pragma unroll
                    for (int i = 0; i < P; ++i) o[i] = mul2(a, g[i]);
                    ln.store(p.dx, at, o);
                }
                if constexpr (GATE) {
                    if (gate_sums) {
                        if constexpr (SUMS) {
#pragma unroll
                            for (int i = 0; i < P; ++i) dgt[i] = fma2(u[i], g[i], dgt[i]);
                            if constexpr (OWN) {
                                if (walk.left == 1) {
                                    ln.store(p.dgate, gate_row * p.cols, dgt);
#pragma unroll
                                    for (int i = 0; i < P; ++i) dgt[i] = make_float2(0.0f, 0.0f);
                                }
                            }
                        }
                    } else if (p.gate_period == 1 && p.dgate != nullptr) {
#pragma unroll
                        for (int i = 0; i < P; ++i) u[i] = mul2(u[i], g[i]);
                        ln.store(p.dgate, at, u);
                    }
#pragma unroll
                    for (int i = 0; i < P; ++i) g[i] = mul2(g[i], gate.pair(i));
                }
                if (p.drop) ln.drop(keep, g);
                float2 q[POST ? P : 1];  // Norm(f)
                if constexpr (POST) {
                    ln.row_values(p.f, at, stage, 3, q);
                    const float2 s = both(st.y), c = both(-st.x);
#pragma unroll
                    for (int i = 0; i < P; ++i) q[i] = mul2(add2(q[i], c), s);
                }
                if constexpr (POST) {
                    float2 s3 = make_float2(0.0f, 0.0f), s4 = s3;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        if constexpr (SUMS) {
                            dpw[i] = fma2(g[i], q[i], dpw[i]);
                            dpb[i] = add2(dpb[i], g[i]);
                        }
                        g[i] = mul2(g[i], pw.pair(i));  // 0 past the row
                        s3 = add2(s3, g[i]);
                        s4 = fma2(g[i], q[i], s4);
                    }
                    s3 = ln.template row_sum<2>(make_float2(s3.x + s3.y, s4.x + s4.y));
                    const float2 s = both(st.y), m3 = both(p.layer ? -s3.x * p.inv_cols : 0.0f), m4 = both(-s3.y * p.inv_cols);
#pragma unroll
                    for (int i = 0; i < P; ++i) g[i] = mul2(s, add2(fma2(q[i], m4, g[i]), m3));
                }
                if (p.df != nullptr) ln.store(p.df, at, g);
            });
        if constexpr (GATE && SUMS && !OWN) {
            if (gate_sums && p.dgate != nullptr) {
                // whole segments are finished here; one that other units share
                // goes to the unit's first or last slot
                const bool whole = seg_lo == seg_gate * p.gate_period && seg_hi == (seg_gate + 1) * p.gate_period;
                float* slot = p.partial + (4 * static_cast<int64_t>(p.units) + 2 * unit + (seg_lo == unit_lo ? 0 : 1)) * p.cols;
                flush_columns<T, NV, VEC, NARROW>(ln, buf, dgt, slot, whole ? static_cast<T*>(p.dgate) + seg_gate * p.cols : nullptr);
            }
        }
        seg_lo = seg_hi;
        if constexpr (!VEC) {
            if (seg_lo < unit_hi) ln.group_sync();  // the segment's copies are read before the next one's begin
        }
    }
    if constexpr (SUMS) {
    const int64_t plane = static_cast<int64_t>(p.units) * p.cols;
    flush_columns<T, NV, VEC, NARROW>(ln, buf, dw, p.partial + unit * p.cols, nullptr);
    flush_columns<T, NV, VEC, NARROW>(ln, buf, db, p.partial + plane + unit * p.cols, nullptr);
    if constexpr (POST) {
        flush_columns<T, NV, VEC, NARROW>(ln, buf, dpw, p.partial + 2 * plane + unit * p.cols, nullptr);
        flush_columns<T, NV, VEC, NARROW>(ln, buf, dpb, p.partial + 3 * plane + unit * p.cols, nullptr);
    }
    }
}

// Column sums in a pass of their own: a thread takes 8 columns (aligned rows)
// or one over the rows of a unit, the next row's values on their way while one
// is added, and leaves partial sums, or finished gate rows, as the kernel above
// does.
constexpr int kPassThreads = 128;

template <typename T, bool VEC, bool POST, bool GATE>
__global__ void __launch_bounds__(kPassThreads, 4) residual_norm_column_pass_kernel(const RnParams p) {
    pdl_wait();
    constexpr int V = VEC ? 8 : 2;  // values held (one column uses the first)
    constexpr int P = V / 2;
    constexpr int STEP = VEC ? 8 : 1;
    using R = Raw<T, V>;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * kPassThreads + threadIdx.x) * STEP;
    if (c >= p.cols) return;
    const int64_t unit = blockIdx.y;
    const int64_t lo = unit_begin(unit, p.rows, p.units), hi = unit_begin(unit + 1, p.rows, p.units);
    auto load = [&](const void* tensor, int64_t at, R& w) {
        const T* src = static_cast<const T*>(tensor) + at + c;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w.vec(i, __ldg(reinterpret_cast<const uint4*>(src) + i));
        } else {
            w.set(0, src[0]);
            w.set(1, from_f<T>(0.0f));
        }
    };
    auto fill = [&](R& w, float v) {
#pragma unroll
        for (int i = 0; i < V; ++i) w.set(i, from_f<T>(v));
    };
    struct Row {
        R x, h, g, f;
        float4 st;
        float2 m;
    };
    auto fetch = [&](int64_t r, Row& w) {
        const int64_t at = r * p.cols;
        if (p.gh != nullptr) {
            load(p.x, at, w.x);
            load(p.gh, at, w.h);
            w.m = p.means[r];
        }
        if ((POST || GATE) && p.gx != nullptr) load(p.gx, at, w.g);
        load(p.f, at, w.f);
        w.st = p.stats[r];
    };
    R w, pw, pb, gate;
    fill(w, 1.0f);
    fill(pw, 1.0f);
    fill(pb, 0.0f);
    fill(gate, 1.0f);
    if (p.weight != nullptr) load(p.weight, 0, w);
    if (POST && p.post_weight != nullptr) load(p.post_weight, 0, pw);
    if (POST && p.post_bias != nullptr) load(p.post_bias, 0, pb);
    const float2 zero = make_float2(0.0f, 0.0f);
    float2 dw[P], db[P], dpw[POST ? P : 1], dpb[POST ? P : 1];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        dw[i] = db[i] = zero;
        if constexpr (POST) dpw[i] = dpb[i] = zero;
    }
    const bool gate_sums = GATE && p.gate_period > 1 && p.dgate != nullptr;
    const float2 a = both(p.a), drop_scale = both(p.drop ? p.dropout.scale : 1.0f);
    Row next;
    fill(next.x, 0.0f);
    fill(next.h, 0.0f);
    fill(next.g, 0.0f);
    next.m = zero;
    fetch(lo, next);
    int64_t seg_lo = lo;
    while (seg_lo < hi) {
        const int64_t gate_row = GATE ? seg_lo / p.gate_period : 0;
        const int64_t seg_hi = GATE ? min(hi, (gate_row + 1) * p.gate_period) : hi;
        float2 dgt[GATE ? P : 1];
        if constexpr (GATE) {
            load(p.gate, gate_row * p.cols, gate);
#pragma unroll
            for (int i = 0; i < P; ++i) dgt[i] = zero;
        }
        for (int64_t r = seg_lo; r < seg_hi; ++r) {
            const Row now = next;
            if (r + 1 < hi) fetch(r + 1, next);
            uint32_t keep = 0xFFu;
            if (p.drop) {
                const uint64_t e = static_cast<uint64_t>(r * p.cols + c);
                if constexpr (VEC) {
                    keep = dropout_keep8(p.dropout, static_cast<uint32_t>(e / 8));
                } else {
                    keep = dropout_keep4(p.dropout, static_cast<uint32_t>(e / 4)) >> (e & 3);
                }
            }
            const float2 q_c = both(-now.st.x), q_s = both(now.st.y), n_c = both(-now.st.z), n_s = both(now.st.w);
            const float2 m1 = both(-now.m.x), m2 = both(-now.m.y);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                float2 u = now.f.pair(i), q = zero;
                if constexpr (POST) {
                    q = mul2(add2(u, q_c), q_s);
                    u = fma2(q, pw.pair(i), pb.pair(i));
                }
                const bool k0 = (keep >> (2 * i)) & 1u, k1 = (keep >> (2 * i + 1)) & 1u;
                if (p.drop) {
                    u = mul2(u, drop_scale);
                    u = make_float2(k0 ? u.x : 0.0f, k1 ? u.y : 0.0f);
                }
                const float2 h = now.h.pair(i);
                float2 n = GATE ? mul2(u, gate.pair(i)) : u;
                n = mul2(add2(fma2(a, now.x.pair(i), n), n_c), n_s);
                dw[i] = fma2(h, n, dw[i]);
                db[i] = add2(db[i], h);
                if constexpr (POST || GATE) {
                    float2 g = fma2(add2(fma2(n, m2, mul2(h, w.pair(i))), m1), n_s, now.g.pair(i));
                    if constexpr (GATE) {
                        dgt[i] = fma2(g, u, dgt[i]);
                        g = mul2(g, gate.pair(i));
                    }
                    if constexpr (POST) {
                        if (p.drop) {
                            g = mul2(g, drop_scale);
                            g = make_float2(k0 ? g.x : 0.0f, k1 ? g.y : 0.0f);
                        }
                        dpw[i] = fma2(g, q, dpw[i]);
                        dpb[i] = add2(dpb[i], g);
                    }
                }
            }
        }
        if constexpr (GATE) {
            if (gate_sums) {
                const bool whole = seg_lo == gate_row * p.gate_period && seg_hi == (gate_row + 1) * p.gate_period;
                float* slot = p.partial + (4 * static_cast<int64_t>(p.units) + 2 * unit + (seg_lo == lo ? 0 : 1)) * p.cols + c;
#pragma unroll
                for (int i = 0; i < STEP; ++i) {
                    const float v = i % 2 ? dgt[i / 2].y : dgt[i / 2].x;
                    if (whole) {
                        static_cast<T*>(p.dgate)[gate_row * p.cols + c + i] = from_f<T>(v);
                    } else {
                        slot[i] = v;
                    }
                }
            }
        }
        seg_lo = seg_hi;
    }
    const int64_t plane = static_cast<int64_t>(p.units) * p.cols;
    float* out = p.partial + unit * p.cols + c;
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
        out[i] = i % 2 ? dw[i / 2].y : dw[i / 2].x;
        out[plane + i] = i % 2 ? db[i / 2].y : db[i / 2].x;
        if constexpr (POST) {
            out[2 * plane + i] = i % 2 ? dpw[i / 2].y : dpw[i / 2].x;
            out[3 * plane + i] = i % 2 ? dpb[i / 2].y : dpb[i / 2].x;
        }
    }
}

constexpr int kColLanes = 32;

// The units' partial sums added in a fixed order, rounded once.  The first
// `vectors` items are the parameter vectors asked for (plane[i] of the partial
// sums to out[i]), blockDim.y units at a time.  The others finish gate rows that
// several units share, `share` units at a time and blockDim.y / share gate rows
// per item: gate row g, or (by_unit, fewer units than gate rows) the gate row
// that unit g ends and unit g + 1 continues, for g below `gates`.
struct ColumnJobs {
    void* out[4];
    int plane[4];
    int vectors, col_blocks, share;
    int64_t gates;
    bool by_unit;
};

template <typename T>
__global__ void __launch_bounds__(1024) residual_norm_columns_kernel(const RnParams p, const __grid_constant__ ColumnJobs j) {
    pdl_wait();
    __shared__ float part[32][kColLanes + 1];
    const int item = static_cast<int>(blockIdx.x) / j.col_blocks;
    const int64_t c = static_cast<int64_t>(blockIdx.x - item * j.col_blocks) * kColLanes + threadIdx.x;
    const bool vector = item < j.vectors;
    const int share = vector ? static_cast<int>(blockDim.y) : j.share;
    const int sub = vector ? 0 : static_cast<int>(threadIdx.y) / share, y = static_cast<int>(threadIdx.y) - sub * share;
    float s = 0.0f;
    T* out = nullptr;  // none: nothing to finish
    if (vector) {
        out = static_cast<T*>(j.out[item]);
        if (c < p.cols) {
            const float* src = p.partial + static_cast<int64_t>(j.plane[item]) * p.units * p.cols + c;
#pragma unroll 4
            for (int u = y; u < p.units; u += share) s += src[static_cast<int64_t>(u) * p.cols];
        }
    } else {
        const int per = static_cast<int>(blockDim.y) / share;
        int64_t row = static_cast<int64_t>(item - j.vectors) * per + sub, first = 0, last = 0;
        if (sub < per && row < j.gates) {
            bool mine = true;
            if (j.by_unit) {
                const int64_t start = unit_begin(row + 1, p.rows, p.units);
                first = unit_of(start / p.gate_period * p.gate_period, p.rows, p.units);
                mine = start % p.gate_period != 0 && first == row;
                row = start / p.gate_period;
            } else {
                first = unit_of(row * p.gate_period, p.rows, p.units);
            }
            last = unit_of((row + 1) * p.gate_period - 1, p.rows, p.units);
            // else one unit held the row and finished it, or another item does
            if (mine && first != last) out = static_cast<T*>(p.dgate) + row * p.cols;
        }
        if (out != nullptr && c < p.cols) {
            const float* src = p.partial + 4 * static_cast<int64_t>(p.units) * p.cols + c;
#pragma unroll 4
            for (int64_t u = first + y; u <= last; u += share) {
                const int64_t slot = 2 * u + (unit_begin(u, p.rows, p.units) / p.gate_period == row ? 0 : 1);
                s += src[slot * p.cols];
            }
        }
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (y == 0 && out != nullptr && c < p.cols) {
        s = 0.0f;
        for (int i = 0; i < share; ++i) s += part[threadIdx.y + i][threadIdx.x];
        out[c] = from_f<T>(s);
    }
}

// ---- host ----------------------------------------------------------------------

// NV octets per thread, W warps per row and CTA, CTAs per row.  A warp's work
// for a row is about two octets' worth of sums and addresses and NV octets, so
// the least W * (2 + NV) is taken (8192 x 4096 with both norms, forward: NV 1
// 91 us, 2 58 us, 4 60 us).  Registers rule some out, at 128 for up to 512
// threads: NV 3 with a post norm spills 212 to 284 bytes (43690 x 768: 55.5 us,
// with NV 4 53.7; without one it spills 48 to 88 and stays, as fp32 NV 2 with one
// does at 64 to 256); the backward pass keeps two sums per column up to NV 2 (NV 3: 154
// against 93 us), five at NV 1 (NV 2: 198 against 153 us).  fp32 doubles the
// bytes of a row's copy: NV 1 (2331 x 1151 forward: 32 us, with NV 2 40 us),
// and forward 2 where that spares a cluster.
enum Pass { kForward, kSums2, kSums5, kNoSums };

struct Geometry {
    int nv, warps, cluster, lanes, groups;
    bool narrow() const { return lanes < 32; }
};

// Half a warp's columns: up to here the lanes of one warp take several rows
// (100000 x 64 in fp16: forward 57 -> 18 us, backward 75 -> 22; 400000 x 8: 214
// -> 9 and 284 -> 16; 100000 x 63 with a post norm: 139 -> 47 and 177 -> 58.
// Calls with too few rows to fill the GPU gain nothing: 75 x 64 the same, 75 x
// 63 5.0 -> 5.5 and 7.5 -> 8.1).
constexpr int kNarrowCols = 128;

Geometry geometry(int64_t cols, bool f16, Pass pass, bool post) {
    if (cols <= kNarrowCols) {
        int lanes = 1;
        while (lanes * 8 < cols) lanes *= 2;
        return {1, 1, 1, lanes, 256 / lanes};
    }
    Geometry best = {1, 1, 1, 32, 1};
    int64_t best_cost = INT64_MAX;
    const int nv_max = pass == kForward ? (f16 ? 4 : cols > 4096 ? 2 : 1) : pass == kSums5 || !f16 ? 1 : 2;
    for (int nv = nv_max; nv >= 1; --nv) {
        if (nv == 3 && post) continue;
        const int64_t per_warp = 256 * nv;
        const int max_warps = nv == 3 ? 8 : kMaxThreads / 32;
        const int64_t need = ceil_div(cols, per_warp);
        int cluster = 1;
        while (cluster * max_warps < need && cluster < kMaxCluster) cluster *= 2;
        const int64_t warps = ceil_div(need, cluster);
        if (warps > max_warps) continue;
        const int64_t cost = warps * cluster * (2 + nv) * (cluster > 1 ? 2 : 1);
        if (cost < best_cost) {
            best_cost = cost;
            best = {nv, static_cast<int>(warps), cluster, 32, 1};
        }
    }
    best.groups = best.cluster > 1 ? 1 : std::max(1, 8 / best.warps);
    return best;
}

using Kernel = void (*)(RnParams);

template <typename T, bool VEC>
Kernel forward_kernel(const Geometry& g, bool post) {
    if (g.narrow()) return post ? residual_norm_kernel<T, 1, VEC, true, true> : residual_norm_kernel<T, 1, VEC, false, true>;
    const int nv = g.nv;
    if constexpr (sizeof(T) == 2) {
        if (nv == 4) return post ? residual_norm_kernel<T, 4, VEC, true> : residual_norm_kernel<T, 4, VEC, false>;
        if (nv == 3) return residual_norm_kernel<T, 3, VEC, false>;
    }
    if (nv == 2) return post ? residual_norm_kernel<T, 2, VEC, true> : residual_norm_kernel<T, 2, VEC, false>;
    return post ? residual_norm_kernel<T, 1, VEC, true> : residual_norm_kernel<T, 1, VEC, false>;
}

template <typename T, int NV, bool VEC, bool SUMS, bool NARROW, Gate GATED>
Kernel backward_kernel_of(bool post) {
    return post ? residual_norm_backward_kernel<T, NV, VEC, true, GATED, SUMS, NARROW> : residual_norm_backward_kernel<T, NV, VEC, false, GATED, SUMS, NARROW>;
}

template <typename T, int NV, bool VEC, bool SUMS, bool NARROW = false>
Kernel backward_kernel_of(bool post, Gate gate) {
    if constexpr (SUMS) {
        if (gate == kGateOwn) return backward_kernel_of<T, NV, VEC, SUMS, NARROW, kGateOwn>(post);
    }
    return gate != kNoGate ? backward_kernel_of<T, NV, VEC, SUMS, NARROW, kGate>(post) : backward_kernel_of<T, NV, VEC, SUMS, NARROW, kNoGate>(post);
}

template <typename T, bool VEC>
Kernel backward_kernel(const Geometry& g, bool post, Gate gate, bool sums) {
    if (g.narrow()) return backward_kernel_of<T, 1, VEC, true, true>(post, gate);  // never without sums
    if constexpr (sizeof(T) == 2) {
        if (g.nv == 2) return sums ? residual_norm_backward_kernel<T, 2, VEC, false, kNoGate, true> : backward_kernel_of<T, 2, VEC, false>(post, gate);
    }
    return sums ? backward_kernel_of<T, 1, VEC, true>(post, gate) : backward_kernel_of<T, 1, VEC, false>(post, gate);
}

template <typename T>
Kernel backward_kernel(const Geometry& g, bool vec, bool post, Gate gate, bool sums) {
    return vec ? backward_kernel<T, true>(g, post, gate, sums) : backward_kernel<T, false>(g, post, gate, sums);
}

template <typename T, bool VEC>
Kernel column_pass_of(bool post, bool gate) {
    if (post) return gate ? residual_norm_column_pass_kernel<T, VEC, true, true> : residual_norm_column_pass_kernel<T, VEC, true, false>;
    return gate ? residual_norm_column_pass_kernel<T, VEC, false, true> : residual_norm_column_pass_kernel<T, VEC, false, false>;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const char* who, const tk_residual_norm_desc_t& d) {
    TK_CHECK_ARG(d.dtype == TK_DTYPE_F16 || d.dtype == TK_DTYPE_F32, "%s: bad dtype %d", who, static_cast<int>(d.dtype));
    TK_CHECK_ARG(d.norm == TK_NORM_LAYER || d.norm == TK_NORM_RMS, "%s: bad norm %d", who, static_cast<int>(d.norm));
    TK_CHECK_ARG(d.rows >= 0 && d.cols >= 1, "%s: rows must not be negative and cols must be positive", who);
    if (d.cols > kMaxCols) TK_FAIL(TK_ERR_UNSUPPORTED, "%s: at most %lld columns, got %lld", who, static_cast<long long>(kMaxCols), static_cast<long long>(d.cols));
    TK_CHECK_ARG(d.rows <= INT64_MAX / 8 / d.cols, "%s: too many elements", who);
    TK_CHECK_ARG(d.p >= 0.0 && d.p <= 1.0, "%s: p must be in [0, 1], got %g", who, d.p);
    if (d.p > 0.0 && d.rows * d.cols >= (1ll << 34)) TK_FAIL(TK_ERR_UNSUPPORTED, "%s: dropout of 2^34 elements or more", who);
    TK_CHECK_ARG(d.post_norm || (d.post_weight == nullptr && d.post_bias == nullptr), "%s: post_weight and post_bias need post_norm", who);
    // no rows: a gate for each sample of an empty batch has none either
    TK_CHECK_ARG(d.gate == nullptr || (d.gate_rows >= 1 && d.rows % d.gate_rows == 0) || (d.gate_rows == 0 && d.rows == 0), "%s: gate_rows must divide rows", who);
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
constexpr int kSmemMost = 227 * 1024;

size_t stage_bytes(const Geometry& g, bool f16, bool vec, int tensors) {
    const size_t row = static_cast<size_t>(g.warps) * g.lanes * g.nv * (f16 ? 16 : 32);
    return (row + (vec ? 0 : kTailPad)) * g.groups * tensors;
}

// The launch's shape and its dynamic shared memory: a ring of three rows per
// group (two in flight while one is used) where that leaves room for the CTAs
// that the registers admit, fewer rows otherwise.
size_t configure(RnParams& p, const Geometry& g, bool f16, bool vec, int tensors, bool backward) {
    p.cluster = g.cluster;
    p.warps = g.warps;
    p.lanes = g.lanes;
    p.groups = g.groups;
    const size_t one = stage_bytes(g, f16, vec, tensors);
    const size_t fold = backward && g.groups > 1 ? static_cast<size_t>(g.warps) * g.lanes * g.groups * 8 * g.nv * sizeof(float) : 0;
    const int resident = std::max(1, 512 / (g.warps * g.lanes * g.groups));  // CTAs that registers admit
    p.stages = 3;
    while (p.stages > (vec ? 1 : 2) && (red_bytes(g) + p.stages * one + 1024) * resident > kSmemPerSm) --p.stages;
    return red_bytes(g) + std::max(p.stages * one, fold);
}

int launch(Kernel k, const RnParams& p, size_t smem, cudaStream_t s, const char* what) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.units) * p.cluster);
    cfg.blockDim = dim3(p.warps * p.lanes * p.groups);
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
    TK_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
    TK_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, reinterpret_cast<const void*>(k), p.warps * p.lanes * p.groups, smem));
    if (per_sm < 1) TK_FAIL(TK_ERR_CUDA, "residual norm: the kernel does not fit an SM");
    return TK_OK;
}

// Whether groups take whole gate rows: by the rows that one group works off in
// turn, where the groups of a CTA that share a gate row add up its gradient in
// about the time of two rows (samples x tokens x columns, backward and column
// sums: 20000 x 3 x 64 in fp16 155 -> 18 us, 50000 x 2 x 8 537 -> 13, 4000 x 25 x
// 64 52 -> 37, 2000 x 8 x 200 59 -> 18; 3000 x 40 x 128 in fp32 127 -> 131).
bool whole_gate_rows(const RnParams& p, const Geometry& g, int64_t resident) {
    if (g.groups == 1 || p.gate_period > INT32_MAX) return false;
    const int64_t gates = p.rows / p.gate_period;
    const int64_t own = ceil_div(gates, std::min(resident, ceil_div(gates, g.groups)) * g.groups) * p.gate_period;
    const int64_t units = std::min(resident, ceil_div(p.rows, g.groups));
    const int64_t shared = ceil_div(gates, units) * (ceil_div(std::min(p.gate_period, ceil_div(p.rows, units)), g.groups) + 2);
    return own <= shared;
}

// CTAs per SM the backward pass may use: its partial sums are sized by it.
constexpr int kBackwardPerSm = 4;

// Rows that one CTA cannot hold together with their column sums.
bool is_wide(const tk_residual_norm_desc_t& d) {
    const bool sums5 = d.post_norm != 0 || d.gate != nullptr;
    return d.cols > (sums5 || d.dtype == TK_DTYPE_F32 ? 1 : 2) * 256 * (kMaxThreads / 32);
}

// Row ranges of the column pass: one resident wave of four blocks per SM.
int column_units(int device, int64_t rows, int64_t cols, bool vec) {
    const int64_t blocks = ceil_div(cols, kPassThreads * (vec ? 8 : 1));
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, 4 * sm_count(device) / blocks)));
}

template <typename T>
int columns(const RnParams& p, const tk_residual_norm_grad_desc_t& g, bool gate_items, cudaStream_t s) {
    ColumnJobs j = {};
    void* const outs[4] = {g.dweight, g.dbias, g.dpost_weight, g.dpost_bias};
    for (int i = 0; i < 4; ++i) {
        if (outs[i] == nullptr || (i >= 2 && !g.fwd.post_norm)) continue;
        j.out[j.vectors] = outs[i];
        j.plane[j.vectors++] = i;
    }
    j.col_blocks = static_cast<int>(ceil_div(p.cols, kColLanes));
    const int64_t gates = p.rows / p.gate_period;
    j.by_unit = gate_items && gates > p.units;
    j.gates = !gate_items ? 0 : j.by_unit ? p.units - 1 : gates;
    const int rows = std::max(1, std::min(32, (p.units + 3) / 4));  // about four partial sums per thread
    // and two of a gate row (a block for each gate row: 300 of 30 x 256 took 42
    // us, now 5, 4000 of 100 x 64 13, now 5; 7 of 333 x 1151 8.4, now 9.2)
    j.share = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, (p.units / gates + 2 + 1) / 2)));
    const int items = j.vectors + static_cast<int>(ceil_div(j.gates, rows / j.share));
    if (items == 0) return TK_OK;
    cudaError_t e = launch_pdl(residual_norm_columns_kernel<T>, dim3(static_cast<unsigned>(items) * j.col_blocks), dim3(kColLanes, rows), 0, s, p, j);
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
    const Geometry g = geometry(p.cols, f16, kForward, d.post_norm != 0);
    const size_t smem = configure(p, g, f16, vec, 2, false);
    const Kernel k = f16 ? (vec ? forward_kernel<__half, true>(g, d.post_norm) : forward_kernel<__half, false>(g, d.post_norm))
                         : (vec ? forward_kernel<float, true>(g, d.post_norm) : forward_kernel<float, false>(g, d.post_norm));
    int per_sm = 0;
    if (int rc = resident_ctas(k, p, smem, per_sm)) return rc;
    p.units = max_units(current_device(), p.rows, g, per_sm);
    return launch(k, p, smem, static_cast<cudaStream_t>(stream), "residual_norm");
}

size_t tk_residual_norm_backward_workspace_size(const tk_residual_norm_grad_desc_t* desc) {
    using namespace tk;
    if (desc == nullptr || check("tk_residual_norm_backward", desc->fwd) != TK_OK) return 0;
    // [4 + 2][units][cols] fp32 partial sums, `units` at its largest, and two
    // means per row where a pass of its own adds the columns
    const tk_residual_norm_desc_t& d = desc->fwd;
    const int device = current_device();
    const int64_t units = is_wide(d) ? column_units(device, std::max<int64_t>(1, d.rows), d.cols, true)
                                     : std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(sm_count(device)) * kBackwardPerSm, d.rows));
    return static_cast<size_t>(6 * units * d.cols) * sizeof(float) + (is_wide(d) ? round_up(static_cast<size_t>(d.rows) * sizeof(float2), 16) : 0) + 256;
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
    TK_CHECK_ARG(d.post_norm || (!desc->dpost_weight && !desc->dpost_bias), "tk_residual_norm_backward: dpost_weight and dpost_bias need post_norm");
    TK_CHECK_ARG(d.gate || !desc->dgate, "tk_residual_norm_backward: dgate without a gate");
    TK_CHECK_ARG(d.x && d.f && d.stats && aligned16(d.stats), "tk_residual_norm_backward: x, f and 16-byte aligned stats are needed");
    TK_CHECK_ARG(desc->grad_x_new || desc->grad_h, "tk_residual_norm_backward: no incoming gradient");
    RnParams p = params(d);
    p.x_new = nullptr;
    p.h = nullptr;
    p.bias = nullptr;
    p.gx = desc->grad_x_new;
    p.gh = desc->grad_h;
    p.dx = desc->dx;
    p.df = desc->df;
    p.dgate = d.gate != nullptr ? desc->dgate : nullptr;
    const bool gate = d.gate != nullptr, post = d.post_norm != 0;
    const bool vec = vectorised(p);
    const bool wide = is_wide(d);
    const Geometry g = geometry(p.cols, f16, wide ? kNoSums : gate || post ? kSums5 : kSums2, post);
    const size_t smem = configure(p, g, f16, vec, 4, !wide);
    Gate gated = gate ? kGate : kNoGate;
    const auto pick = [&] { return f16 ? backward_kernel<__half>(g, vec, post, gated, !wide) : backward_kernel<float>(g, vec, post, gated, !wide); };
    Kernel k = pick();
    int per_sm = 0;
    if (int rc = resident_ctas(k, p, smem, per_sm)) return rc;
    p.units = max_units(current_device(), p.rows, g, std::min(per_sm, kBackwardPerSm));
    if (!wide && p.dgate != nullptr && p.gate_period > 1 &&
        whole_gate_rows(p, g, static_cast<int64_t>(sm_count(current_device())) * std::min(per_sm, kBackwardPerSm) / g.cluster)) {
        gated = kGateOwn;
        k = pick();
        if (int rc = resident_ctas(k, p, smem, per_sm)) return rc;
        p.units = max_units(current_device(), p.rows / p.gate_period, g, std::min(per_sm, kBackwardPerSm));
    }
    const int pass_units = column_units(current_device(), p.rows, p.cols, vec);
    const size_t means = wide ? round_up(static_cast<size_t>(p.rows) * sizeof(float2), 16) : 0;
    const size_t need = means + static_cast<size_t>(6) * (wide ? pass_units : p.units) * p.cols * sizeof(float);
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
        TK_FAIL(TK_ERR_WORKSPACE, "tk_residual_norm_backward: 16-byte aligned workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    p.means = static_cast<float2*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + means);
    if (int rc = launch(k, p, smem, s, "residual_norm_backward")) return rc;
    const bool sums = desc->dweight || desc->dbias || desc->dpost_weight || desc->dpost_bias || (p.dgate != nullptr && p.gate_period > 1);
    if (wide && sums) {
        p.units = pass_units;
        const Kernel pass = f16 ? (vec ? column_pass_of<__half, true>(post, gate) : column_pass_of<__half, false>(post, gate))
                                : (vec ? column_pass_of<float, true>(post, gate) : column_pass_of<float, false>(post, gate));
        const cudaError_t e = launch_pdl(pass, dim3(static_cast<unsigned>(ceil_div(p.cols, kPassThreads * (vec ? 8 : 1))), p.units), dim3(kPassThreads), 0, s, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            TK_FAIL(TK_ERR_CUDA, "residual norm column pass launch failed: %s", cudaGetErrorString(e));
        }
    }
    const bool gate_items = p.dgate != nullptr && p.gate_period > 1 && gated != kGateOwn;
    return f16 ? columns<__half>(p, *desc, gate_items, s) : columns<float>(p, *desc, gate_items, s);
}

}  // extern "C"
