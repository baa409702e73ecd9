// cross_entropy.cu -- softmax cross entropy of a linear layer over a large
// vocabulary, without its logits, and the gradients.
//
//   z = x W^T + b;  loss_i = logsumexp(z_i) - z_i[t_i]
//   dz_i = g_i (softmax(z_i) - onehot(t_i));  dx = dz W;  dW = dz^T x;  db = sum_i dz_i
//
// Rows whose target is ignore_index are dropped before any product: a scan
// lists the others, their rows of x are packed, and every later kernel takes
// its row count from that list on the device.
//
// Forward: one tcgen05 GEMM whose epilogue keeps, per row and 128 columns,
// the maximum and the sum of exponentials (base 2); a small kernel joins them
// and computes the target's logit as a dot product of its own.  Backward: the
// vocabulary is taken in pieces whose dz fits a workspace; per piece the
// logits are computed again, the epilogue stores dz as binary16, and two
// GEMMs read it in place (dz and x^T / W^T in MN-major shared-memory tiles, so
// nothing is transposed).
//
// binary16 dz: softmax - onehot lies in [-1, 1]; rows are scaled by g_i / max
// |g| and 2^14, so values down to 2^-28 of the largest gradient keep all 11
// bits and the rest lose at most 2^-39 of it.  The scale is taken out again
// in binary32 when dx and dW are rounded.
//
// fp32 operands are split into two binary16 planes of a power-of-two multiple
// (hi = rn(v s), lo = rn(v s - hi), the tensor's largest value in [2^14,
// 2^15)), 22 bits or 2^-40 of the largest value, and a product is the sum
// hi*hi + hi*lo + lo*hi: the K loop runs over three pairs of planes.
//
// GEMM kernel (one persistent CTA per SM, 320 threads): warp 0 loads 64-deep
// stages by TMA (128-byte swizzle), warp 1 issues tcgen05.mma kind::f16 into
// two 256-column accumulators in TMEM, warps 2..9 run the epilogue of one
// while the other fills.  Tiles are 128 x 256.
#include <cuda_fp16.h>

#include <algorithm>

#include "tk_internal.h"
#include "tk_ptx.cuh"

namespace tk {
namespace {

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int GEMM_SMEM = STAGES * STAGE_BYTES + 1024 + 256;
constexpr int TMEM_COLS = 512;
static_assert(GEMM_SMEM <= 232448, "shared memory budget");

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kDzScale = 16384.0f;
constexpr int kRowPad = 256;  // packed rows are zero up to a multiple of this

// Device scalars of one call.
struct Scalars {
    int count;           // rows with a target
    unsigned amax_x;     // binary32 bits of the largest finite |x|, |W| (fp32 operands)
    unsigned amax_w;
    float z_log2;        // accumulator -> base-2 logit
    float gmax;          // max |g_i|
    float dx_scale, dw_scale, db_scale;  // accumulators -> gradients
};

enum Epilogue { kStats, kDlogits, kGradX, kGradW };

struct GemmParams {
    const Scalars* sc;
    int n_tiles;
    int m_tiles;   // < 0: from sc->count
    int k_blocks;  // per pair of planes; < 0: from sc->count
    int pairs;     // 1 (fp16 operands) or 3 (two planes each)
    int max_units; // tiles x K splits the workspace of a split reduction holds
    int group;     // M tiles that neighbouring CTAs share
    unsigned* err;
    // kStats / kDlogits
    const float* bias2;  // bias * log2(e), or NULL
    int64_t vocab0, vocab;  // the piece's first column, all columns
    float2* part;           // [2 * n_tiles][rows_pad] maximum and sum
    int64_t rows_pad;
    const float* lse2;
    const float* grow;   // g_i / max |g|
    const int* target;
    __half* dz;          // [planes][rows_pad][dz_ld]
    int64_t dz_ld, dz_plane;
    // kGradX / kGradW
    void* out;
    const int* index;    // kGradX: output row of a packed row
    int64_t out_rows, out_cols;
    int out_f32, out_vec;
    float* acc;          // [rows_pad][out_cols] sums over earlier pieces
    int first, last;     // piece (kGradX)
    float* split;        // [max_units][BM][BN] partial tiles
};

// Split of the K loop into chunks that fill the GPU when tiles are few: at
// least eight blocks per chunk, tiles * splits within max_units.
__device__ __forceinline__ int k_splits(const GemmParams& p, int tiles, int blocks) {
    if (tiles <= 0) return 1;
    return max(1, min(p.max_units / tiles, blocks / 8));
}

struct Shape {
    int m_tiles, blocks, splits, units;
};
template <int EPI>
__device__ __forceinline__ Shape shape_of(const GemmParams& p) {
    const int count = p.sc->count;
    Shape s;
    s.m_tiles = p.m_tiles >= 0 ? p.m_tiles : (count + BM - 1) / BM;
    s.blocks = (p.k_blocks >= 0 ? p.k_blocks : (count + BK - 1) / BK) * p.pairs;
    s.splits = EPI == kGradX || EPI == kGradW ? k_splits(p, s.m_tiles * p.n_tiles, s.blocks) : 1;
    s.units = s.m_tiles * p.n_tiles * s.splits;
    return s;
}

// Work unit -> (K chunk, M tile, N tile); the chunk varies slowest, tiles run
// in groups of p.group M tiles so neighbours share operands in L2.
__device__ __forceinline__ void decode_unit(const GemmParams& p, const Shape& s, int u, int& mt, int& nt, int& ks) {
    const int tiles = s.m_tiles * p.n_tiles;
    ks = u / tiles;
    u -= ks * tiles;
    const int width = p.group * p.n_tiles;
    const int g = u / width;
    const int first = g * p.group;
    const int size = min(s.m_tiles - first, p.group);
    const int r = u - g * width;
    mt = first + r % size;
    nt = r / size;
}

__device__ __forceinline__ void tc_mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptor of an MN-major tile written by TMA with 128-byte swizzling: boxes
// of 64 M/N elements (128 bytes) by 64 K rows, 8 KB apart along M/N (leading
// byte offset), 8-row swizzle atoms 1 KB apart along K (stride byte offset).
__device__ __forceinline__ uint64_t smem_desc_mnmajor_sw128(uint32_t saddr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((BK * 128) >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// kind::f16 with binary16 operands and binary32 accumulators: D format F32 (1)
// at bit 4, A and B formats F16 (0), A / B MN-major at bits 15 / 16, N >> 3 at
// bit 17, M >> 4 at bit 24.
constexpr uint32_t idesc_f16(int m, int n, bool a_mn, bool b_mn) {
    return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ float exp2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 consecutive columns of one row: base-2 logits from the accumulators.
__device__ __forceinline__ void logits2(const uint32_t (&acc)[32], float k, const float* bias2, int64_t col, int64_t vocab, float (&y)[32]) {
    if (bias2 != nullptr) {
        if (col + 32 <= vocab) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 b = __ldg(reinterpret_cast<const float4*>(bias2 + col + i));
                y[i] = fmaf(__uint_as_float(acc[i]), k, b.x);
                y[i + 1] = fmaf(__uint_as_float(acc[i + 1]), k, b.y);
                y[i + 2] = fmaf(__uint_as_float(acc[i + 2]), k, b.z);
                y[i + 3] = fmaf(__uint_as_float(acc[i + 3]), k, b.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = col + i < vocab ? fmaf(__uint_as_float(acc[i]), k, __ldg(bias2 + col + i)) : -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(acc[i]) * k;
        if (col + 32 > vocab) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i >= vocab) y[i] = -INFINITY;
        }
    }
}

// Joins two (maximum, sum) pairs of base-2 exponentials.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    const float ref = top == -INFINITY ? 0.0f : top;
    s = s * exp2_sfu(m - ref) + s2 * exp2_sfu(m2 - ref);
    m = top;
}

__device__ __forceinline__ void store_out(const GemmParams& p, int64_t row, int64_t col, const float (&v)[32]) {
    if (p.out_f32) {
        float* o = static_cast<float*>(p.out) + row * p.out_cols + col;
        if (p.out_vec) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                if (col + i < p.out_cols) *reinterpret_cast<float4*>(o + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i < p.out_cols) o[i] = v[i];
        }
    } else {
        __half* o = static_cast<__half*>(p.out) + row * p.out_cols + col;
        if (p.out_vec) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
                if (col + i < p.out_cols)
                    *reinterpret_cast<uint4*>(o + i) = make_uint4(half2_bits(v[i], v[i + 1]), half2_bits(v[i + 2], v[i + 3]),
                                                                  half2_bits(v[i + 4], v[i + 5]), half2_bits(v[i + 6], v[i + 7]));
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i < p.out_cols) o[i] = __float2half_rn(v[i]);
        }
    }
}

// A finished chunk of 32 columns of a gradient tile: joined with the earlier
// pieces' sum, kept for the next piece or rounded and stored.
template <int EPI>
__device__ __forceinline__ void finish_grad(const GemmParams& p, int64_t m, int64_t rows, int64_t col, float scale, float (&v)[32]) {
    if (m >= rows || col >= p.out_cols) return;
    if (EPI == kGradX && !(p.first && p.last)) {
        float* a = p.acc + m * p.out_cols + col;
        if (!p.first) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i < p.out_cols) v[i] += a[i];
        }
        if (!p.last) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i < p.out_cols) a[i] = v[i];
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= scale;
    store_out(p, EPI == kGradX ? p.index[m] : m, col, v);
}

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1)
ce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmParams p) {
    constexpr bool A_MN = EPI == kGradW, B_MN = EPI == kGradX || EPI == kGradW;
    constexpr uint32_t IDESC = idesc_f16(BM, BN, A_MN, B_MN);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
    uint64_t* full_bar = bars;               // [STAGES] TMA -> MMA
    uint64_t* empty_bar = bars + STAGES;     // [STAGES] MMA -> TMA
    uint64_t* acc_full = bars + 2 * STAGES;  // [2] MMA -> epilogue
    uint64_t* acc_empty = acc_full + 2;      // [2] epilogue -> MMA
    uint64_t* drain_bar = acc_empty + 2;     // MMA teardown
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(full_bar + s), 1);
            mbar_init(smem_u32(empty_bar + s), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(acc_full + i), 1);
            mbar_init(smem_u32(acc_empty + i), EPI_WARPS);
        }
        mbar_init(smem_u32(drain_bar), 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    const Shape sh = shape_of<EPI>(p);

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        int stage = 0;
        uint32_t phase = 0;
        uint32_t last_phase[STAGES];
        bool used[STAGES];
        for (int s = 0; s < STAGES; ++s) {
            used[s] = false;
            last_phase[s] = 0;
        }
        const int per_pair = sh.blocks / p.pairs;
        bool ok = true;
        for (int u = blockIdx.x; u < sh.units && ok; u += gridDim.x) {
            int mt, nt, ks;
            decode_unit(p, sh, u, mt, nt, ks);
            const int kb1 = static_cast<int>(static_cast<int64_t>(ks + 1) * sh.blocks / sh.splits);
            for (int kb = static_cast<int>(static_cast<int64_t>(ks) * sh.blocks / sh.splits); kb < kb1; ++kb) {
                if (!mbar_wait_bounded(smem_u32(empty_bar + stage), phase ^ 1u, abort_flag, p.err, kDevErrWaitEmpty)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    const int pair = kb / per_pair;
                    const int kx = (kb - pair * per_pair) * BK;
                    const int pa = pair == 2 ? 1 : 0, pb = pair == 1 ? 1 : 0;
                    const uint32_t fb = smem_u32(full_bar + stage);
                    const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES);
                    mbar_arrive_expect_tx(fb, STAGE_BYTES);
                    if constexpr (A_MN) {
#pragma unroll
                        for (int i = 0; i < BM / 64; ++i) tma_load_3d(sa + i * BK * 128, &tmA, fb, mt * BM + i * 64, kx, pa);
                    } else {
                        tma_load_3d(sa, &tmA, fb, kx, mt * BM, pa);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int i = 0; i < BN / 64; ++i) tma_load_3d(sa + A_BYTES + i * BK * 128, &tmB, fb, nt * BN + i * 64, kx, pb);
                    } else {
                        tma_load_3d(sa + A_BYTES, &tmB, fb, kx, nt * BN, pb);
                    }
                }
                __syncwarp();
                used[stage] = true;
                last_phase[stage] = phase;
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        // Drain: every box this warp issued has landed before the CTA exits.
        for (int s = 0; s < STAGES; ++s) {
            if (used[s]) {
                volatile int no_abort = 0;
                mbar_wait_bounded(smem_u32(full_bar + s), last_phase[s], &no_abort, p.err, kDevErrWaitDrain);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        int local = 0;
        for (int u = blockIdx.x; u < sh.units && ok; u += gridDim.x, ++local) {
            const int buf = local & 1;
            if (!mbar_wait_bounded(smem_u32(acc_empty + buf), ((local >> 1) & 1) ^ 1u, abort_flag, p.err, kDevErrWaitAccEmpty)) break;
            tc_fence_after();
            const uint32_t acc = tmem_base + buf * BN;
            int mt, nt, ks;
            decode_unit(p, sh, u, mt, nt, ks);
            const int kb0 = static_cast<int>(static_cast<int64_t>(ks) * sh.blocks / sh.splits);
            const int kb1 = static_cast<int>(static_cast<int64_t>(ks + 1) * sh.blocks / sh.splits);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(smem_u32(full_bar + stage), phase, abort_flag, p.err, kDevErrWaitFull)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES);
                    const uint64_t da = A_MN ? smem_desc_mnmajor_sw128(sa) : smem_desc_kmajor_sw128(sa);
                    const uint64_t db = B_MN ? smem_desc_mnmajor_sw128(sa + A_BYTES) : smem_desc_kmajor_sw128(sa + A_BYTES);
                    // 16 K values on: 32 bytes inside the swizzled row of a
                    // K-major tile, two 1 KB atoms of an MN-major one
                    constexpr uint64_t step_a = (A_MN ? 2048 : 32) >> 4, step_b = (B_MN ? 2048 : 32) >> 4;
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk)
                        tc_mma_f16(acc, da + kk * step_a, db + kk * step_b, IDESC, kb > kb0 || kk > 0 ? 1u : 0u);
                    tc_commit(smem_u32(empty_bar + stage));
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) break;
            if (lane == 0) tc_commit(smem_u32(acc_full + buf));
            __syncwarp();
        }
        // Drain: all MMAs of this thread complete before TMEM is freed.
        if (lane == 0) tc_commit(smem_u32(drain_bar));
        __syncwarp();
        volatile int no_abort = 0;
        mbar_wait_bounded(smem_u32(drain_bar), 0, &no_abort, p.err, kDevErrWaitDrain);
    } else {
        // ---------------- epilogue (warps 2..9) ----------------
        // A warp reads TMEM lanes [32 * (warp % 4), + 32), one row per lane,
        // and half of the tile's columns.
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int rows = p.sc->count;
        float scale = 1.0f;
        if constexpr (EPI == kStats || EPI == kDlogits) scale = p.sc->z_log2;
        if constexpr (EPI == kGradX) scale = p.sc->dx_scale;
        if constexpr (EPI == kGradW) scale = p.sc->dw_scale;
        int local = 0;
        for (int u = blockIdx.x; u < sh.units; u += gridDim.x, ++local) {
            int mt, nt, ks;
            decode_unit(p, sh, u, mt, nt, ks);
            const int buf = local & 1;
            if (!mbar_wait_bounded(smem_u32(acc_full + buf), (local >> 1) & 1, abort_flag, p.err, kDevErrWaitAccFull)) break;
            tc_fence_after();
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * BN + half * (BN / 2);
            const int64_t m = static_cast<int64_t>(mt) * BM + quarter * 32 + lane;
            const int64_t col0 = static_cast<int64_t>(nt) * BN + half * (BN / 2);
            if constexpr (EPI == kStats) {
                float top = -INFINITY, sum = 0.0f;
#pragma unroll 1
                for (int c = 0; c < BN / 2; c += 32) {
                    uint32_t acc[32];
                    float y[32];
                    tmem_ld_32x32b_x32(t0 + c, acc);
                    tc_wait_ld();
                    logits2(acc, scale, p.bias2, col0 + c, p.vocab, y);
                    float cm = y[0];
#pragma unroll
                    for (int i = 1; i < 32; ++i) cm = fmaxf(cm, y[i]);
                    const float ref = cm == -INFINITY ? 0.0f : cm;
                    float cs = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) cs += exp2_sfu(y[i] - ref);
                    join(top, sum, cm, cs);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(acc_empty + buf));
                p.part[(static_cast<int64_t>(nt) * 2 + half) * p.rows_pad + m] = make_float2(top, sum);
            } else if constexpr (EPI == kDlogits) {
                const bool live = m < rows;
                const float lse = live ? p.lse2[m] : 0.0f;
                const float g = live ? p.grow[m] * kDzScale : 0.0f;
                const int64_t hit = live ? p.target[m] - p.vocab0 : -1;
#pragma unroll 1
                for (int c = 0; c < BN / 2; c += 32) {
                    uint32_t acc[32];
                    float y[32];
                    tmem_ld_32x32b_x32(t0 + c, acc);
                    tc_wait_ld();
                    const int64_t col = col0 + c;
                    logits2(acc, scale, p.bias2, p.vocab0 + col, p.vocab, y);
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = live ? exp2_sfu(y[i] - lse) * g : 0.0f;
                    if (hit >= col && hit < col + 32) {
                        const int j = static_cast<int>(hit - col);
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] -= i == j ? g : 0.0f;
                    }
                    __half* o = p.dz + m * p.dz_ld + col;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        const uint4 hi = make_uint4(half2_bits(y[i], y[i + 1]), half2_bits(y[i + 2], y[i + 3]),
                                                    half2_bits(y[i + 4], y[i + 5]), half2_bits(y[i + 6], y[i + 7]));
                        *reinterpret_cast<uint4*>(o + i) = hi;
                        if (p.dz_plane != 0) {
                            const __half2* h = reinterpret_cast<const __half2*>(&hi);
                            uint32_t lo[4];
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const float2 f = __half22float2(h[t]);
                                lo[t] = half2_bits(y[i + 2 * t] - f.x, y[i + 2 * t + 1] - f.y);
                            }
                            *reinterpret_cast<uint4*>(o + p.dz_plane + i) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(acc_empty + buf));
            } else {
                const bool some = static_cast<int64_t>(ks + 1) * sh.blocks / sh.splits > static_cast<int64_t>(ks) * sh.blocks / sh.splits;
                const int64_t limit = EPI == kGradX ? rows : p.out_rows;
#pragma unroll 1
                for (int c = 0; c < BN / 2; c += 32) {
                    uint32_t acc[32];
                    float v[32];
                    tmem_ld_32x32b_x32(t0 + c, acc);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = some ? __uint_as_float(acc[i]) : 0.0f;
                    if (sh.splits > 1) {
                        float* t = p.split + (static_cast<int64_t>(u) * BM + quarter * 32 + lane) * BN + half * (BN / 2) + c;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(t + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    } else {
                        finish_grad<EPI>(p, m, limit, col0 + c, scale, v);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(acc_empty + buf));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// Adds the K chunks of split tiles in their order.  One block per 8 rows of a
// tile, 8 threads of 32 columns per row.
template <int EPI>
__global__ void __launch_bounds__(64) ce_split_kernel(const GemmParams p) {
    pdl_wait();
    const Shape sh = shape_of<EPI>(p);
    if (sh.splits <= 1) return;
    const int tiles = sh.m_tiles * p.n_tiles;
    const int64_t limit = EPI == kGradX ? p.sc->count : p.out_rows;
    const float scale = EPI == kGradX ? p.sc->dx_scale : p.sc->dw_scale;
    for (int b = blockIdx.x; b < tiles * (BM / 8); b += gridDim.x) {
        const int tile = b / (BM / 8);
        const int row = (b % (BM / 8)) * 8 + static_cast<int>(threadIdx.x) / 8;
        const int c = static_cast<int>(threadIdx.x % 8) * 32;
        int mt, nt, ks;
        decode_unit(p, sh, tile, mt, nt, ks);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.0f;
        for (int k = 0; k < sh.splits; ++k) {
            const float4* t = reinterpret_cast<const float4*>(p.split + ((static_cast<int64_t>(k) * tiles + tile) * BM + row) * BN + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 f = t[i];
                v[4 * i] += f.x;
                v[4 * i + 1] += f.y;
                v[4 * i + 2] += f.z;
                v[4 * i + 3] += f.w;
            }
        }
        finish_grad<EPI>(p, static_cast<int64_t>(mt) * BM + row, limit, static_cast<int64_t>(nt) * BN + c, scale, v);
    }
}

// ---- small kernels ---------------------------------------------------------------

__device__ __forceinline__ float load_f(const __half* p, int64_t i) { return __half2float(p[i]); }
__device__ __forceinline__ float load_f(const float* p, int64_t i) { return p[i]; }

constexpr int kIndexThreads = 1024;

// Lists the rows that have a target (in order), their targets, and their
// count; writes the ignored rows' losses (0) where there is one per row.
__global__ void __launch_bounds__(kIndexThreads)
ce_index_kernel(const int64_t* target, int64_t rows, int64_t vocab, int64_t ignore, int* index, int* packed_target, Scalars* sc,
                float* row_loss_out) {
    __shared__ int warp_sum[32];
    __shared__ int total;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int base = 0;
    for (int64_t r0 = 0; r0 < rows; r0 += kIndexThreads) {
        const int64_t r = r0 + threadIdx.x;
        const int64_t t = r < rows ? target[r] : ignore;
        const bool used = r < rows && t != ignore;
        const unsigned ballot = __ballot_sync(0xFFFFFFFFu, used);
        if (lane == 0) warp_sum[warp] = __popc(ballot);
        __syncthreads();
        if (warp == 0) {
            int v = warp_sum[lane], s = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
                if (lane >= d) s += o;
            }
            warp_sum[lane] = s - v;
            if (lane == 31) total = s;
        }
        __syncthreads();
        if (used) {
            const int at = base + warp_sum[warp] + __popc(ballot & ((1u << lane) - 1u));
            index[at] = static_cast<int>(r);
            packed_target[at] = t >= 0 && t < vocab ? static_cast<int>(t) : -1;  // -1: the loss is NaN
        } else if (r < rows && row_loss_out != nullptr) {
            row_loss_out[r] = 0.0f;
        }
        base += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        sc->count = base;
        sc->amax_x = 0;
        sc->amax_w = 0;
        sc->z_log2 = kLog2e;
    }
}

// Largest finite |v| of x's listed rows (blockIdx.y 0) and of W (1).
__global__ void __launch_bounds__(256) ce_amax_kernel(const float* x, const float* w, const int* index, Scalars* sc, int64_t cols, int64_t vocab) {
    pdl_wait();
    const bool is_w = blockIdx.y == 1;
    const int64_t rows = is_w ? vocab : sc->count;
    unsigned top = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* src = is_w ? w + r * cols : x + static_cast<int64_t>(index[r]) * cols;
        for (int64_t c = threadIdx.x; c < cols; c += 256) {
            const unsigned b = __float_as_uint(src[c]) & 0x7FFFFFFFu;
            if (b < 0x7F800000u) top = max(top, b);
        }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0 && top != 0) atomicMax(is_w ? &sc->amax_w : &sc->amax_x, top);
}

// The power of two that takes the largest value into [2^14, 2^15).
__device__ __forceinline__ float plane_scale(unsigned amax_bits) {
    if (amax_bits == 0) return 1.0f;
    const int e = max(static_cast<int>(amax_bits >> 23), 1) - 127;
    return exp2f(static_cast<float>(max(-126, min(126, 14 - e))));
}

// Rows as binary16 planes with a padded row length: x's listed rows (and zero
// rows up to a multiple of kRowPad) or W's rows.
template <typename T, int PLANES>
__global__ void __launch_bounds__(128)
ce_pack_kernel(const T* src, const int* index, const Scalars* sc, int64_t src_rows, int64_t cols, __half* dst, int64_t ld, int64_t plane, bool vec) {
    pdl_wait();
    const int64_t live = index != nullptr ? sc->count : src_rows;
    const int64_t rows = index != nullptr ? (live + kRowPad - 1) / kRowPad * kRowPad : src_rows;
    float s = 1.0f;
    if constexpr (PLANES == 2) s = plane_scale(index != nullptr ? sc->amax_x : sc->amax_w);
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* from = r < live ? src + (index != nullptr ? static_cast<int64_t>(index[r]) : r) * cols : nullptr;
        __half* to = dst + r * ld;
        for (int64_t c = static_cast<int64_t>(threadIdx.x) * 8; c < ld; c += 128 * 8) {
            float v[8];
            if (from == nullptr) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
            } else if (vec) {  // 16-byte aligned rows, cols a multiple of 8
                if constexpr (sizeof(T) == 2) {
                    const uint4 u = *reinterpret_cast<const uint4*>(from + c);
                    *reinterpret_cast<uint4*>(to + c) = u;
                    continue;
                } else {
                    const float4 a = *reinterpret_cast<const float4*>(from + c), b = *reinterpret_cast<const float4*>(from + c + 4);
                    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
                    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? load_f(from, c + i) : 0.0f;
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float a = v[2 * t] * s, b = v[2 * t + 1] * s;
                hi[t] = half2_bits(a, b);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[t]));
                // a non-finite value is all in its high plane
                lo[t] = half2_bits(isfinite(f.x) ? a - f.x : 0.0f, isfinite(f.y) ? b - f.y : 0.0f);
            }
            *reinterpret_cast<uint4*>(to + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(to + plane + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) ce_bias_kernel(const T* bias, int64_t vocab, float* bias2) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < vocab) bias2[i] = load_f(bias, i) * kLog2e;
}

__global__ void ce_scale_kernel(Scalars* sc) {
    pdl_wait();
    sc->z_log2 = kLog2e / plane_scale(sc->amax_x) / plane_scale(sc->amax_w);
}

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    return v;
}

constexpr int kRowLanes = 32, kRowSlices = 16;

// Joins the statistics of 32 rows and forms their losses: lse2 (base 2) for
// the backward pass, the loss per packed row, and per row where asked for.
template <typename T>
__global__ void __launch_bounds__(kRowLanes* kRowSlices)
ce_rows_kernel(const T* x, const T* w, const T* bias, const int* index, const int* target, const Scalars* sc, const float2* part,
               int parts, int64_t rows_pad, int64_t cols, float* lse2, float* loss, float* row_loss_out) {
    pdl_wait();
    __shared__ float2 stat[kRowSlices][kRowLanes];
    __shared__ float hit[kRowLanes];
    const int rows = sc->count;
    const int lane = threadIdx.x, slice = threadIdx.y;
    for (int r0 = blockIdx.x * kRowLanes; r0 < rows; r0 += gridDim.x * kRowLanes) {
        const int m = r0 + lane;
        float top = -INFINITY, sum = 0.0f;
        for (int i = slice; i < parts; i += kRowSlices) {
            const float2 v = part[static_cast<int64_t>(i) * rows_pad + m];
            join(top, sum, v.x, v.y);
        }
        stat[slice][lane] = make_float2(top, sum);
        for (int k = slice; k < kRowLanes; k += kRowSlices) {  // a warp takes one row's target logit
            const int r = r0 + k;
            const int t = r < rows ? target[r] : -1;
            float dot = 0.0f;
            if (t >= 0) {
                const T* xr = x + static_cast<int64_t>(index[r]) * cols;
                const T* wr = w + static_cast<int64_t>(t) * cols;
                float d2 = 0.0f;
                int64_t c = lane;
                for (; c + 32 < cols; c += 64) {
                    dot = fmaf(load_f(xr, c), load_f(wr, c), dot);
                    d2 = fmaf(load_f(xr, c + 32), load_f(wr, c + 32), d2);
                }
                if (c < cols) dot = fmaf(load_f(xr, c), load_f(wr, c), dot);
                dot = warp_add(dot + d2);
                if (bias != nullptr) dot += load_f(bias, t);
            }
            if (lane == 0) hit[k] = t >= 0 ? dot : NAN;
        }
        __syncthreads();
        if (slice == 0 && m < rows) {
            for (int i = 1; i < kRowSlices; ++i) join(top, sum, stat[i][lane].x, stat[i][lane].y);
            const float l2 = top + log2f(sum);
            const float v = l2 * kLn2 - hit[lane];
            lse2[m] = target[m] >= 0 ? l2 : NAN;
            loss[m] = v;
            if (row_loss_out != nullptr) row_loss_out[index[m]] = v;
        }
        __syncthreads();
    }
}

// Sum or mean of the packed rows' losses, in a fixed order.
__global__ void __launch_bounds__(1024) ce_loss_kernel(const float* loss, const Scalars* sc, bool mean, float* out) {
    pdl_wait();
    __shared__ double part[32];
    const int rows = sc->count;
    double s = 0.0;
    for (int i = threadIdx.x; i < rows; i += 1024) s += loss[i];
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int i = 0; i < 32; ++i) s += part[i];
        *out = static_cast<float>(mean ? s / rows : s);  // no rows: 0 / 0, as torch's mean
    }
}

// g_i / max |g| per packed row, the maximum, and the gradients' scales.
__global__ void __launch_bounds__(1024)
ce_grad_rows_kernel(const float* grad, int reduction, const int* index, Scalars* sc, float* grow, int planes) {
    pdl_wait();
    __shared__ unsigned warp_top[32];
    const int rows = sc->count;
    const float g1 = reduction == TK_REDUCE_NONE ? 0.0f : reduction == TK_REDUCE_MEAN ? grad[0] / static_cast<float>(rows) : grad[0];
    unsigned top = reduction == TK_REDUCE_NONE ? 0u : __float_as_uint(g1) & 0x7FFFFFFFu;
    if (reduction == TK_REDUCE_NONE)
        for (int i = threadIdx.x; i < rows; i += 1024) top = max(top, __float_as_uint(grad[index[i]]) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xFFFFFFFFu, warp_top[threadIdx.x & 31]);
    const float gmax = rows > 0 ? __uint_as_float(top) : 0.0f;
    for (int i = threadIdx.x; i < rows; i += 1024) {
        const float g = reduction == TK_REDUCE_NONE ? grad[index[i]] : g1;
        grow[i] = gmax == 0.0f ? 0.0f : __fdiv_rn(g, gmax);
    }
    if (threadIdx.x == 0) {
        const float unit = gmax / kDzScale;
        sc->gmax = gmax;
        sc->db_scale = unit;
        sc->dx_scale = planes == 2 ? unit / plane_scale(sc->amax_w) : unit;
        sc->dw_scale = planes == 2 ? unit / plane_scale(sc->amax_x) : unit;
    }
}

// Zero gradients for the ignored rows.
__global__ void __launch_bounds__(128) ce_ignored_rows_kernel(const int64_t* target, int64_t ignore, int64_t rows, int64_t row_bytes, uint8_t* dx) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        if (target[r] != ignore) continue;
        uint8_t* o = dx + r * row_bytes;
        if (((reinterpret_cast<uintptr_t>(o) | row_bytes) & 15) == 0) {
            for (int64_t c = threadIdx.x * 16; c < row_bytes; c += 128 * 16) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
        } else {
            for (int64_t c = threadIdx.x * 2; c < row_bytes; c += 128 * 2) *reinterpret_cast<uint16_t*>(o + c) = 0;
        }
    }
}

constexpr int kDbThreads = 256;

// Column sums of a piece's dz: chunk blockIdx.y of the rows, 8 columns per
// lane, 8 rows at a time, into partial[chunk][dz_ld].
__global__ void __launch_bounds__(kDbThreads)
ce_dbias_part_kernel(const __half* dz, int64_t dz_ld, int64_t dz_plane, const Scalars* sc, float* partial) {
    pdl_wait();
    __shared__ float sums[8][32][9];
    const int rows = sc->count;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 256 + lane * 8;
    const int lo = static_cast<int>(static_cast<int64_t>(blockIdx.y) * rows / gridDim.y);
    const int hi = static_cast<int>(static_cast<int64_t>(blockIdx.y + 1) * rows / gridDim.y);
    float s[8] = {};
    for (int r = lo + warp; r < hi; r += 8) {
        for (int64_t off = 0;; off = dz_plane) {
            const uint4 u = *reinterpret_cast<const uint4*>(dz + off + r * dz_ld + col);
            const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float2 f = __half22float2(h[t]);
                s[2 * t] += f.x;
                s[2 * t + 1] += f.y;
            }
            if (off == dz_plane) break;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[warp][lane][i] = s[i];
    __syncthreads();
    for (int c = threadIdx.x; c < 256; c += kDbThreads) {
        float t = 0.0f;
        for (int w = 0; w < 8; ++w) t += sums[w][c / 8][c % 8];
        partial[static_cast<int64_t>(blockIdx.y) * dz_ld + static_cast<int64_t>(blockIdx.x) * 256 + c] = t;
    }
}

__global__ void __launch_bounds__(256)
ce_dbias_kernel(const float* partial, int chunks, int64_t dz_ld, int64_t cols, const Scalars* sc, void* out, int out_f32) {
    pdl_wait();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int i = 0; i < chunks; ++i) s += partial[i * dz_ld + c];
    s *= sc->db_scale;
    if (out_f32) {
        static_cast<float*>(out)[c] = s;
    } else {
        static_cast<__half*>(out)[c] = __float2half_rn(s);
    }
}

// ---- host --------------------------------------------------------------------------

constexpr int64_t kDzBytes = 512ll << 20;   // one piece's dz
constexpr int kSplitUnitsPerSm = 2;
constexpr int64_t kMaxSize = 0x7FFFFF00;

size_t align(size_t v) { return round_up(v, 1024); }

struct Plan {
    bool f16, w_direct;
    int planes;
    int64_t rows_pad, ld;    // packed rows and their length
    int64_t n_tiles;         // vocabulary tiles
    int64_t piece;           // vocabulary columns per piece (a multiple of BN)
    int64_t pieces;
    int split_units;
    int db_chunks;
    // state: kept from the forward to the backward pass
    size_t s_scalars, s_index, s_target, s_lse, state_bytes;
    // workspace
    size_t w_x, w_w, w_bias, w_part, w_loss, fwd_bytes;
    size_t b_grow, b_dz, b_acc, b_split, b_db, bwd_bytes;
};

int check(const char* who, const tk_linear_ce_desc_t& d) {
    TK_CHECK_ARG(d.dtype == TK_DTYPE_F16 || d.dtype == TK_DTYPE_F32, "%s: bad dtype %d", who, static_cast<int>(d.dtype));
    TK_CHECK_ARG(d.reduction == TK_REDUCE_NONE || d.reduction == TK_REDUCE_MEAN || d.reduction == TK_REDUCE_SUM, "%s: bad reduction %d", who, d.reduction);
    TK_CHECK_ARG(d.rows >= 0 && d.cols >= 1 && d.vocab >= 1, "%s: rows must not be negative, cols and vocab must be positive", who);
    if (d.rows > kMaxSize || d.cols > kMaxSize || d.vocab > kMaxSize) TK_FAIL(TK_ERR_UNSUPPORTED, "%s: sizes must be below 2^31 - 256", who);
    return TK_OK;
}

Plan make_plan(const tk_linear_ce_desc_t& d) {
    Plan p = {};
    p.f16 = d.dtype == TK_DTYPE_F16;
    p.planes = p.f16 ? 1 : 2;
    p.rows_pad = static_cast<int64_t>(round_up(static_cast<size_t>(std::max<int64_t>(d.rows, 1)), kRowPad));
    p.ld = static_cast<int64_t>(round_up(static_cast<size_t>(d.cols), 8));
    p.w_direct = p.f16 && d.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(d.weight) & 15) == 0;
    p.n_tiles = ceil_div(d.vocab, BN);
    // pieces of equal size whose dz planes fit kDzBytes (one tile at least)
    const int64_t most = std::max<int64_t>(1, kDzBytes / (p.rows_pad * 2 * p.planes * BN));
    p.pieces = ceil_div(p.n_tiles, most);
    p.piece = ceil_div(p.n_tiles, p.pieces) * BN;
    p.pieces = ceil_div(p.n_tiles * BN, p.piece);
    p.split_units = sm_count(current_device()) * kSplitUnitsPerSm;
    p.db_chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(d.rows, 64), ceil_div(4 * sm_count(current_device()), p.piece / 256))));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += align(bytes);
        return o;
    };
    p.s_scalars = take(sizeof(Scalars));
    p.s_index = take(p.rows_pad * sizeof(int));
    p.s_target = take(p.rows_pad * sizeof(int));
    p.s_lse = take(p.rows_pad * sizeof(float));
    p.state_bytes = at;
    at = 0;
    p.w_x = take(static_cast<size_t>(p.planes) * p.rows_pad * p.ld * 2);
    p.w_w = take(p.w_direct ? 0 : static_cast<size_t>(p.planes) * d.vocab * p.ld * 2);
    p.w_bias = take(d.bias != nullptr ? static_cast<size_t>(d.vocab) * sizeof(float) : 0);
    const size_t common = at;
    p.w_part = take(static_cast<size_t>(2 * p.n_tiles) * p.rows_pad * sizeof(float2));
    p.w_loss = take(p.rows_pad * sizeof(float));
    p.fwd_bytes = at + p.state_bytes;  // a call without a state keeps its own
    at = common;
    p.b_grow = take(p.rows_pad * sizeof(float));
    p.b_dz = take(static_cast<size_t>(p.planes) * p.rows_pad * p.piece * 2);
    p.b_acc = take(p.pieces > 1 ? static_cast<size_t>(p.rows_pad) * d.cols * sizeof(float) : 0);
    p.b_split = take(static_cast<size_t>(p.split_units) * BM * BN * sizeof(float));
    p.b_db = take(d.bias != nullptr ? static_cast<size_t>(p.db_chunks) * p.piece * sizeof(float) : 0);
    p.bwd_bytes = at;
    return p;
}

// A [planes][rows][inner] binary16 tensor read in boxes of 64 x box_rows.
int make_map(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int64_t planes, int64_t ld, int64_t plane, int box_rows) {
    EncodeTiledFn encode = tensor_map_encoder();
    if (encode == nullptr) TK_FAIL(TK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(plane) * 2};
    const cuuint32_t box[3] = {BK, static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t unit[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, unit,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) TK_FAIL(TK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return TK_OK;
}

#define CE_TRY(expr)                   \
    do {                               \
        if (int _rc = (expr)) return _rc; \
    } while (0)

template <typename... K, typename... A>
int launch_chain(const char* what, void (*k)(K...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... a) {
    const cudaError_t e = launch_pdl(k, grid, block, smem, s, std::forward<A>(a)...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        TK_FAIL(TK_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    }
    return TK_OK;
}

template <int EPI>
int gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmParams& p, int64_t most_units, cudaStream_t s) {
    TK_CUDA_TRY(cudaFuncSetAttribute(ce_gemm_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMM_SMEM));
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(sm_count(current_device()), most_units));
    return launch_chain("cross entropy GEMM", ce_gemm_kernel<EPI>, dim3(static_cast<unsigned>(grid)), dim3(THREADS), GEMM_SMEM, s, a, b, p);
}

int blocks_for(int64_t rows) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, 148 * 16))); }

// Packed operands (x's listed rows; W unless it is read in place; the bias).
template <typename T, int PLANES>
int pack(const tk_linear_ce_desc_t& d, const Plan& p, uint8_t* ws, const int* index, Scalars* sc, bool scan, cudaStream_t s) {
    const T* x = static_cast<const T*>(d.x);
    const T* w = static_cast<const T*>(d.weight);
    const bool xv = d.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const bool wv = d.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
    if constexpr (PLANES == 2) {
        if (scan) {
            CE_TRY(launch_chain("cross entropy amax", ce_amax_kernel, dim3(296, 2), dim3(256), 0, s, reinterpret_cast<const float*>(x),
                                reinterpret_cast<const float*>(w), index, sc, d.cols, d.vocab));
            CE_TRY(launch_chain("cross entropy scale", ce_scale_kernel, dim3(1), dim3(1), 0, s, sc));
        }
    }
    CE_TRY(launch_chain("cross entropy pack", ce_pack_kernel<T, PLANES>, dim3(blocks_for(p.rows_pad)), dim3(128), 0, s, x, index,
                        static_cast<const Scalars*>(sc), d.rows, d.cols, reinterpret_cast<__half*>(ws + p.w_x), p.ld, p.rows_pad * p.ld, xv));
    if (!p.w_direct)
        CE_TRY(launch_chain("cross entropy pack", ce_pack_kernel<T, PLANES>, dim3(blocks_for(d.vocab)), dim3(128), 0, s, w,
                            static_cast<const int*>(nullptr), static_cast<const Scalars*>(sc), d.vocab, d.cols,
                            reinterpret_cast<__half*>(ws + p.w_w), p.ld, d.vocab * p.ld, wv));
    if (d.bias != nullptr) {
        ce_bias_kernel<T><<<static_cast<unsigned>(ceil_div(d.vocab, 256)), 256, 0, s>>>(static_cast<const T*>(d.bias), d.vocab,
                                                                                       reinterpret_cast<float*>(ws + p.w_bias));
        CE_TRY(launch_status("cross entropy bias"));
    }
    return TK_OK;
}

int pack_any(const tk_linear_ce_desc_t& d, const Plan& p, uint8_t* ws, const int* index, Scalars* sc, bool scan, cudaStream_t s) {
    return p.f16 ? pack<__half, 1>(d, p, ws, index, sc, scan, s) : pack<float, 2>(d, p, ws, index, sc, scan, s);
}

struct Operands {
    const void* w;
    int64_t w_ld, w_plane;
};

Operands operands(const tk_linear_ce_desc_t& d, const Plan& p, uint8_t* ws) {
    if (p.w_direct) return {d.weight, d.cols, d.vocab * d.cols};
    return {ws + p.w_w, p.ld, d.vocab * p.ld};
}

GemmParams base_params(const tk_linear_ce_desc_t& d, const Plan& p, uint8_t* ws, const Scalars* sc) {
    GemmParams g = {};
    g.sc = sc;
    g.pairs = p.planes == 2 ? 3 : 1;
    g.m_tiles = -1;
    g.k_blocks = static_cast<int>(ceil_div(d.cols, BK));
    g.group = 16;
    g.max_units = p.split_units;
    g.err = device_error_word(current_device());
    g.bias2 = d.bias != nullptr ? reinterpret_cast<const float*>(ws + p.w_bias) : nullptr;
    g.vocab = d.vocab;
    g.rows_pad = p.rows_pad;
    return g;
}

}  // namespace
}  // namespace tk

extern "C" {

size_t tk_linear_ce_state_size(const tk_linear_ce_desc_t* desc) {
    if (desc == nullptr || tk::check("tk_linear_ce", *desc) != TK_OK) return 0;
    return tk::make_plan(*desc).state_bytes;
}

size_t tk_linear_ce_workspace_size(const tk_linear_ce_desc_t* desc) {
    if (desc == nullptr || tk::check("tk_linear_ce", *desc) != TK_OK) return 0;
    return tk::make_plan(*desc).fwd_bytes;
}

int tk_linear_ce(const tk_linear_ce_desc_t* desc, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace tk;
    TK_CHECK_ARG(desc != nullptr, "tk_linear_ce: NULL descriptor");
    const tk_linear_ce_desc_t& d = *desc;
    CE_TRY(check("tk_linear_ce", d));
    TK_CHECK_ARG(d.loss != nullptr || (d.rows == 0 && d.reduction == TK_REDUCE_NONE), "tk_linear_ce: loss is NULL");
    TK_CHECK_ARG(d.rows == 0 || (d.x && d.weight && d.target), "tk_linear_ce: NULL pointer");
    const Plan p = make_plan(d);
    if (workspace == nullptr || workspace_bytes < p.fwd_bytes || (reinterpret_cast<uintptr_t>(workspace) & 1023) != 0)
        TK_FAIL(TK_ERR_WORKSPACE, "tk_linear_ce: 1024-byte aligned workspace of %zu bytes needed, got %zu", p.fwd_bytes, workspace_bytes);
    TK_CHECK_ARG((reinterpret_cast<uintptr_t>(d.state) & 15) == 0, "tk_linear_ce: state must be 16-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint8_t* st = d.state != nullptr ? static_cast<uint8_t*>(d.state) : ws + (p.fwd_bytes - p.state_bytes);
    Scalars* sc = reinterpret_cast<Scalars*>(st + p.s_scalars);
    int* index = reinterpret_cast<int*>(st + p.s_index);
    int* target = reinterpret_cast<int*>(st + p.s_target);
    float* lse2 = reinterpret_cast<float*>(st + p.s_lse);
    float* loss = reinterpret_cast<float*>(ws + p.w_loss);
    float* per_row = d.reduction == TK_REDUCE_NONE ? d.loss : nullptr;
    ce_index_kernel<<<1, kIndexThreads, 0, s>>>(d.target, d.rows, d.vocab, d.ignore_index, index, target, sc, per_row);
    CE_TRY(launch_status("cross entropy index"));
    if (d.rows > 0) {
        CE_TRY(pack_any(d, p, ws, index, sc, true, s));
        const Operands o = operands(d, p, ws);
        CUtensorMap tx, tw;
        CE_TRY(make_map(&tx, ws + p.w_x, d.cols, p.rows_pad, p.planes, p.ld, p.rows_pad * p.ld, BM));
        CE_TRY(make_map(&tw, o.w, d.cols, d.vocab, p.planes, o.w_ld, o.w_plane, BN));
        GemmParams g = base_params(d, p, ws, sc);
        g.n_tiles = static_cast<int>(p.n_tiles);
        g.part = reinterpret_cast<float2*>(ws + p.w_part);
        CE_TRY(gemm<kStats>(tx, tw, g, p.n_tiles * ceil_div(d.rows, BM), s));
        const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(d.rows, kRowLanes), 148 * 4))), block(kRowLanes, kRowSlices);
        const float2* part = g.part;
        const int parts = static_cast<int>(2 * p.n_tiles);
        if (p.f16) {
            CE_TRY(launch_chain("cross entropy rows", ce_rows_kernel<__half>, grid, block, 0, s, static_cast<const __half*>(d.x),
                                static_cast<const __half*>(d.weight), static_cast<const __half*>(d.bias), static_cast<const int*>(index),
                                static_cast<const int*>(target), static_cast<const Scalars*>(sc), part, parts, p.rows_pad, d.cols, lse2, loss, per_row));
        } else {
            CE_TRY(launch_chain("cross entropy rows", ce_rows_kernel<float>, grid, block, 0, s, static_cast<const float*>(d.x),
                                static_cast<const float*>(d.weight), static_cast<const float*>(d.bias), static_cast<const int*>(index),
                                static_cast<const int*>(target), static_cast<const Scalars*>(sc), part, parts, p.rows_pad, d.cols, lse2, loss, per_row));
        }
    }
    if (d.reduction != TK_REDUCE_NONE)
        CE_TRY(launch_chain("cross entropy loss", ce_loss_kernel, dim3(1), dim3(1024), 0, s, static_cast<const float*>(loss),
                            static_cast<const Scalars*>(sc), d.reduction == TK_REDUCE_MEAN, d.loss));
    return TK_OK;
}

size_t tk_linear_ce_backward_workspace_size(const tk_linear_ce_grad_desc_t* desc) {
    if (desc == nullptr || tk::check("tk_linear_ce_backward", desc->fwd) != TK_OK) return 0;
    return tk::make_plan(desc->fwd).bwd_bytes;
}

int tk_linear_ce_backward(const tk_linear_ce_grad_desc_t* desc, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace tk;
    TK_CHECK_ARG(desc != nullptr, "tk_linear_ce_backward: NULL descriptor");
    const tk_linear_ce_desc_t& d = desc->fwd;
    CE_TRY(check("tk_linear_ce_backward", d));
    TK_CHECK_ARG(desc->dbias == nullptr || d.bias != nullptr, "tk_linear_ce_backward: dbias without a bias");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d.rows == 0) {
        if (desc->dweight) TK_CUDA_TRY(cudaMemsetAsync(desc->dweight, 0, static_cast<size_t>(d.vocab) * d.cols * dtype_size(d.dtype), s));
        if (desc->dbias) TK_CUDA_TRY(cudaMemsetAsync(desc->dbias, 0, static_cast<size_t>(d.vocab) * dtype_size(d.dtype), s));
        return TK_OK;
    }
    TK_CHECK_ARG(d.x && d.weight && d.target && d.state && desc->grad_loss, "tk_linear_ce_backward: NULL pointer");
    TK_CHECK_ARG((reinterpret_cast<uintptr_t>(d.state) & 15) == 0, "tk_linear_ce_backward: state must be 16-byte aligned");
    const Plan p = make_plan(d);
    if (workspace == nullptr || workspace_bytes < p.bwd_bytes || (reinterpret_cast<uintptr_t>(workspace) & 1023) != 0)
        TK_FAIL(TK_ERR_WORKSPACE, "tk_linear_ce_backward: 1024-byte aligned workspace of %zu bytes needed, got %zu", p.bwd_bytes, workspace_bytes);
    if (!desc->dx && !desc->dweight && !desc->dbias) return TK_OK;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint8_t* st = static_cast<uint8_t*>(d.state);
    Scalars* sc = reinterpret_cast<Scalars*>(st + p.s_scalars);
    const int* index = reinterpret_cast<const int*>(st + p.s_index);
    float* grow = reinterpret_cast<float*>(ws + p.b_grow);
    __half* dz = reinterpret_cast<__half*>(ws + p.b_dz);
    CE_TRY(pack_any(d, p, ws, index, sc, false, s));
    CE_TRY(launch_chain("cross entropy gradient rows", ce_grad_rows_kernel, dim3(1), dim3(1024), 0, s, desc->grad_loss, static_cast<int>(d.reduction),
                        index, sc, grow, p.planes));
    if (desc->dx) {
        ce_ignored_rows_kernel<<<blocks_for(d.rows), 128, 0, s>>>(d.target, d.ignore_index, d.rows, d.cols * static_cast<int64_t>(dtype_size(d.dtype)),
                                                                  static_cast<uint8_t*>(desc->dx));
        CE_TRY(launch_status("cross entropy ignored rows"));
    }
    const Operands o = operands(d, p, ws);
    const int64_t x_plane = p.rows_pad * p.ld, dz_plane = p.rows_pad * p.piece;
    CUtensorMap tx, tx_mn;
    CE_TRY(make_map(&tx, ws + p.w_x, d.cols, p.rows_pad, p.planes, p.ld, x_plane, BM));
    CE_TRY(make_map(&tx_mn, ws + p.w_x, d.cols, p.rows_pad, p.planes, p.ld, x_plane, BK));
    const int64_t row_tiles = ceil_div(d.rows, BM), col_tiles = ceil_div(d.cols, BN);
    const size_t esz = dtype_size(d.dtype);
    const bool cols16 = d.cols * esz % 16 == 0;
    for (int64_t i = 0; i < p.pieces; ++i) {
        const int64_t v0 = i * p.piece, width = std::min(p.piece, d.vocab - v0);
        const uint8_t* wbase = static_cast<const uint8_t*>(o.w) + v0 * o.w_ld * 2;
        CUtensorMap tw, tw_mn, tdz, tdz_mn;
        CE_TRY(make_map(&tw, wbase, d.cols, width, p.planes, o.w_ld, o.w_plane, BN));
        CE_TRY(make_map(&tw_mn, wbase, d.cols, width, p.planes, o.w_ld, o.w_plane, BK));
        CE_TRY(make_map(&tdz, dz, width, p.rows_pad, p.planes, p.piece, dz_plane, BM));
        CE_TRY(make_map(&tdz_mn, dz, width, p.rows_pad, p.planes, p.piece, dz_plane, BK));
        GemmParams g = base_params(d, p, ws, sc);
        g.n_tiles = static_cast<int>(ceil_div(width, BN));
        g.vocab0 = v0;
        g.lse2 = reinterpret_cast<const float*>(st + p.s_lse);
        g.grow = grow;
        g.target = reinterpret_cast<const int*>(st + p.s_target);
        g.dz = dz;
        g.dz_ld = p.piece;
        g.dz_plane = p.planes == 2 ? dz_plane : 0;
        CE_TRY(gemm<kDlogits>(tx, tw, g, row_tiles * g.n_tiles, s));
        GemmParams r = base_params(d, p, ws, sc);
        r.out_cols = d.cols;
        r.out_f32 = p.f16 ? 0 : 1;
        r.n_tiles = static_cast<int>(col_tiles);
        r.split = reinterpret_cast<float*>(ws + p.b_split);
        if (desc->dx) {
            r.k_blocks = static_cast<int>(ceil_div(width, BK));
            r.out = desc->dx;
            r.out_vec = cols16 && (reinterpret_cast<uintptr_t>(desc->dx) & 15) == 0;
            r.index = index;
            r.acc = reinterpret_cast<float*>(ws + p.b_acc);
            r.first = i == 0;
            r.last = i + 1 == p.pieces;
            CE_TRY(gemm<kGradX>(tdz, tw_mn, r, std::max<int64_t>(row_tiles * col_tiles, p.split_units), s));
            CE_TRY(launch_chain("cross entropy split", ce_split_kernel<kGradX>, dim3(static_cast<unsigned>(p.split_units) * 4), dim3(64), 0, s, r));
        }
        if (desc->dweight) {
            r.m_tiles = static_cast<int>(ceil_div(width, BM));
            r.k_blocks = -1;
            r.out = static_cast<uint8_t*>(desc->dweight) + v0 * d.cols * esz;
            r.out_vec = cols16 && (reinterpret_cast<uintptr_t>(r.out) & 15) == 0;
            r.out_rows = width;
            CE_TRY(gemm<kGradW>(tdz_mn, tx_mn, r, std::max<int64_t>(r.m_tiles * col_tiles, p.split_units), s));
            if (2 * r.m_tiles * col_tiles <= p.split_units)
                CE_TRY(launch_chain("cross entropy split", ce_split_kernel<kGradW>, dim3(static_cast<unsigned>(p.split_units) * 4), dim3(64), 0, s, r));
        }
        if (desc->dbias) {
            float* part = reinterpret_cast<float*>(ws + p.b_db);
            CE_TRY(launch_chain("cross entropy bias sums", ce_dbias_part_kernel, dim3(static_cast<unsigned>(p.piece / 256), p.db_chunks), dim3(kDbThreads), 0, s,
                                static_cast<const __half*>(dz), p.piece, g.dz_plane, static_cast<const Scalars*>(sc), part));
            CE_TRY(launch_chain("cross entropy bias sums", ce_dbias_kernel, dim3(static_cast<unsigned>(ceil_div(width, 256))), dim3(256), 0, s,
                                static_cast<const float*>(part), p.db_chunks, p.piece, width, static_cast<const Scalars*>(sc),
                                static_cast<void*>(static_cast<uint8_t*>(desc->dbias) + v0 * esz), p.f16 ? 0 : 1));
        }
    }
    return TK_OK;
}

}  // extern "C"
