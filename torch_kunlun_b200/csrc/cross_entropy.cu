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
// the maximum and the sum of exponentials (base 2), and the target's logit; a
// small kernel joins them.  logsumexp and the target's logit carry the same
// rounding, so no loss is negative and that of a row whose target dominates is
// not lost in it (with a dot product of its own for the target, 512 columns and
// logits of 500 gave losses of -2.7e-3).  Backward: the
// vocabulary is taken in pieces whose dz fits a workspace; per piece the
// logits are computed again, the epilogue stores dz as binary16, and two
// GEMMs read it in place (dz and x^T / W^T in MN-major shared-memory tiles, so
// nothing is transposed).
//
// binary16 dz: softmax - onehot lies in [-1, 1] and is held at 2^14 times its
// value, so entries down to 2^-28 keep all 11 bits (22 with fp32's two planes,
// down to 2^-17) and no entry loses more than 2^-39.  One g for all rows is
// applied in binary32 when dx, dW and db are rounded.  Where rows have gradients
// of their own, g_i = m_i 2^k_i with m_i in [1, 2): dz takes m_i, dx's row takes
// 2^k_i in its epilogue, so rows do not touch one another whatever their
// gradients (one NaN, or six decades between them, would otherwise spoil the
// others' dx), and dW reads x's rows times 2^k_i, their largest |x g| in [2^14,
// 2^15): again 2^-39 of the largest is all that a term can lose.
//
// fp32 operands are split into two binary16 planes of a power-of-two multiple
// (hi = rn(v s), lo = rn(v s - hi), the largest value of W and of each row of x
// in [2^14, 2^15)), 22 bits or 2^-40 of that largest value, and a product is the
// sum hi*hi + hi*lo + lo*hi: a K block takes two stages, one for each plane of both
// operands, and three products.
//
// GEMM kernel (persistent pairs of CTAs, one CTA per SM):
// a pair computes 256 x 256 tiles, CTA r holding rows [128 r, + 128) of A and
// of B in shared memory and of the result in TMEM, so each SM loads 32 KB per
// 64 K values of a 256 x 256 tile.  Warp 0 of both CTAs loads its halves by
// TMA (128-byte swizzle) onto the leader's barriers, warp 1 of the leader
// issues tcgen05.mma cta_group::2 kind::f16 into two 256-column accumulators,
// the other warps of both CTAs run the epilogue of one while the other fills.
//
// The tensor core adds each 16-deep step into a binary32 accumulator that it
// cuts rather than rounds, a bias that grows with K.  Where outputs are
// binary32 (fp32 gradients, the loss) the K loop is cut into chunks that the
// epilogue adds in registers.  dz's logits are summed as the statistics' were:
// summed otherwise, a target's probability of 1 came back 1e-3 off at logits of
// 50 over 4096 columns, and that much of its row of W in dx.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "tk_internal.h"
#include "tk_ptx.cuh"

namespace tk {
namespace {

constexpr int BM = 256, BN = 256, BK = 64;  // a pair's tile
constexpr int HM = BM / 2, HN = BN / 2;     // one CTA's operand rows
constexpr int A_BYTES = HM * BK * 2, B_BYTES = HN * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
// An epilogue warp turns 32 rows x 16 columns through its own 2.5 KB, so that
// four lanes store whole sectors of a row (80-byte pitch: no bank conflicts for
// 16-byte accesses).
constexpr int TURN = 16;
constexpr int PITCH = TURN + 4;

// kPlain: eight epilogue warps, six stages.  kWide: sixteen warps for dz and dW
// where the K loop is short (dz of 2384 rows by 30011 words at 768 columns, 12
// K blocks: 177 -> 166 us; at 64 K blocks five stages cost 3 %; dW of 9 rows,
// 110320 x 325: 101 -> 90 us; dx of 122 rows, 1199 x 235: 12.0 -> 12.5, and the
// statistics of 9 x 325 by 110320: 31.0 -> 32.7, so they stay plain).
// kChunked: sums in registers, 128 columns per thread.  kPlanes: the same for
// fp32 operands.  kPlanesWide: sixteen warps where fp32's K loop is one chunk (13 x 64 by 82545
// words: logits 25 -> 19, dz 52 -> 29, dW 35 -> 22 us).
enum Mode { kPlain, kWide, kChunked, kPlanes, kPlanesWide };
constexpr int kWideBlocks = 24;  // K blocks up to which kWide is taken

template <int MODE>
struct Config {
    static constexpr int PLANES = MODE == kPlanes || MODE == kPlanesWide ? 2 : 1;
    static constexpr bool CHUNKED = MODE == kChunked || MODE == kPlanes;
    static constexpr bool WIDE = MODE == kWide || MODE == kPlanesWide;
    static constexpr int STAGES = MODE == kWide ? 5 : MODE == kPlanesWide ? 4 : 6;  // a multiple of PLANES
    static constexpr int EPI_WARPS = WIDE ? 16 : 8;
    static constexpr int COLS = BN / (EPI_WARPS / 4);  // of a tile row, per warp
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int TURN_BYTES = EPI_WARPS * 32 * PITCH * 4;
    static constexpr int SMEM = STAGES * STAGE_BYTES + TURN_BYTES + 1024 + 256;
    static_assert(SMEM <= 232448, "shared memory budget");
};

// K blocks per accumulator chunk: 24 steps of 16 (two blocks, three products)
// where every output is binary32, 64 for the logits of fp16 operands (measured at
// 4096 columns: the loss 1e-6 off without chunks, and the same time; dz of 8192
// rows by 65536 words 3.29 -> 3.56 ms, of 300 x 1536 by 30011 46 -> 58 us).
constexpr int kChunkF32 = 2, kChunkStats = 16;

constexpr int TMEM_COLS = 512;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kDzScale = 16384.0f;
constexpr int kRowPad = 256;  // rows of a tile: packed rows have room up to a multiple of this

// Device scalars of one call.
struct Scalars {
    int count;           // rows with a target
    unsigned amax_w;     // binary32 bits of the largest finite |W| (fp32 operands)
    unsigned rows_done;  // blocks of ce_rows_kernel that finished
};

// Device scalars of one backward pass: accumulators -> gradients.
struct GradScalars {
    float dx_scale, dw_scale, db_scale;
    int top;  // largest exponent of x_i g_i, where x's rows are scaled for dW
};

enum Epilogue { kStats, kDlogits, kGradX, kGradW };

struct GemmParams {
    const Scalars* sc;
    const GradScalars* gs;
    int n_tiles;
    int m_tiles;   // < 0: from sc->count
    int k_blocks;  // < 0: from sc->count
    int planes;    // 1 (fp16 operands) or 2 (fp32)
    int chunk;     // K blocks per accumulator chunk
    int max_units; // tiles x K splits the workspace of a split reduction holds
    int group;     // M tiles that neighbouring CTAs share
    unsigned* err;
    // kStats / kDlogits
    int64_t vocab0, vocab;  // the piece's first column, all columns
    const float* bias2;  // bias * log2(e), or NULL
    float2* part;        // [rows][n_tiles][BN / COLS] maximum and sum
    float* hit2;         // kStats: the target's logit, base 2
    const float* lse2;
    const float* xs;     // kStats, kDlogits: what the rows' planes were multiplied by; NULL: 1 (fp16 operands)
    const float* grow;   // kDlogits, kGradX: g_i; NULL: one for all rows
    const int* target;
    __half* dz;          // [planes][rows_pad][dz_ld]
    int64_t dz_ld, dz_plane;
    // kGradX / kGradW
    void* out;
    const int* index;    // kGradX: output row of a packed row
    int64_t out_rows, out_cols;
    int out_f32, out_vec;
    float* acc;          // [rows_pad][acc_ld] sums over earlier pieces
    int64_t acc_ld;
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
    s.blocks = p.k_blocks >= 0 ? p.k_blocks : (count + BK - 1) / BK;
    s.splits = EPI == kGradX || EPI == kGradW ? k_splits(p, s.m_tiles * p.n_tiles, s.blocks) : 1;
    s.units = s.m_tiles * p.n_tiles * s.splits;
    return s;
}

// First K block of a split.
__device__ __forceinline__ int split_begin(const Shape& s, int ks) {
    return static_cast<int>(static_cast<int64_t>(ks) * s.blocks / s.splits);
}

// Work unit -> (K split, M tile, N tile); the split varies slowest, tiles run
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

// D[tmem of both CTAs] (+)= A B^T over the pair's shared memory.
__device__ __forceinline__ void tc_mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrive on the mbarrier at this offset in both CTAs of the pair once all
// prior tcgen05 operations of this thread have completed.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

// The same on this CTA's mbarrier alone (one kernel uses one .cta_group).
__device__ __forceinline__ void tc_commit_pair_local(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// One box into this CTA's shared memory, completing on a barrier of the pair
// (a shared::cluster address); c0, innermost, is a multiple of 8 elements.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void* tmap, uint32_t cluster_bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
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

// The power of two that takes the largest value into [2^14, 2^15).
__device__ __forceinline__ float plane_scale(unsigned amax_bits) {
    if (amax_bits == 0) return 1.0f;
    const int e = max(static_cast<int>(amax_bits >> 23), 1) - 127;
    return exp2f(static_cast<float>(max(-126, min(126, 14 - e))));
}

// g = mantissa * 2^exponent, the mantissa in [1, 2) (below 1 for subnormal and
// zero g; a NaN or infinity is its own mantissa).
__device__ __forceinline__ int exponent_of(float g) {
    const int e = static_cast<int>(__float_as_uint(g) >> 23 & 0xFFu);
    return e == 255 ? 0 : max(e, 1) - 127;
}
__device__ __forceinline__ float pow2(int e) {  // 2^e, 0 below the subnormal numbers, at most 2^127
    return __uint_as_float(e >= -126 ? static_cast<uint32_t>(min(127, e) + 127) << 23 : e >= -149 ? 1u << (e + 149) : 0u);
}
__device__ __forceinline__ float mantissa_of(float g) {
    const uint32_t b = __float_as_uint(g), e = b >> 23 & 0xFFu;
    return e == 255 ? g : e == 0 ? g * pow2(126) : __uint_as_float((b & 0x807FFFFFu) | 0x3F800000u);
}

// 32 consecutive columns of one row: base-2 logits from the accumulators.
__device__ __forceinline__ void logits2(const float* acc, float k, const float* bias2, int64_t col, int64_t vocab, float (&y)[32]) {
    if (bias2 != nullptr) {
        if (col + 32 <= vocab) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 b = __ldg(reinterpret_cast<const float4*>(bias2 + col + i));
                y[i] = fmaf(acc[i], k, b.x);
                y[i + 1] = fmaf(acc[i + 1], k, b.y);
                y[i + 2] = fmaf(acc[i + 2], k, b.z);
                y[i + 3] = fmaf(acc[i + 3], k, b.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = col + i < vocab ? fmaf(acc[i], k, __ldg(bias2 + col + i)) : -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = acc[i] * k;
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

// The 32 x 16 block that the warp's lanes hold by rows (v: this lane's row) in
// shared memory, for its lanes to read by columns.
__device__ __forceinline__ void turn_in(float* buf, int lane, const float* v) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < TURN; i += 4) *reinterpret_cast<float4*>(buf + lane * PITCH + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    __syncwarp();
}
// Hands the block out as f(row, column, four values), four lanes per row.
template <typename F>
__device__ __forceinline__ void turn_out4(const float* buf, int lane, F f) {
#pragma unroll
    for (int r = 0; r < 32; r += 8) {
        const int row = r + lane / 4, col = lane % 4 * 4;
        f(row, col, *reinterpret_cast<const float4*>(buf + row * PITCH + col));
    }
}
// Hands it out as f(row, column, value), 16 lanes per row.
template <typename F>
__device__ __forceinline__ void turn_out1(const float* buf, int lane, F f) {
#pragma unroll 4
    for (int r = 0; r < 32; r += 2) f(r + lane / 16, lane % 16, buf[(r + lane / 16) * PITCH + lane % 16]);
}

// N (four or one) finished values of a gradient: joined with the
// earlier pieces' sum, kept for the next piece, or scaled, rounded and stored.
template <int EPI, int N>
__device__ __forceinline__ void finish(const GemmParams& p, int64_t m, int64_t rows, int64_t col, float scale, float4 f) {
    if (m >= rows || col >= p.out_cols) return;
    float v[4] = {f.x, f.y, f.z, f.w};
    if (EPI == kGradX && !(p.first && p.last)) {
        float* a = p.acc + m * p.acc_ld + col;  // acc_ld is a multiple of four
        if (!p.first) {
            if constexpr (N == 4) {
                const float4 e = *reinterpret_cast<const float4*>(a);
                v[0] += e.x, v[1] += e.y, v[2] += e.z, v[3] += e.w;
            } else {
                v[0] += *a;
            }
        }
        if (!p.last) {
            if constexpr (N == 4) {
                *reinterpret_cast<float4*>(a) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                *a = v[0];
            }
            return;
        }
    }
    const int64_t at = (EPI == kGradX ? p.index[m] : m) * p.out_cols + col;
    if (EPI == kGradX && p.grow != nullptr) scale *= pow2(exponent_of(p.grow[m]));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= scale;
    if constexpr (N == 4) {  // out_cols a multiple of 16 bytes, out 16-byte aligned
        if (p.out_f32) {
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = make_uint2(half2_bits(v[0], v[1]), half2_bits(v[2], v[3]));
        }
    } else {
        if (p.out_f32) {
            static_cast<float*>(p.out)[at] = v[0];
        } else {
            static_cast<__half*>(p.out)[at] = __float2half_rn(v[0]);
        }
    }
}

// The scale that takes an accumulator of row m to a base-2 logit.
__device__ __forceinline__ float z_scale(const GemmParams& p, int64_t m) {
    return p.xs == nullptr ? kLog2e : kLog2e / p.xs[m] / plane_scale(p.sc->amax_w);
}

template <int EPI, int MODE>
__global__ void __launch_bounds__(Config<MODE>::THREADS, 1)
ce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmParams p) {
    constexpr bool A_MN = EPI == kGradW, B_MN = EPI == kGradX || EPI == kGradW;
    constexpr uint32_t IDESC = idesc_f16(BM, BN, A_MN, B_MN);
    using C = Config<MODE>;
    constexpr bool CHUNKED = C::CHUNKED;
    constexpr int PLANES = C::PLANES;
    constexpr int STAGES = C::STAGES, EPI_WARPS = C::EPI_WARPS, COLS = C::COLS;
    static_assert(STAGES % PLANES == 0, "both planes' stages are neighbours");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* turn_buf = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + C::TURN_BYTES);
    uint64_t* full_bar = bars;               // [STAGES] both CTAs' TMA -> MMA (leader's)
    uint64_t* empty_bar = bars + STAGES;     // [STAGES] MMA -> TMA (each CTA's)
    uint64_t* acc_full = bars + 2 * STAGES;  // [2] MMA -> epilogue (each CTA's)
    uint64_t* acc_empty = acc_full + 2;      // [2] both CTAs' epilogue -> MMA (leader's)
    uint64_t* drain_bar = acc_empty + 2;     // MMA teardown (leader's)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(full_bar + s), 1);
            mbar_init(smem_u32(empty_bar + s), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(acc_full + i), 1);
            mbar_init(smem_u32(acc_empty + i), 2 * EPI_WARPS);
        }
        mbar_init(smem_u32(drain_bar), 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the pair's barriers are set before either CTA signals them
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    const Shape sh = shape_of<EPI>(p);
    const int first_unit = blockIdx.x >> 1, unit_step = gridDim.x >> 1;

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        int stage = 0;
        uint32_t phase = 0;
        uint32_t last_phase[STAGES];
        bool used[STAGES];
        for (int s = 0; s < STAGES; ++s) {
            used[s] = false;
            last_phase[s] = 0;
        }
        bool ok = true;
        for (int u = first_unit; u < sh.units && ok; u += unit_step) {
            int mt, nt, ks;
            decode_unit(p, sh, u, mt, nt, ks);
            const int kb1 = split_begin(sh, ks + 1);
            const int a0 = mt * BM + static_cast<int>(rank) * HM, b0 = nt * BN + static_cast<int>(rank) * HN;
            // a stage for each plane of each K block
            for (int i = split_begin(sh, ks) * PLANES; i < kb1 * PLANES; ++i) {
                if (!mbar_wait_bounded(smem_u32(empty_bar + stage), phase ^ 1u, abort_flag, p.err, kDevErrWaitEmpty)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    const int kx = i / PLANES * BK, plane = i % PLANES;
                    if (leader) mbar_arrive_expect_tx(smem_u32(full_bar + stage), 2 * STAGE_BYTES);
                    const uint32_t fb = mapa_shared(smem_u32(full_bar + stage), 0);
                    const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES);
                    if constexpr (A_MN) {
#pragma unroll
                        for (int j = 0; j < HM / 64; ++j) tma_load_3d_pair(sa + j * BK * 128, &tmA, fb, a0 + j * 64, kx, plane);
                    } else {
                        tma_load_3d_pair(sa, &tmA, fb, kx, a0, plane);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int j = 0; j < HN / 64; ++j) tma_load_3d_pair(sa + A_BYTES + j * BK * 128, &tmB, fb, b0 + j * 64, kx, plane);
                    } else {
                        tma_load_3d_pair(sa + A_BYTES, &tmB, fb, kx, b0, plane);
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
        // Drain: every box of the pair has landed before either CTA exits (the
        // leader's barriers count both; the peer waits at the cluster barrier).
        if (leader) {
            for (int s = 0; s < STAGES; ++s) {
                if (used[s]) {
                    volatile int no_abort = 0;
                    mbar_wait_bounded(smem_u32(full_bar + s), last_phase[s], &no_abort, p.err, kDevErrWaitDrain);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader) ----------------
        if (leader) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            int local = 0;  // accumulator chunks so far
            for (int u = first_unit; u < sh.units && ok; u += unit_step) {
                int mt, nt, ks;
                decode_unit(p, sh, u, mt, nt, ks);
                int kb = split_begin(sh, ks);
                const int kb1 = split_begin(sh, ks + 1);
                do {
                    const int c0 = kb, c1 = CHUNKED ? min(kb1, kb + p.chunk) : kb1;
                    const int buf = local & 1;
                    if (!mbar_wait_bounded_cluster(smem_u32(acc_empty + buf), ((local >> 1) & 1) ^ 1u, abort_flag, p.err, kDevErrWaitAccEmpty)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t acc = tmem_base + buf * BN;
                    for (; kb < c1; ++kb) {
                        // PLANES divides STAGES: the planes' stages are neighbours
                        for (int j = 0; j < PLANES && ok; ++j)
                            ok = mbar_wait_bounded(smem_u32(full_bar + stage + j), phase, abort_flag, p.err, kDevErrWaitFull);
                        if (!ok) break;
                        tc_fence_after();
                        if (lane == 0) {
                            const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES);
                            uint64_t da[PLANES], db[PLANES];
#pragma unroll
                            for (int j = 0; j < PLANES; ++j) {
                                const uint32_t s = sa + j * STAGE_BYTES;
                                da[j] = A_MN ? smem_desc_mnmajor_sw128(s) : smem_desc_kmajor_sw128(s);
                                db[j] = B_MN ? smem_desc_mnmajor_sw128(s + A_BYTES) : smem_desc_kmajor_sw128(s + A_BYTES);
                            }
                            // 16 K values on: 32 bytes inside the swizzled row of a
                            // K-major tile, two 1 KB atoms of an MN-major one
                            constexpr uint64_t step_a = (A_MN ? 2048 : 32) >> 4, step_b = (B_MN ? 2048 : 32) >> 4;
#pragma unroll
                            for (int kk = 0; kk < BK / 16; ++kk) {
                                tc_mma_f16_pair(acc, da[0] + kk * step_a, db[0] + kk * step_b, IDESC, kb > c0 || kk > 0 ? 1u : 0u);
                                if constexpr (PLANES == 2) {
                                    tc_mma_f16_pair(acc, da[0] + kk * step_a, db[1] + kk * step_b, IDESC, 1u);
                                    tc_mma_f16_pair(acc, da[1] + kk * step_a, db[0] + kk * step_b, IDESC, 1u);
                                }
                            }
#pragma unroll
                            for (int j = 0; j < PLANES; ++j) tc_commit_pair(smem_u32(empty_bar + stage + j));
                        }
                        __syncwarp();
                        stage += PLANES;
                        if (stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    if (!ok) break;
                    if (lane == 0) tc_commit_pair(smem_u32(acc_full + buf));
                    __syncwarp();
                    ++local;
                } while (kb < kb1);
            }
            // Drain: all MMAs of this thread complete before TMEM is freed.
            if (lane == 0) tc_commit_pair_local(smem_u32(drain_bar));
            __syncwarp();
            volatile int no_abort = 0;
            mbar_wait_bounded(smem_u32(drain_bar), 0, &no_abort, p.err, kDevErrWaitDrain);
        }
    } else {
        // ---------------- epilogue (the other warps of both CTAs) ----------------
        // A warp reads TMEM lanes [32 * (warp % 4), + 32), one row per lane,
        // and COLS of the tile's columns.
        const int quarter = warp & 3, share = (warp - 2) >> 2;
        float* const buf_turn = turn_buf + (warp - 2) * 32 * PITCH;
        const int rows = p.sc->count;
        float scale = 1.0f;
        if constexpr (EPI == kGradX) scale = p.gs->dx_scale;
        if constexpr (EPI == kGradW) scale = p.gs->dw_scale;
        int local = 0;
        bool ok = true;
        for (int u = first_unit; u < sh.units && ok; u += unit_step) {
            int mt, nt, ks;
            decode_unit(p, sh, u, mt, nt, ks);
            const int blocks = split_begin(sh, ks + 1) - split_begin(sh, ks);
            const int64_t m0 = static_cast<int64_t>(mt) * BM + rank * HM + quarter * 32;  // the warp's first row
            const int64_t m = m0 + lane;
            const int64_t col0 = static_cast<int64_t>(nt) * BN + share * COLS;
            float top = -INFINITY, sum = 0.0f;  // kStats
            const bool live = m < rows;         // kStats, kDlogits
            if constexpr (EPI == kStats || EPI == kDlogits) scale = live ? z_scale(p, m) : 0.0f;
            const float lse = EPI == kDlogits && live ? p.lse2[m] : 0.0f;
            const float g = EPI == kDlogits && live ? (p.grow != nullptr ? mantissa_of(p.grow[m]) * kDzScale : kDzScale) : 0.0f;
            const int64_t hit = (EPI == kStats || EPI == kDlogits) && live ? p.target[m] - p.vocab0 : -1;
            // rows that the warp works for: dz is read (as K) up to a multiple of BK
            const int64_t limit = EPI == kGradW ? p.out_rows : EPI == kDlogits ? (rows + BK - 1) / BK * BK : rows;
            const bool idle = m0 >= limit;
            // 32 columns of this lane's row, from column col0 + c of the tile
            auto take = [&](int c, const float* acc) {
                const int64_t col = col0 + c;
                if constexpr (EPI == kStats) {
                    float y[32];
                    logits2(acc, scale, p.bias2, col, p.vocab, y);
                    if (hit >= col && hit < col + 32) {
                        const int j = static_cast<int>(hit - col);
                        float h = y[0];
#pragma unroll
                        for (int i = 1; i < 32; ++i) h = i == j ? y[i] : h;
                        p.hit2[m] = h;
                    }
                    float cm = y[0];
#pragma unroll
                    for (int i = 1; i < 32; ++i) cm = fmaxf(cm, y[i]);
                    const float ref = cm == -INFINITY ? 0.0f : cm;
                    float cs = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) cs += exp2_sfu(y[i] - ref);
                    join(top, sum, cm, cs);
                } else if constexpr (EPI == kDlogits) {
                    float y[32];
                    logits2(acc, scale, p.bias2, p.vocab0 + col, p.vocab, y);
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = live ? exp2_sfu(y[i] - lse) * g : 0.0f;
                    if (hit >= col && hit < col + 32) {
                        const int j = static_cast<int>(hit - col);
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] -= i == j ? g : 0.0f;
                    }
#pragma unroll
                    for (int h = 0; h < 32; h += TURN) {
                        turn_in(buf_turn, lane, y + h);
                        turn_out4(buf_turn, lane, [&](int r, int cc, float4 f) {
                            __half* o = p.dz + (m0 + r) * p.dz_ld + col + h + cc;
                            const uint2 hi = make_uint2(half2_bits(f.x, f.y), half2_bits(f.z, f.w));
                            *reinterpret_cast<uint2*>(o) = hi;
                            if (p.dz_plane != 0) {
                                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
                                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                                *reinterpret_cast<uint2*>(o + p.dz_plane) = make_uint2(half2_bits(f.x - a.x, f.y - a.y), half2_bits(f.z - b.x, f.w - b.y));
                            }
                        });
                    }
                } else {
                    if (col >= p.out_cols && sh.splits == 1) return;
#pragma unroll
                    for (int h = 0; h < 32; h += TURN) {
                        turn_in(buf_turn, lane, acc + h);
                        if (sh.splits > 1) {
                            turn_out4(buf_turn, lane, [&](int r, int cc, float4 f) {
                                *reinterpret_cast<float4*>(p.split + (static_cast<int64_t>(u) * BM + rank * HM + quarter * 32 + r) * BN + share * COLS + c + h + cc) = f;
                            });
                        } else if (p.out_vec) {
                            turn_out4(buf_turn, lane, [&](int r, int cc, float4 f) { finish<EPI, 4>(p, m0 + r, limit, col + h + cc, scale, f); });
                        } else {
                            turn_out1(buf_turn, lane, [&](int r, int cc, float f) {
                                finish<EPI, 1>(p, m0 + r, limit, col + h + cc, scale, make_float4(f, 0.0f, 0.0f, 0.0f));
                            });
                        }
                    }
                }
            };
            const int chunks = CHUNKED ? max(1, (blocks + p.chunk - 1) / p.chunk) : 1;
            float v[CHUNKED ? COLS : 32];
            if constexpr (CHUNKED) {
#pragma unroll
                for (int i = 0; i < COLS; ++i) v[i] = 0.0f;
            }
            for (int k = 0; k < chunks; ++k, ++local) {
                const int buf = local & 1;
                if (!mbar_wait_bounded(smem_u32(acc_full + buf), (local >> 1) & 1, abort_flag, p.err, kDevErrWaitAccFull)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * BN + share * COLS;
                if (idle) {
                } else if constexpr (CHUNKED) {
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        uint32_t acc[32];
                        tmem_ld_32x32b_x32(t0 + c, acc);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[c + i] += blocks > 0 ? __uint_as_float(acc[i]) : 0.0f;
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < COLS; c += 32) {
                        uint32_t acc[32];
                        tmem_ld_32x32b_x32(t0 + c, acc);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = blocks > 0 ? __uint_as_float(acc[i]) : 0.0f;
                        take(c, v);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(acc_empty + buf), 0));
            }
            if (!ok) break;
            if (idle) continue;
            if constexpr (CHUNKED) {
#pragma unroll
                for (int c = 0; c < COLS; c += 32) take(c, v + c);
            }
            if constexpr (EPI == kStats) p.part[(m * p.n_tiles + nt) * (BN / COLS) + share] = make_float2(top, sum);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA leaves while the other signals it or reads its operands
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem_base, TMEM_COLS);
}

// Adds the K splits of the tiles in a fixed order, 64 threads by four columns
// to a row.  Few tiles have many splits: the block's four groups of 64 share
// those of one row; otherwise each takes a row of its own.
template <int EPI>
__global__ void __launch_bounds__(256) ce_split_kernel(const GemmParams p) {
    pdl_wait();
    __shared__ float4 part[4][64];
    const Shape sh = shape_of<EPI>(p);
    if (sh.splits <= 1) return;
    const int tiles = sh.m_tiles * p.n_tiles;
    const int64_t limit = EPI == kGradX ? p.sc->count : p.out_rows;
    const float scale = EPI == kGradX ? p.gs->dx_scale : p.gs->dw_scale;
    const int quad = threadIdx.x % 64, group = threadIdx.x / 64;
    const int shares = sh.splits >= 16 ? 4 : 1, rows = 4 / shares;
    const int share = shares == 4 ? group : 0;
    const int k0 = share * sh.splits / shares, k1 = (share + 1) * sh.splits / shares;
    for (int b = blockIdx.x; b < tiles * (BM / rows); b += gridDim.x) {
        const int tile = b / (BM / rows), row = b % (BM / rows) * rows + (shares == 4 ? 0 : group);
        int mt, nt, ks;
        decode_unit(p, sh, tile, mt, nt, ks);
        const int64_t m = static_cast<int64_t>(mt) * BM + row, col = static_cast<int64_t>(nt) * BN + quad * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (m < limit) {
#pragma unroll 4
            for (int k = k0; k < k1; ++k) {
                const float4 f = *reinterpret_cast<const float4*>(p.split + ((static_cast<int64_t>(k) * tiles + tile) * BM + row) * BN + quad * 4);
                v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
            }
        }
        if (shares == 4) {
            part[share][quad] = v;
            __syncthreads();
#pragma unroll
            for (int i = 1; i < 4; ++i)
                if (share == 0) v.x += part[i][quad].x, v.y += part[i][quad].y, v.z += part[i][quad].z, v.w += part[i][quad].w;
            __syncthreads();
        }
        if (share != 0) continue;
        if (p.out_vec) {
            finish<EPI, 4>(p, m, limit, col, scale, v);
        } else {
            finish<EPI, 1>(p, m, limit, col, scale, make_float4(v.x, 0.0f, 0.0f, 0.0f));
            finish<EPI, 1>(p, m, limit, col + 1, scale, make_float4(v.y, 0.0f, 0.0f, 0.0f));
            finish<EPI, 1>(p, m, limit, col + 2, scale, make_float4(v.z, 0.0f, 0.0f, 0.0f));
            finish<EPI, 1>(p, m, limit, col + 3, scale, make_float4(v.w, 0.0f, 0.0f, 0.0f));
        }
    }
}

// ---- small kernels ---------------------------------------------------------------

__device__ __forceinline__ float load_f(const __half* p, int64_t i) { return __half2float(p[i]); }
__device__ __forceinline__ float load_f(const float* p, int64_t i) { return p[i]; }

constexpr int kIndexThreads = 1024;

// Lists the rows that have a target (in order), their targets, and their
// count; writes the ignored rows' losses (0) where there is one per row.
// kIndexRows: rows per thread and step (16384 rows: 23 us with one, 11 us with
// eight; up to 1024 rows 1.8 us with one).
template <int kIndexRows>
__global__ void __launch_bounds__(kIndexThreads)
ce_index_kernel(const int64_t* target, int64_t rows, int64_t vocab, int64_t ignore, int* index, int* packed_target, Scalars* sc,
                float* row_loss_out) {
    __shared__ int before[kIndexRows][32];  // listed rows of a step before each warp's
    __shared__ int total;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int base = 0;
    for (int64_t r0 = 0; r0 < rows; r0 += kIndexThreads * kIndexRows) {
        int64_t t[kIndexRows];
        unsigned used[kIndexRows];
#pragma unroll
        for (int k = 0; k < kIndexRows; ++k) {
            const int64_t r = r0 + k * kIndexThreads + threadIdx.x;
            t[k] = r < rows ? target[r] : ignore;
        }
#pragma unroll
        for (int k = 0; k < kIndexRows; ++k) {
            used[k] = __ballot_sync(0xFFFFFFFFu, t[k] != ignore);
            if (lane == 0) before[k][warp] = __popc(used[k]);
        }
        __syncthreads();
        if (warp == 0) {
            int sum = 0;
#pragma unroll
            for (int k = 0; k < kIndexRows; ++k) {
                const int v = before[k][lane];
                int s = v;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
                    if (lane >= d) s += o;
                }
                before[k][lane] = sum + s - v;
                sum += __shfl_sync(0xFFFFFFFFu, s, 31);
            }
            if (lane == 0) total = sum;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kIndexRows; ++k) {
            const int64_t r = r0 + k * kIndexThreads + threadIdx.x;
            if ((used[k] >> lane) & 1u) {
                const int at = base + before[k][warp] + __popc(used[k] & ((1u << lane) - 1u));
                index[at] = static_cast<int>(r);
                packed_target[at] = t[k] >= 0 && t[k] < vocab ? static_cast<int>(t[k]) : -1;  // -1: the loss is NaN
            } else if (r < rows && row_loss_out != nullptr) {
                row_loss_out[r] = 0.0f;
            }
        }
        base += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        sc->count = base;
        sc->amax_w = 0;
        sc->rows_done = 0;
    }
}

__device__ __forceinline__ unsigned finite_magnitude(float v) {
    const unsigned b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0u;
}

// Largest finite |v| of n consecutive values, shared out over `of` blocks.
__device__ __forceinline__ unsigned amax_span(const float* p, int64_t n, int64_t block, int64_t of) {
    unsigned top = 0;
    const int64_t head = min(n, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) / 4 % 4));  // up to a 16-byte boundary
    const int64_t quads = (n - head) / 4, tail = head + quads * 4;
    if (block == 0) {
        if (threadIdx.x < head) top = finite_magnitude(p[threadIdx.x]);
        if (tail + threadIdx.x < n) top = max(top, finite_magnitude(p[tail + threadIdx.x]));
    }
    const float4* q = reinterpret_cast<const float4*>(p + head);
    const int64_t step = of * blockDim.x;
    int64_t i = block * blockDim.x + threadIdx.x;
    for (; i + 3 * step < quads; i += 4 * step) {
        float4 f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = __ldg(q + i + k * step);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            top = max(max(top, max(finite_magnitude(f[k].x), finite_magnitude(f[k].y))), max(finite_magnitude(f[k].z), finite_magnitude(f[k].w)));
    }
    for (; i < quads; i += step) {
        const float4 f = __ldg(q + i);
        top = max(max(top, max(finite_magnitude(f.x), finite_magnitude(f.y))), max(finite_magnitude(f.z), finite_magnitude(f.w)));
    }
    return top;
}

// Largest finite |W|.
__global__ void __launch_bounds__(256) ce_amax_kernel(const float* w, int64_t n, Scalars* sc) {
    pdl_wait();
    unsigned top = amax_span(w, n, blockIdx.x, gridDim.x);
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0 && top != 0) atomicMax(&sc->amax_w, top);
}

// Eight consecutive elements of a row whose address is off a 16-byte boundary:
// whole 16-byte vectors around them, shifted into place (`begin` and `end` bound
// the tensor; vectors that would leave it, and the end of a row, go one element
// at a time).
template <typename T>
__device__ __forceinline__ void load8_any(const T* p, int64_t left, const void* begin, const void* end, float (&v)[8]) {
    constexpr int W = sizeof(T) == 2 ? 8 : 12;  // 32-bit words of the vectors read
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uintptr_t a = at & ~static_cast<uintptr_t>(15);
    if (left < 8 || a < reinterpret_cast<uintptr_t>(begin) || a + 4 * W > reinterpret_cast<uintptr_t>(end)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? load_f(p, i) : 0.0f;
        return;
    }
    uint32_t w[W + 2];
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(a + 16 * i);
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
    }
    w[W] = w[W + 1] = 0;
    const int shift = static_cast<int>(at - a) >> 2;
    if (shift & 2) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = w[i + 2];
    }
    if (shift & 1) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = w[i + 1];
    }
    if constexpr (sizeof(T) == 2) {
        const int half = at & 2 ? 16 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __funnelshift_r(w[i], w[i + 1], half);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
}

// Rows as binary16 planes, `ld` elements apart (a multiple of 8, zero past cols).
template <typename T>
struct PackJob {
    const T* src;
    const int* index;  // row r of the planes is row index[r] of src; NULL: r
    __half* dst;       // NULL: nothing to pack
    int64_t rows, cols, ld, plane;
    bool vec;          // 16-byte aligned rows, cols a multiple of 8
};

// Packs the octet at column c of the planes' row r from a row of src (NULL:
// zeros).
template <typename T, int PLANES>
__device__ __forceinline__ void pack_octet(const PackJob<T>& j, const T* from, int64_t r, int64_t c, float s) {
    __half* to = j.dst + r * j.ld + c;
    float v[8];
    if (from == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if (j.vec) {
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from + c);
            return;
        } else {
            const float4 a = *reinterpret_cast<const float4*>(from + c), b = *reinterpret_cast<const float4*>(from + c + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    } else {
        load8_any(from + c, j.cols - c, j.src, j.src + j.rows * j.cols, v);
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
    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(to + j.plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

template <typename T, int PLANES>
__device__ __forceinline__ void pack_row(const PackJob<T>& j, const T* from, int64_t r, float s) {
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * 8; c < j.ld; c += blockDim.x * 8) pack_octet<T, PLANES>(j, from, r, c, s);
}

// W's octets and the bias in base 2: blocks [0, w_blocks), the rest.  Octets are
// dealt out over rows, since a row may have few (110320 x 325 in fp16: 64 -> 32
// us against a row per block; 82545 x 64 in fp32: 22 -> 7).
template <typename T, int PLANES>
__device__ __forceinline__ void pack_weight_and_bias(const PackJob<T>& w, float s, int block, int w_blocks, const T* bias, float* bias2) {
    if (block < w_blocks) {
        const int64_t row = w.ld / 8, octets = w.rows * row, step = static_cast<int64_t>(w_blocks) * blockDim.x;
        int64_t i = static_cast<int64_t>(block) * blockDim.x + threadIdx.x;
        int64_t r = i / row, o = i - r * row;
        const int64_t dr = step / row, dn = step - dr * row;
#pragma unroll 2
        for (; i < octets; i += step) {
            pack_octet<T, PLANES>(w, w.src + r * w.cols, r, 8 * o, s);
            r += dr;
            o += dn;
            if (o >= row) {
                o -= row;
                ++r;
            }
        }
    } else {
        const int64_t i = static_cast<int64_t>(block - w_blocks) * blockDim.x + threadIdx.x;
        if (i < w.rows) bias2[i] = load_f(bias, i) * kLog2e;
    }
}

constexpr int kPackThreads = 128;

// What a row's planes are multiplied by: its largest value goes to [2^14, 2^15).
// A row of zeros takes the largest scale, so that it bounds no other row's.
__device__ __forceinline__ float row_scale(const float* row, int64_t cols) {
    __shared__ unsigned tops[kPackThreads / 32];
    const unsigned top = __reduce_max_sync(0xFFFFFFFFu, amax_span(row, cols, 0, 1));
    __syncthreads();  // the last row's maxima are read
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    unsigned all = 0;
    for (int i = 0; i < kPackThreads / 32; ++i) all = max(all, tops[i]);
    return all == 0 ? pow2(126) : plane_scale(all);
}

// Packs x's listed rows (zero rows after them up to a multiple of BK; blocks
// [0, x_blocks)), W where it is not read in place, and the bias in base 2.
template <typename T, int PLANES>
__global__ void __launch_bounds__(kPackThreads)
ce_pack_kernel(const PackJob<T> x, const PackJob<T> w, const Scalars* sc, int x_blocks, int w_blocks, const T* bias, float* bias2, float* xs) {
    pdl_wait();
    const int b = static_cast<int>(blockIdx.x);
    if (b >= x_blocks) {
        pack_weight_and_bias<T, PLANES>(w, PLANES == 2 ? plane_scale(sc->amax_w) : 1.0f, b - x_blocks, w_blocks, bias, bias2);
        return;
    }
    const int64_t live = sc->count;
    for (int64_t r = b; r < (live + BK - 1) / BK * BK; r += x_blocks) {
        const T* row = r < live ? x.src + static_cast<int64_t>(x.index[r]) * x.cols : nullptr;
        float s = 1.0f;
        if constexpr (PLANES == 2) {
            if (row != nullptr) s = row_scale(row, x.cols);
            if (threadIdx.x == 0) xs[r] = s;
        }
        pack_row<T, PLANES>(x, row, r, s);
    }
}

// ce_index_kernel and ce_pack_kernel in one launch, for up to 1024 rows of
// fp16: every block that packs a row lists the rows itself, block 0 writes the
// list down (8 rows by 30011 words, forward: kernels 23.0 -> 22.2 us, a pass 26.5
// -> 22.3).
constexpr int kListRows = 1024;

__global__ void __launch_bounds__(kPackThreads)
ce_list_pack_kernel(const int64_t* target, int rows, int64_t vocab, int64_t ignore, int* index, int* packed_target, Scalars* sc, float* row_loss_out,
                    const PackJob<__half> x, const PackJob<__half> w, int x_blocks, int w_blocks, const __half* bias, float* bias2) {
    pdl_wait();
    const int b = static_cast<int>(blockIdx.x);
    if (b >= x_blocks) {
        pack_weight_and_bias<__half, 1>(w, 1.0f, b - x_blocks, w_blocks, bias, bias2);
        return;
    }
    constexpr int WARPS = kPackThreads / 32, SPANS = kListRows / 32;
    __shared__ unsigned used[SPANS];
    __shared__ int before[SPANS], total, mine;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int s = warp; s < SPANS; s += WARPS) {
        const int r = s * 32 + lane;
        const unsigned u = __ballot_sync(0xFFFFFFFFu, r < rows && target[r] != ignore);
        if (lane == 0) used[s] = u;
    }
    __syncthreads();
    if (warp == 0) {
        const int v = __popc(used[lane]);
        int s = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
            if (lane >= d) s += o;
        }
        before[lane] = s - v;
        if (lane == 31) total = s;
    }
    __syncthreads();
    for (int s = warp; s < SPANS; s += WARPS) {
        const int r = s * 32 + lane;
        if ((used[s] >> lane) & 1u) {
            const int at = before[s] + __popc(used[s] & ((1u << lane) - 1u));
            if (at == b) mine = r;
            if (b == 0) {
                const int64_t t = target[r];
                index[at] = r;
                packed_target[at] = t >= 0 && t < vocab ? static_cast<int>(t) : -1;  // -1: the loss is NaN
            }
        } else if (b == 0 && r < rows && row_loss_out != nullptr) {
            row_loss_out[r] = 0.0f;
        }
    }
    __syncthreads();
    if (b == 0 && threadIdx.x == 0) {
        sc->count = total;
        sc->rows_done = 0;
    }
    if (b < (total + BK - 1) / BK * BK) pack_row<__half, 1>(x, b < total ? x.src + static_cast<int64_t>(mine) * x.cols : nullptr, b, 1.0f);
}
static_assert(kListRows == 32 * 32, "one warp sums the spans");

constexpr int kRowWarps = 8;

// A warp joins the statistics of a row and forms its loss: lse2 (base 2) for the
// backward pass, the loss per packed row, and per row where asked for.  The block that finishes last adds the losses of
// all rows, in a fixed order.
__global__ void __launch_bounds__(32 * kRowWarps)
ce_rows_kernel(const int* index, const int* target, Scalars* sc, const float2* part, int parts, const float* hit2, float* lse2, float* loss, int reduction,
               float* out) {
    pdl_wait();
    const int rows = sc->count;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int m = blockIdx.x * kRowWarps + warp; m < rows; m += gridDim.x * kRowWarps) {
        float top = -INFINITY, sum = 0.0f;
        const float2* row = part + static_cast<int64_t>(m) * parts;
#pragma unroll 4
        for (int i = lane; i < parts; i += 32) join(top, sum, row[i].x, row[i].y);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) join(top, sum, __shfl_xor_sync(0xFFFFFFFFu, top, k), __shfl_xor_sync(0xFFFFFFFFu, sum, k));
        if (lane == 0) {
            // top >= hit2 and sum >= 1: the loss is never negative
            const bool inside = target[m] >= 0;
            const float l2 = log2f(sum), v = inside ? (top - hit2[m] + l2) * kLn2 : NAN;
            lse2[m] = inside ? top + l2 : NAN;
            loss[m] = v;
            if (reduction == TK_REDUCE_NONE) out[index[m]] = v;
        }
    }
    if (reduction == TK_REDUCE_NONE) return;
    __shared__ bool last;
    __shared__ double total[kRowWarps];
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&sc->rows_done, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < rows; i += 32 * kRowWarps) s += __ldcg(loss + i);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, k);
    if (lane == 0) total[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int i = 0; i < kRowWarps; ++i) s += total[i];
        *out = static_cast<float>(reduction == TK_REDUCE_MEAN ? s / rows : s);  // no rows: 0 / 0, as torch's mean
    }
}

static_assert(kDzScale == 16384.0f, "2^14, in the exponents below");

constexpr int kNoTop = -100000;  // below every exponent of a finite x_i g_i

// Block 0: the gradients' scales, g_i per packed row where each has its own, and
// (fp32 operands) the largest exponent of x_i g_i.  The others: zero gradients
// for the ignored rows.
__global__ void __launch_bounds__(1024)
ce_grad_rows_kernel(const float* grad, int reduction, const int* index, const Scalars* sc, GradScalars* gs, float* grow, const float* xs,
                    const int64_t* target, int64_t ignore, int64_t all_rows, int64_t row_bytes, uint8_t* dx) {
    pdl_wait();
    if (blockIdx.x > 0) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int64_t r = (blockIdx.x - 1) * 32ll + warp; r < all_rows; r += (gridDim.x - 1) * 32ll) {
            if (target[r] != ignore) continue;
            uint8_t* o = dx + r * row_bytes;
            if (((reinterpret_cast<uintptr_t>(o) | row_bytes) & 15) == 0) {
                for (int64_t c = lane * 16; c < row_bytes; c += 32 * 16) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
            } else {
                for (int64_t c = lane * 2; c < row_bytes; c += 32 * 2) *reinterpret_cast<uint16_t*>(o + c) = 0;
            }
        }
        return;
    }
    const int rows = sc->count;
    const bool own = reduction == TK_REDUCE_NONE;
    int top = kNoTop;
    for (int i = threadIdx.x; i < rows && (own || xs != nullptr); i += 1024) {
        float g = 1.0f;
        if (own) grow[i] = g = grad[index[i]];
        if (xs != nullptr && g != 0.0f && isfinite(g)) top = max(top, 14 - exponent_of(xs[i]) + exponent_of(g));
    }
    __shared__ int tops[32];
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x < 32) top = __reduce_max_sync(0xFFFFFFFFu, tops[threadIdx.x]);
    if (threadIdx.x == 0) {
        // no rows: every sum is zero
        const float g = own ? 1.0f : rows == 0 ? 0.0f : reduction == TK_REDUCE_MEAN ? grad[0] / static_cast<float>(rows) : grad[0];
        const float unit = g / kDzScale;
        gs->db_scale = own ? 1.0f : unit;  // the sums take 2^(k_i - 14) row by row
        gs->dx_scale = xs != nullptr ? unit / plane_scale(sc->amax_w) : unit;
        gs->dw_scale = unit;  // ce_scale_rows_kernel adds the exponent of x's rows
        gs->top = top;
    }
}

// The largest exponent of x_i g_i over the packed rows of fp16 operands, a warp
// to a row.
__global__ void __launch_bounds__(256)
ce_top_kernel(const __half* x, int64_t ld, const Scalars* sc, GradScalars* gs, const float* grow) {
    pdl_wait();
    const int lane = threadIdx.x & 31, rows = sc->count;
    int top = kNoTop;
    for (int r = blockIdx.x * 8 + static_cast<int>(threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
        const float g = grow[r];
        if (g == 0.0f || !isfinite(g)) continue;
        uint32_t most = 0;  // binary16 bits of the row's largest finite |x|
        for (int64_t c = lane * 8; c < ld; c += 32 * 8) {
            const uint4 u = *reinterpret_cast<const uint4*>(x + r * ld + c);
            for (uint32_t w : {u.x, u.y, u.z, u.w})
                for (uint32_t h : {w & 0x7FFFu, w >> 16 & 0x7FFFu})
                    if (h < 0x7C00u) most = max(most, h);
        }
        most = __reduce_max_sync(0xFFFFFFFFu, most);
        if (most != 0) top = max(top, exponent_of(__half2float(__ushort_as_half(static_cast<unsigned short>(most)))) + exponent_of(g));
    }
    if (lane == 0) atomicMax(&gs->top, top);
}

// x's packed rows (zero rows up to a multiple of BK included) times 2^k_i, with
// one scale for all rows, the power of two that takes the largest into [2^14,
// 2^15), for dW.
template <int PLANES>
__global__ void __launch_bounds__(kPackThreads)
ce_scale_rows_kernel(const __half* x, __half* to, int64_t ld, int64_t plane, const Scalars* sc, GradScalars* gs, const float* grow, const float* xs) {
    pdl_wait();
    const int64_t live = sc->count;
    const int shift = gs->top > kNoTop ? 14 - gs->top : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {  // in two steps: the exponent can be past a power of two's
        const int half = shift / 2;
        gs->dw_scale = gs->dw_scale * pow2(-half) * pow2(half - shift);
    }
    for (int64_t r = blockIdx.x; r < (live + BK - 1) / BK * BK; r += gridDim.x) {
        const float g = r >= live ? 0.0f : grow != nullptr ? grow[r] : 1.0f;
        const int e = exponent_of(g) + shift - (PLANES == 2 && r < live ? exponent_of(xs[r]) : 0);
        const float a = g == 0.0f ? 0.0f : pow2(e / 2), b = pow2(e - e / 2);  // a row that `top` does not bound takes no part
        for (int64_t c = static_cast<int64_t>(threadIdx.x) * 8; c < ld; c += kPackThreads * 8) {
            const int64_t at = r * ld + c;
            const uint4 h = *reinterpret_cast<const uint4*>(x + at);
            uint4 l = make_uint4(0, 0, 0, 0);
            if constexpr (PLANES == 2) l = *reinterpret_cast<const uint4*>(x + plane + at);
            const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hs[t])), d = __half22float2(*reinterpret_cast<const __half2*>(&ls[t]));
                const float v0 = (f.x + d.x) * a * b, v1 = (f.y + d.y) * a * b;  // exact: hi + lo has 22 bits
                hi[t] = half2_bits(v0, v1);
                const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&hi[t]));
                lo[t] = half2_bits(isfinite(q.x) ? v0 - q.x : 0.0f, isfinite(q.y) ? v1 - q.y : 0.0f);
            }
            *reinterpret_cast<uint4*>(to + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(to + plane + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
}

constexpr int kDbThreads = 256;

// Column sums of a piece's dz, rows times 2^(k_i - 14) where each has its own
// gradient: chunk blockIdx.y of the rows, 8 columns per lane, 8 rows at a time,
// into partial[chunk][dz_ld].
__global__ void __launch_bounds__(kDbThreads)
ce_dbias_part_kernel(const __half* dz, int64_t dz_ld, int64_t dz_plane, const Scalars* sc, const float* grow, float* partial) {
    pdl_wait();
    __shared__ float sums[8][32][9];
    const int rows = sc->count;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 256 + lane * 8;
    const int lo = static_cast<int>(static_cast<int64_t>(blockIdx.y) * rows / gridDim.y);
    const int hi = static_cast<int>(static_cast<int64_t>(blockIdx.y + 1) * rows / gridDim.y);
    float s[8] = {};
    for (int64_t off = 0;; off = dz_plane) {
        const __half* d = dz + off + col;
        for (int r = lo + warp; r < hi; r += 32) {
            uint4 u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = r + 8 * k < hi ? *reinterpret_cast<const uint4*>(d + (r + 8 * k) * dz_ld) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __half2* h = reinterpret_cast<const __half2*>(&u[k]);
                const float a = grow != nullptr && r + 8 * k < hi ? pow2(exponent_of(grow[r + 8 * k]) - 14) : 1.0f;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float2 f = __half22float2(h[t]);
                    s[2 * t] = fmaf(f.x, a, s[2 * t]);
                    s[2 * t + 1] = fmaf(f.y, a, s[2 * t + 1]);
                }
            }
        }
        if (off == dz_plane) break;
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
ce_dbias_kernel(const float* partial, int chunks, int64_t dz_ld, int64_t cols, const GradScalars* gs, void* out, int out_f32) {
    pdl_wait();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int i = 0; i < chunks; ++i) s += partial[i * dz_ld + c];
    s *= gs->db_scale;
    if (out_f32) {
        static_cast<float*>(out)[c] = s;
    } else {
        static_cast<__half*>(out)[c] = __float2half_rn(s);
    }
}

// ---- host --------------------------------------------------------------------------

constexpr int64_t kDzBytes = 512ll << 20;   // one piece's dz
constexpr int64_t kMaxSize = 0x7FFFFF00, kMaxTiles = 1 << 30;

size_t align(size_t v) { return round_up(v, 1024); }

struct Plan {
    bool f16;
    bool w_kept;             // W is packed into the state: by type and width, never by address
    bool w_direct;           // W is read in place; neither: packed into the workspace of each pass
    int planes;
    int64_t rows_pad, ld;    // packed rows and their length
    int64_t rows_read;       // rows that the products read; tiles end in zeros of their own
    int64_t n_tiles;         // vocabulary tiles
    int64_t piece;           // vocabulary columns per piece (a multiple of BN)
    int64_t pieces;
    int64_t acc_ld;
    int64_t parts;           // statistics per row
    int split_units;
    int db_chunks;
    // state: kept from the forward to the backward pass
    size_t s_scalars, s_index, s_target, s_lse, s_xs, s_x, s_bias, s_w, state_bytes;
    // workspaces
    size_t w_part, w_hit, w_loss, w_w, fwd_bytes;
    size_t b_scalars, b_grow, b_dz, b_acc, b_split, b_db, b_w, b_x, bwd_bytes;
};

int check(const char* who, const tk_linear_ce_desc_t& d) {
    TK_CHECK_ARG(d.dtype == TK_DTYPE_F16 || d.dtype == TK_DTYPE_F32, "%s: bad dtype %d", who, static_cast<int>(d.dtype));
    TK_CHECK_ARG(d.reduction == TK_REDUCE_NONE || d.reduction == TK_REDUCE_MEAN || d.reduction == TK_REDUCE_SUM, "%s: bad reduction %d", who, d.reduction);
    TK_CHECK_ARG(d.rows >= 0 && d.cols >= 1 && d.vocab >= 1, "%s: rows must not be negative, cols and vocab must be positive", who);
    if (d.rows > kMaxSize || d.cols > kMaxSize || d.vocab > kMaxSize) TK_FAIL(TK_ERR_UNSUPPORTED, "%s: sizes must be below 2^31 - 256", who);
    const int64_t m = ceil_div(d.rows, BM), n = ceil_div(d.vocab, BN), k = ceil_div(d.cols, BN);
    if (m * n > kMaxTiles || m * k > kMaxTiles || n * k > kMaxTiles) TK_FAIL(TK_ERR_UNSUPPORTED, "%s: a product has more than 2^30 tiles of 256 x 256", who);
    return TK_OK;
}

template <int EPI>
Mode mode_of(int planes, int64_t k_blocks) {
    if (planes == 2) return k_blocks <= kChunkF32 ? kPlanesWide : kPlanes;
    if ((EPI == kStats || EPI == kDlogits) && k_blocks > kChunkStats) return kChunked;
    if (EPI == kStats) return kPlain;
    return (EPI == kDlogits || EPI == kGradW) && k_blocks <= kWideBlocks ? kWide : kPlain;
}

// Statistics per row and tile.
int stats_parts(int planes, int64_t cols) {
    const Mode m = mode_of<kStats>(planes, ceil_div(cols, BK));
    return BN / (m == kPlanesWide ? Config<kPlanesWide>::COLS : Config<kChunked>::COLS);
}

Plan make_plan(const tk_linear_ce_desc_t& d) {
    Plan p = {};
    p.f16 = d.dtype == TK_DTYPE_F16;
    p.planes = p.f16 ? 1 : 2;
    p.rows_pad = static_cast<int64_t>(round_up(static_cast<size_t>(std::max<int64_t>(d.rows, 1)), kRowPad));
    p.rows_read = static_cast<int64_t>(round_up(static_cast<size_t>(std::max<int64_t>(d.rows, 1)), BK));
    p.ld = static_cast<int64_t>(round_up(static_cast<size_t>(d.cols), 8));
    // The state's layout follows from sizes and types alone: the backward pass
    // may see the weight at another address than the forward pass did.
    p.w_kept = !p.f16 || d.cols % 8 != 0;
    p.w_direct = !p.w_kept && (reinterpret_cast<uintptr_t>(d.weight) & 15) == 0;
    const size_t w_bytes = static_cast<size_t>(p.planes) * d.vocab * p.ld * 2;
    p.n_tiles = ceil_div(d.vocab, BN);
    // pieces of equal size whose dz planes fit kDzBytes (one tile at least)
    const int64_t most = std::max<int64_t>(1, kDzBytes / (p.rows_pad * 2 * p.planes * BN));
    p.pieces = ceil_div(p.n_tiles, most);
    p.piece = ceil_div(p.n_tiles, p.pieces) * BN;
    p.pieces = ceil_div(p.n_tiles * BN, p.piece);
    p.acc_ld = static_cast<int64_t>(round_up(static_cast<size_t>(d.cols), 4));
    p.split_units = sm_count(current_device());  // two per pair of CTAs
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
    p.s_xs = take(p.planes == 2 ? p.rows_pad * sizeof(float) : 0);
    p.s_x = take(static_cast<size_t>(p.planes) * p.rows_pad * p.ld * 2);
    p.s_bias = take(static_cast<size_t>(d.vocab) * sizeof(float));  // with a bias or without
    p.s_w = take(p.w_kept ? w_bytes : 0);
    p.state_bytes = at;
    at = 0;
    p.parts = stats_parts(p.planes, d.cols) * p.n_tiles;
    p.w_part = take(static_cast<size_t>(p.parts) * p.rows_pad * sizeof(float2));
    p.w_hit = take(p.rows_pad * sizeof(float));
    p.w_loss = take(p.rows_pad * sizeof(float));
    p.w_w = take(p.w_kept || p.w_direct ? 0 : w_bytes);
    p.fwd_bytes = at + p.state_bytes;  // a call without a state keeps its own
    at = 0;
    const bool own = d.reduction == TK_REDUCE_NONE;  // each row has its own gradient
    p.b_scalars = take(sizeof(GradScalars));
    p.b_grow = take(own ? p.rows_pad * sizeof(float) : 0);
    p.b_x = take(own || p.planes == 2 ? static_cast<size_t>(p.planes) * p.rows_pad * p.ld * 2 : 0);
    p.b_dz = take(static_cast<size_t>(p.planes) * p.rows_pad * p.piece * 2);
    p.b_acc = take(p.pieces > 1 ? static_cast<size_t>(p.rows_pad) * p.acc_ld * sizeof(float) : 0);
    p.b_split = take(static_cast<size_t>(p.split_units) * BM * BN * sizeof(float));
    p.b_db = take(d.bias != nullptr ? static_cast<size_t>(p.db_chunks) * p.piece * sizeof(float) : 0);
    p.b_w = take(p.w_kept || p.w_direct ? 0 : w_bytes);
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

template <int EPI, int MODE>
int gemm_launch(const CUtensorMap& a, const CUtensorMap& b, const GemmParams& p, int64_t most_units, cudaStream_t s) {
    auto* kernel = ce_gemm_kernel<EPI, MODE>;
    static std::atomic<int> resident[64];  // pairs of CTAs each device holds at once; 0: not asked yet
    const int device = current_device();
    int pairs = device < 64 ? resident[device].load(std::memory_order_relaxed) : 0;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(Config<MODE>::THREADS);
    cfg.dynamicSmemBytes = Config<MODE>::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (pairs == 0) {
        TK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Config<MODE>::SMEM));
        TK_CUDA_TRY(cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg));
        if (pairs < 1) TK_FAIL(TK_ERR_CUDA, "cross entropy GEMM: no pair of CTAs fits the GPU");
        if (device < 64) resident[device].store(pairs, std::memory_order_relaxed);
    }
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::max<int64_t>(1, std::min<int64_t>(pairs, most_units))));
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, b, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        TK_FAIL(TK_ERR_CUDA, "cross entropy GEMM launch failed: %s", cudaGetErrorString(e));
    }
    return TK_OK;
}

// k_most: the most K blocks there can be, where the device's list decides.
template <int EPI>
int gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmParams& p, int64_t most_units, cudaStream_t s, int64_t k_most = 0) {
    switch (mode_of<EPI>(p.planes, p.k_blocks >= 0 ? p.k_blocks : k_most)) {
        case kPlanes: return gemm_launch<EPI, kPlanes>(a, b, p, most_units, s);
        case kPlanesWide: return gemm_launch<EPI, kPlanesWide>(a, b, p, most_units, s);
        case kWide: return gemm_launch<EPI, EPI == kDlogits || EPI == kGradW ? kWide : kPlain>(a, b, p, most_units, s);
        case kChunked: return gemm_launch<EPI, EPI == kStats || EPI == kDlogits ? kChunked : kPlain>(a, b, p, most_units, s);
        default: return gemm_launch<EPI, kPlain>(a, b, p, most_units, s);
    }
}

int blocks_for(int64_t rows) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, 148 * 16))); }

// W as planes at `to`.
template <typename T>
PackJob<T> weight_job(const tk_linear_ce_desc_t& d, const Plan& p, __half* to) {
    return {static_cast<const T*>(d.weight), nullptr, to, d.vocab, d.cols, p.ld, d.vocab * p.ld,
            d.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(d.weight) & 15) == 0};
}

int weight_blocks(const tk_linear_ce_desc_t& d, const Plan& p) {
    return p.w_direct ? 0 : blocks_for(ceil_div(d.vocab * (p.ld / 8), kPackThreads));
}

// The list of rows, x's listed rows, W unless it is read in place (to `w_at`),
// and the bias.
template <typename T, int PLANES>
int list_and_pack(const tk_linear_ce_desc_t& d, const Plan& p, uint8_t* st, uint8_t* w_at, cudaStream_t s) {
    const T* x = static_cast<const T*>(d.x);
    const T* bias = static_cast<const T*>(d.bias);
    Scalars* sc = reinterpret_cast<Scalars*>(st + p.s_scalars);
    int* index = reinterpret_cast<int*>(st + p.s_index);
    int* target = reinterpret_cast<int*>(st + p.s_target);
    float* bias2 = reinterpret_cast<float*>(st + p.s_bias);
    float* row_loss = d.reduction == TK_REDUCE_NONE ? d.loss : nullptr;
    const PackJob<T> jx = {x, index, reinterpret_cast<__half*>(st + p.s_x), d.rows, d.cols, p.ld, p.rows_pad * p.ld,
                           d.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0};
    const PackJob<T> jw = weight_job<T>(d, p, reinterpret_cast<__half*>(w_at));
    const int w_blocks = weight_blocks(d, p);
    const int64_t b_blocks = d.bias != nullptr ? ceil_div(d.vocab, kPackThreads) : 0;
    if constexpr (PLANES == 1) {
        if (d.rows > 0 && d.rows <= kListRows) {
            const int x_blocks = static_cast<int>(p.rows_read);
            return launch_chain("cross entropy pack", ce_list_pack_kernel, dim3(static_cast<unsigned>(x_blocks + w_blocks + b_blocks)), dim3(kPackThreads),
                                0, s, d.target, static_cast<int>(d.rows), d.vocab, d.ignore_index, index, target, sc, row_loss, jx, jw, x_blocks,
                                w_blocks, bias, bias2);
        }
    }
    auto* list = d.rows <= kIndexThreads ? ce_index_kernel<1> : ce_index_kernel<8>;
    list<<<1, kIndexThreads, 0, s>>>(d.target, d.rows, d.vocab, d.ignore_index, index, target, sc, row_loss);
    CE_TRY(launch_status("cross entropy index"));
    if (d.rows == 0) return TK_OK;
    if constexpr (PLANES == 2)
        CE_TRY(launch_chain("cross entropy amax", ce_amax_kernel, dim3(148 * 4), dim3(256), 0, s, jw.src, d.vocab * d.cols, sc));
    const int x_blocks = blocks_for(p.rows_read);
    return launch_chain("cross entropy pack", ce_pack_kernel<T, PLANES>, dim3(static_cast<unsigned>(x_blocks + w_blocks + b_blocks)), dim3(kPackThreads), 0,
                        s, jx, jw, static_cast<const Scalars*>(sc), x_blocks, w_blocks, bias, bias2, reinterpret_cast<float*>(st + p.s_xs));
}

int rows_loss(const tk_linear_ce_desc_t& d, const Plan& p, uint8_t* st, uint8_t* ws, cudaStream_t s) {
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(d.rows, kRowWarps), 148 * 8)));
    return launch_chain("cross entropy rows", ce_rows_kernel, dim3(grid), dim3(32 * kRowWarps), 0, s, reinterpret_cast<const int*>(st + p.s_index),
                        reinterpret_cast<const int*>(st + p.s_target), reinterpret_cast<Scalars*>(st + p.s_scalars),
                        reinterpret_cast<const float2*>(ws + p.w_part), static_cast<int>(p.parts), reinterpret_cast<const float*>(ws + p.w_hit),
                        reinterpret_cast<float*>(st + p.s_lse), reinterpret_cast<float*>(ws + p.w_loss), static_cast<int>(d.reduction), d.loss);
}

struct Operand {
    const uint8_t* base;
    int64_t ld, plane;
};

Operand weight_operand(const tk_linear_ce_desc_t& d, const Plan& p, const uint8_t* w_at) {
    if (p.w_direct) return {static_cast<const uint8_t*>(d.weight), d.cols, d.vocab * d.cols};
    return {w_at, p.ld, d.vocab * p.ld};
}

GemmParams base_params(const tk_linear_ce_desc_t& d, const Plan& p, const uint8_t* st) {
    GemmParams g = {};
    g.sc = reinterpret_cast<const Scalars*>(st + p.s_scalars);
    g.planes = p.planes;
    g.chunk = p.planes == 2 ? kChunkF32 : kChunkStats;
    g.m_tiles = -1;
    g.k_blocks = static_cast<int>(ceil_div(d.cols, BK));
    g.group = 8;
    g.max_units = p.split_units;
    g.err = device_error_word(current_device());
    g.xs = p.planes == 2 ? reinterpret_cast<const float*>(st + p.s_xs) : nullptr;
    g.bias2 = d.bias != nullptr ? reinterpret_cast<const float*>(st + p.s_bias) : nullptr;
    g.vocab = d.vocab;
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
    uint8_t* w_at = p.w_kept ? st + p.s_w : ws + p.w_w;
    if (p.f16) {
        CE_TRY((list_and_pack<__half, 1>(d, p, st, w_at, s)));
    } else {
        CE_TRY((list_and_pack<float, 2>(d, p, st, w_at, s)));
    }
    if (d.rows > 0) {
        const Operand w = weight_operand(d, p, w_at);
        CUtensorMap tx, tw;
        CE_TRY(make_map(&tx, st + p.s_x, d.cols, p.rows_read, p.planes, p.ld, p.rows_pad * p.ld, HM));
        CE_TRY(make_map(&tw, w.base, d.cols, d.vocab, p.planes, w.ld, w.plane, HN));
        GemmParams g = base_params(d, p, st);
        g.n_tiles = static_cast<int>(p.n_tiles);
        g.part = reinterpret_cast<float2*>(ws + p.w_part);
        g.hit2 = reinterpret_cast<float*>(ws + p.w_hit);
        g.target = reinterpret_cast<const int*>(st + p.s_target);
        CE_TRY(gemm<kStats>(tx, tw, g, p.n_tiles * ceil_div(d.rows, BM), s));
    }
    if (d.rows > 0 || d.reduction != TK_REDUCE_NONE) CE_TRY(rows_loss(d, p, st, ws, s));
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
    TK_CHECK_ARG(d.weight && d.target && d.state && desc->grad_loss, "tk_linear_ce_backward: NULL pointer");
    TK_CHECK_ARG((reinterpret_cast<uintptr_t>(d.state) & 15) == 0, "tk_linear_ce_backward: state must be 16-byte aligned");
    const Plan p = make_plan(d);
    if (workspace == nullptr || workspace_bytes < p.bwd_bytes || (reinterpret_cast<uintptr_t>(workspace) & 1023) != 0)
        TK_FAIL(TK_ERR_WORKSPACE, "tk_linear_ce_backward: 1024-byte aligned workspace of %zu bytes needed, got %zu", p.bwd_bytes, workspace_bytes);
    if (!desc->dx && !desc->dweight && !desc->dbias) return TK_OK;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint8_t* st = static_cast<uint8_t*>(d.state);
    const Scalars* sc = reinterpret_cast<const Scalars*>(st + p.s_scalars);
    const int* index = reinterpret_cast<const int*>(st + p.s_index);
    GradScalars* gs = reinterpret_cast<GradScalars*>(ws + p.b_scalars);
    const bool own = d.reduction == TK_REDUCE_NONE;
    const float* xs = p.planes == 2 ? reinterpret_cast<const float*>(st + p.s_xs) : nullptr;
    float* grow = own ? reinterpret_cast<float*>(ws + p.b_grow) : nullptr;
    __half* dz = reinterpret_cast<__half*>(ws + p.b_dz);
    const size_t esz = dtype_size(d.dtype);
    const int zero_blocks = desc->dx != nullptr ? static_cast<int>(std::min<int64_t>(ceil_div(d.rows, 32), 148 * 2)) : 0;
    CE_TRY(launch_chain("cross entropy gradient rows", ce_grad_rows_kernel, dim3(static_cast<unsigned>(1 + zero_blocks)), dim3(1024), 0, s,
                        desc->grad_loss, static_cast<int>(d.reduction), index, sc, gs, grow, xs, d.target, d.ignore_index, d.rows,
                        static_cast<int64_t>(d.cols * esz), static_cast<uint8_t*>(desc->dx)));
    uint8_t* w_at = p.w_kept ? st + p.s_w : ws + p.b_w;
    if (!p.w_kept && !p.w_direct) {
        CE_TRY(launch_chain("cross entropy pack", ce_pack_kernel<__half, 1>, dim3(static_cast<unsigned>(weight_blocks(d, p))), dim3(kPackThreads), 0, s,
                            PackJob<__half>{}, weight_job<__half>(d, p, reinterpret_cast<__half*>(w_at)), sc, 0,
                            weight_blocks(d, p), static_cast<const __half*>(nullptr), static_cast<float*>(nullptr), static_cast<float*>(nullptr)));
    }
    const Operand w = weight_operand(d, p, w_at);
    const int64_t x_plane = p.rows_pad * p.ld, dz_plane = p.rows_pad * p.piece;
    const __half* x_dw = reinterpret_cast<const __half*>(st + p.s_x);
    if ((own || p.planes == 2) && desc->dweight) {
        __half* to = reinterpret_cast<__half*>(ws + p.b_x);
        if (p.planes == 1)
            CE_TRY(launch_chain("cross entropy row exponents", ce_top_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(d.rows, 8), 148 * 8))), dim3(256),
                                0, s, x_dw, p.ld, sc, gs, static_cast<const float*>(grow)));
        CE_TRY(launch_chain("cross entropy row scales", p.planes == 2 ? ce_scale_rows_kernel<2> : ce_scale_rows_kernel<1>,
                            dim3(static_cast<unsigned>(blocks_for(p.rows_read))), dim3(kPackThreads), 0, s, x_dw, to, p.ld, x_plane, sc, gs,
                            static_cast<const float*>(grow), xs));
        x_dw = to;
    }
    CUtensorMap tx, tx_mn;
    CE_TRY(make_map(&tx, st + p.s_x, d.cols, p.rows_read, p.planes, p.ld, x_plane, HM));
    CE_TRY(make_map(&tx_mn, x_dw, d.cols, p.rows_read, p.planes, p.ld, x_plane, BK));
    const int64_t row_tiles = ceil_div(d.rows, BM), col_tiles = ceil_div(d.cols, BN);
    const bool cols16 = d.cols * esz % 16 == 0;
    for (int64_t i = 0; i < p.pieces; ++i) {
        const int64_t v0 = i * p.piece, width = std::min(p.piece, d.vocab - v0);
        const uint8_t* wbase = w.base + v0 * w.ld * 2;
        CUtensorMap tw, tw_mn, tdz, tdz_mn;
        CE_TRY(make_map(&tw, wbase, d.cols, width, p.planes, w.ld, w.plane, HN));
        CE_TRY(make_map(&tw_mn, wbase, d.cols, width, p.planes, w.ld, w.plane, BK));
        CE_TRY(make_map(&tdz, dz, width, p.rows_read, p.planes, p.piece, dz_plane, HM));
        CE_TRY(make_map(&tdz_mn, dz, width, p.rows_read, p.planes, p.piece, dz_plane, BK));
        GemmParams g = base_params(d, p, st);
        g.n_tiles = static_cast<int>(ceil_div(width, BN));
        g.vocab0 = v0;
        g.lse2 = reinterpret_cast<const float*>(st + p.s_lse);
        g.grow = grow;
        g.target = reinterpret_cast<const int*>(st + p.s_target);
        g.dz = dz;
        g.dz_ld = p.piece;
        g.dz_plane = p.planes == 2 ? dz_plane : 0;
        CE_TRY(gemm<kDlogits>(tx, tw, g, row_tiles * g.n_tiles, s));
        if (desc->dbias) {
            float* part = reinterpret_cast<float*>(ws + p.b_db);
            CE_TRY(launch_chain("cross entropy bias sums", ce_dbias_part_kernel, dim3(static_cast<unsigned>(p.piece / 256), p.db_chunks), dim3(kDbThreads), 0, s,
                                static_cast<const __half*>(dz), p.piece, g.dz_plane, sc, static_cast<const float*>(grow), part));
            CE_TRY(launch_chain("cross entropy bias sums", ce_dbias_kernel, dim3(static_cast<unsigned>(ceil_div(width, 256))), dim3(256), 0, s,
                                static_cast<const float*>(part), p.db_chunks, p.piece, width, static_cast<const GradScalars*>(gs),
                                static_cast<void*>(static_cast<uint8_t*>(desc->dbias) + v0 * esz), p.f16 ? 0 : 1));
        }
        GemmParams r = base_params(d, p, st);
        r.gs = gs;
        r.grow = grow;
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
            r.acc_ld = p.acc_ld;
            r.first = i == 0;
            r.last = i + 1 == p.pieces;
            CE_TRY(gemm<kGradX>(tdz, tw_mn, r, std::max<int64_t>(row_tiles * col_tiles, p.split_units), s));
            CE_TRY(launch_chain("cross entropy split", ce_split_kernel<kGradX>, dim3(static_cast<unsigned>(p.split_units) * 8), dim3(256), 0, s, r));
        }
        if (desc->dweight) {
            r.m_tiles = static_cast<int>(ceil_div(width, BM));
            r.k_blocks = -1;
            r.out = static_cast<uint8_t*>(desc->dweight) + v0 * d.cols * esz;
            r.out_vec = cols16 && (reinterpret_cast<uintptr_t>(r.out) & 15) == 0;
            r.out_rows = width;
            CE_TRY(gemm<kGradW>(tdz_mn, tx_mn, r, std::max<int64_t>(r.m_tiles * col_tiles, p.split_units), s, ceil_div(d.rows, BK)));
            if (2 * r.m_tiles * col_tiles <= p.split_units)  // else no tile is split
                CE_TRY(launch_chain("cross entropy split", ce_split_kernel<kGradW>, dim3(static_cast<unsigned>(p.split_units) * 8), dim3(256), 0, s, r));
        }
    }
    return TK_OK;
}

}  // extern "C"
