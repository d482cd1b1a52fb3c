// mx4_common.hpp -- rows in the OCP microscaling format MXFP4: their arithmetic, their layout, what the kernels share (gfx950).
//
// The arithmetic.  A block of 32 elements shares E = clamp(floor(log2 max|x|) - 2, -127, 125); its elements are E2M1 codes of
// x 2^-E, nearest with ties to even, saturating at 6.  The scale byte is E + 127; a block that holds an infinity or a NaN has
// byte 255 and is NaN as a whole.  Queries are rounded the same way to E2M1 (4 bits) or E2M3 (6 bits, saturating at 7.5).
//   dot(q, x) = sum_blocks 2^(Eq + Ex) sum_j q_j x_j      IP 1 - dot    L2 |q|^2 + |x|^2 - 2 dot    Cosine 1 - dot / (|q| |x|)
// (|.| of the rounded vectors).  A block's inner sum is a multiple of 1/16 below 2^11, so it is exact in fp32, whatever the order.
// E2M3 and not E4M3 for the finer queries: at a block's own scale both keep four digits of its larger elements, the matrix
// instruction takes six-bit operands at the four-bit rate, and it adds up a block of their products exactly (what it does with blocks
// far apart: mx4_slack), where E4M3 products came back up to 3e-4 of the largest product off.
//
// The layout.  32 rows form a panel, laid out as v_mfma_scale_f32_32x32x64_f8f6f4 takes its operand, so that a wave's load of one
// k-step (64 elements of 32 rows) is one contiguous KiB straight into registers, without a pass through LDS:
//   codes  [ks = ceil(dim / 64)][half][row][16 bytes]    element j of block 2 step + half in byte j / 2, low nibble first
//   scales [kg = ceil(ks / 4)][half][row][4 bytes]       byte i: k-step 4 group + i; one dword feeds four instructions (opsel)
//   norms  [32] fp32                                     |x|, rounded once from 64 bits; the sign bit is free (k_mx4_claim)
// 768 elements: 412 bytes a row.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vsg {

typedef int mx4_i4 __attribute__((ext_vector_type(4)));
typedef int mx4_i8 __attribute__((ext_vector_type(8)));
typedef float mx4_f16 __attribute__((ext_vector_type(16)));
typedef float mx4_f4 __attribute__((ext_vector_type(4)));
typedef unsigned int mx4_u4 __attribute__((ext_vector_type(4)));
typedef int mx4_i2 __attribute__((ext_vector_type(2)));
typedef unsigned int mx4_u2 __attribute__((ext_vector_type(2)));
typedef unsigned int mx4_u6 __attribute__((ext_vector_type(6)));
typedef float mx4_f2 __attribute__((ext_vector_type(2)));
typedef float mx4_f32 __attribute__((ext_vector_type(32)));

enum { MX4_F32 = 0, MX4_BF16 = 2, MX4_F16 = 3 };   // VSGPU_F32, _BF16, _F16
enum { MX4_L2 = 0, MX4_IP = 1, MX4_COSINE = 2 };

__host__ __device__ inline uint32_t mx4_steps(uint32_t dim) { return (dim + 63) / 64; }
__host__ __device__ inline uint32_t mx4_groups(uint32_t dim) { return (mx4_steps(dim) + 3) / 4; }
__host__ __device__ inline uint32_t mx4_panel(uint32_t dim) { return mx4_steps(dim) * 1024 + mx4_groups(dim) * 256 + 128; }
// a 32-query tile of the query block: operand bytes of every k-step (16 a lane; E2M3: 8 more a lane behind all of them), scales.
// Whole groups of four steps, zero beyond the last one: a scan multiplies whole groups (the rows' scale bytes there are zero too)
__host__ __device__ inline uint32_t mx4_qtile(uint32_t dim, int bits) { return mx4_groups(dim) * (bits == 6 ? 4 * 1536 + 256 : 4 * 1024 + 256); }

// where rows are: one block of panels, or slabs of 2^shift panels each
struct Mx4Rows {
    char *base;
    char *const *slabs;
    uint32_t shift;
    uint32_t dim, ks, kg, panel;
    uint64_t n;
    // p the same for the whole wave: the slab's address comes through the scalar cache, apart from the loads in flight
    __device__ __forceinline__ uint64_t uniform_at(uint64_t p) const {
        if (!slabs) return reinterpret_cast<uint64_t>(base) + p * panel;
        typedef const __attribute__((address_space(4))) uint64_t *Scalar;
        return ((Scalar)(uintptr_t)slabs)[p >> shift] + (p & ((1u << shift) - 1)) * (size_t)panel;
    }
    __device__ char *at(uint64_t p) const {
        if (slabs) return slabs[p >> shift] + (p & ((1u << shift) - 1)) * (size_t)panel;
        return base + p * panel;
    }
};

// ---------------------------------------------------------------------------------------------------------------- scan
// How far a matrix-core dot may be from the exact one, over |q| |x|.  An instruction adds two blocks, each the exact sum of its 32
// products, to the sum so far and rounds once (2^-24), but leaves a block out when its scales' power of two is 2^32 or more below the
// largest of what it adds: up to 32 x 7.5 x 6 x 2^-32 = 2^-21.51 of that, for each of the two (the largest error of 6 x 10^7 random and
// extreme instructions: 2^-20.508).  Sums whose every step loses that, in one direction, exist, so a step counts with 2^-20, a third
// more than both; eight more steps for the rounded norms, the comparison's own arithmetic and subnormal dots.
__host__ __device__ inline float mx4_slack(uint32_t ks) { return (float)(ks + 8) * 9.5367431640625e-7f; }
constexpr float MX4_EPS = 1.9073486328125e-6f;    // 2^-19, of |q|^2 + |x|^2 (L2): the same for sums of squares
constexpr float MX4_STEP = 9.5367431640625e-7f;   // 2^-20: what rounding a score to fp32 may move it, and more
constexpr float MX4_TINY = 1e-36f;                // L2 scores below it: fp32 has no digits left to rank them by
constexpr float MX4_SHORT = 1e-18f;               // Cosine of shorter vectors: the product of the norms may leave fp32
constexpr float MX4_LONG = 4.611686018427388e18f; // 2^62: a dot of longer vectors may, as a whole or in one of its partial sums

enum { MX4_PROBE = 0, MX4_PROBE_ROWS = 1, MX4_FILTER = 2, MX4_DENSE = 3 };
constexpr uint32_t MX4_SEGMENTS = 1024;           // parts of a query's candidate list at most: one for each workgroup of the filter
struct Mx4Cand {
    uint32_t row;
    float dot, x;                 // of the matrix cores, |x|
};
struct Mx4Scan {
    Mx4Rows rows;
    const char *tiles;            // the queries' operand tiles: a workgroup takes groups x QT of them from blockIdx.y on
    uint32_t qtile_bytes;
    uint32_t nq, metric;
    uint32_t groups;              // waves that share a panel, each with its own query tiles
    const float *qnorm;
    const double *qsq;            // DENSE: |q|^2
    uint64_t n_take;              // panels: all of them, or for a probe number i is (i * every) >> 24
    uint64_t every;
    float *minima;                // PROBE: [nq][2 n_take] upper bounds of 16 rows each; PROBE_ROWS: [nq][n] of each row
    uint64_t minima_stride;
    const float2 *limit;          // FILTER: {alpha, beta} of each query
    uint32_t *counts;             // FILTER: [nq][segments]
    Mx4Cand *cand;                // [nq][segments][segment]
    uint32_t segments, segment;
    float *out;                   // DENSE: [nq][out_stride]
    uint64_t out_stride;
    float slack;
};

// the score's bounds from a matrix-core dot and the two norms
__device__ __forceinline__ void mx4_bounds(uint32_t metric, float d, float x, float y, float slack, float &low, float &up) {
    float s, e;
    if (metric == MX4_L2) {
        const float sum = __fmaf_rn(x, x, y * y);
        s = __fmaf_rn(-2.f, d, sum);
        e = __fmaf_rn(2.f * slack * x, y, __fmaf_rn(MX4_EPS, sum, MX4_TINY));
    } else if (metric == MX4_IP) {
        s = 1.f - d;
        e = __fmaf_rn(slack * x, y, MX4_STEP * fmaxf(1.f, fabsf(s)));
    } else {
        s = 1.f - d / x / y;
        e = slack + MX4_STEP;
        if (x < MX4_SHORT || y < MX4_SHORT) s = 1.f, e = 1.001f;
    }
    if (x > MX4_LONG || y > MX4_LONG) s = 0.f, e = __uint_as_float(0x7F800000u);
    low = s - e;
    up = s + e;
}

// a lower bound from the upper one
__device__ __forceinline__ float mx4_low(uint32_t metric, float up, float x, float y, float slack) {
    if (x > MX4_LONG || y > MX4_LONG) return -__uint_as_float(0x7F800000u);
    if (metric == MX4_L2) return up - 2.f * __fmaf_rn(2.f * slack * x, y, __fmaf_rn(2.f * MX4_EPS, __fmaf_rn(x, x, y * y), MX4_TINY));
    if (metric == MX4_IP) return up - 2.f * __fmaf_rn(2.f * slack * x, y, 2.f * MX4_STEP * fmaxf(1.f, fabsf(up)));
    return x < MX4_SHORT || y < MX4_SHORT ? -1.f : up - 4.f * (slack + MX4_STEP);
}

}  // namespace vsg
