// mx4_kernels.hpp -- rows in the OCP microscaling format MXFP4: writing, reading back, scoring, the k best (gfx950).
//
// The arithmetic.  A block of 32 elements shares E = clamp(floor(log2 max|x|) - 2, -127, 125); its elements are E2M1 codes of
// x 2^-E, nearest with ties to even, saturating at 6.  The scale byte is E + 127; a block that holds an infinity or a NaN has
// byte 255 and is NaN as a whole.  Queries are rounded the same way to E2M1 (4 bits) or E2M3 (6 bits, saturating at 7.5).
//   dot(q, x) = sum_blocks 2^(Eq + Ex) sum_j q_j x_j      IP 1 - dot    L2 |q|^2 + |x|^2 - 2 dot    Cosine 1 - dot / (|q| |x|)
// (|.| of the rounded vectors).  A block's inner sum is a multiple of 1/16 below 2^11, so it is exact in fp32, whatever the order.
// E2M3 and not E4M3 for the finer queries: at a block's own scale both keep four digits of its larger elements, the matrix
// instruction takes six-bit operands at the four-bit rate, and it adds their products without loss (measured over random blocks:
// within 2^-23.4 of sum|q x|, where E4M3 products came back up to 3e-4 of the largest product off).
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
typedef unsigned int mx4_u2 __attribute__((ext_vector_type(2)));

enum { MX4_F32 = 0, MX4_BF16 = 2, MX4_F16 = 3 };   // VSGPU_F32, _BF16, _F16
enum { MX4_L2 = 0, MX4_IP = 1, MX4_COSINE = 2 };

__host__ __device__ inline uint32_t mx4_steps(uint32_t dim) { return (dim + 63) / 64; }
__host__ __device__ inline uint32_t mx4_groups(uint32_t dim) { return (mx4_steps(dim) + 3) / 4; }
__host__ __device__ inline uint32_t mx4_panel(uint32_t dim) { return mx4_steps(dim) * 1024 + mx4_groups(dim) * 256 + 128; }
// a 32-query tile of the query block: operand bytes of every k-step (16 a lane; E2M3: 8 more a lane behind all of them), scales
__host__ __device__ inline uint32_t mx4_qtile(uint32_t dim, int bits) { return mx4_steps(dim) * (bits == 6 ? 1536 : 1024) + mx4_groups(dim) * 256; }

// where rows are: one block of panels, or slabs of 2^shift panels each
struct Mx4Rows {
    char *base;
    char *const *slabs;
    uint32_t shift;
    uint32_t dim, ks, kg, panel;
    uint64_t n;
    __device__ char *at(uint64_t p) const {
        if (slabs) return slabs[p >> shift] + (p & ((1u << shift) - 1)) * (size_t)panel;
        return base + p * panel;
    }
};

__device__ __forceinline__ double mx4_pow2(int e) {   // 2^e, |e| <= 1000
    return __longlong_as_double((long long)(e + 1023) << 52);
}

template <int T> __device__ __forceinline__ float mx4_widen(const void *p, size_t i) {
    if constexpr (T == MX4_F32) return static_cast<const float *>(p)[i];
    else if constexpr (T == MX4_F16) return (float)static_cast<const _Float16 *>(p)[i];
    else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
}
// 32 elements from x on, `have` of them in the row.  WIDE: x is 16-byte aligned
template <int T, bool WIDE> __device__ __forceinline__ void mx4_load32(const void *x, int have, float v[32]) {
    if (WIDE && have >= 32) {
        if constexpr (T == MX4_F32) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const mx4_f4 w = static_cast<const mx4_f4 *>(x)[i];
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const mx4_u4 w = static_cast<const mx4_u4 *>(x)[i];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint16_t h = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
                    v[8 * i + j] = T == MX4_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = j < have ? mx4_widen<T>(x, (size_t)j) : 0.f;
}

// the block's scale byte, and 2^-E for its elements (0 where the block is NaN or zero)
__device__ __forceinline__ int mx4_scale(const float v[32], float &inv) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 32; j++) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);   // (a NaN's bits are above infinity's)
    if (top >= 0x7F800000u) {
        inv = 0.f;
        return 255;
    }
    // exponent field - 2; subnormal and smallest values clamp to byte 0 (E = -127)
    const int byte = max((int)(top >> 23) - 2, 0);
    inv = __uint_as_float((uint32_t)(254 - byte) << 23);   // 2^(127 - byte): the exponent field 254 - byte is 2..254
    return byte;
}
// four dwords of E2M1 codes; returns sum (2 x)^2.  The conversion rounds to nearest even and saturates, as the format asks
// (checked against the definition at every tie and border)
__device__ __forceinline__ int mx4_codes4(const float v[32], float inv, bool bad, mx4_u4 &out) {
    int ss = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        uint32_t d = 0;
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w] * inv, v[8 * w + 1] * inv, 1.f, 0);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w + 2] * inv, v[8 * w + 3] * inv, 1.f, 1);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w + 4] * inv, v[8 * w + 5] * inv, 1.f, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w + 6] * inv, v[8 * w + 7] * inv, 1.f, 3);
        out[w] = bad ? 0u : d;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t c = (out[w] >> (4 * j)) & 7u;
            const int twice = c < 2 ? (int)c : (int)((2u | (c & 1u)) << ((c >> 1) - 1));   // 0 1 2 3 4 6 8 12
            ss += twice * twice;
        }
    }
    return ss;
}
// six dwords of E2M3 codes; returns sum (8 x)^2
__device__ __forceinline__ int mx4_codes6(const float v[32], float inv, bool bad, uint32_t out[6]) {
    uint32_t w[6] = {0, 0, 0, 0, 0, 0};
    int ss = 0;
#pragma unroll
    for (int j = 0; j < 32; j++) {
        const float m = fminf(fabsf(v[j] * inv), 7.5f);
        // steps of 1/8 below 2, 1/4 below 4, 1/2 above: rounding to the step, ties to even
        const float up = m < 2.f ? 8.f : (m < 4.f ? 4.f : 2.f);
        const int eighths = bad ? 0 : (int)(__builtin_rintf(m * up) * (8.f / up));
        ss += eighths * eighths;
        // eighths -> code: below 16 the number itself, then exponent and three digits
        const uint32_t mag = eighths < 16 ? (uint32_t)eighths : (eighths < 32 ? 16u + (((uint32_t)eighths - 16u) >> 1) : 24u + (((uint32_t)eighths - 32u) >> 2));
        const uint32_t c = mag | (__float_as_uint(v[j]) >> 31 << 5);
        const int bit = 6 * j;
        w[bit / 32] |= c << (bit % 32);
        if (bit % 32 > 26) w[bit / 32 + 1] |= c >> (32 - bit % 32);
    }
#pragma unroll
    for (int i = 0; i < 6; i++) out[i] = bad ? 0u : w[i];
    return ss;
}

// ---------------------------------------------------------------------------------------------------------------- write
struct Mx4Write {
    Mx4Rows rows;
    const char *x;
    size_t stride;              // bytes between two vectors
    uint64_t m;
    const void *slots;          // int32 / int64; null: rows first .. first + m - 1
    int slots64;
    uint64_t first;
    uint64_t capacity;          // slots in the table
    int claimed;                // k_mx4_claim has run: a slot's norm says which vector owns it
};
__device__ __forceinline__ int64_t mx4_slot(const void *slots, int is64, uint64_t i, uint64_t first) {
    if (!slots) return (int64_t)(first + i);
    return is64 ? static_cast<const int64_t *>(slots)[i] : (int64_t)static_cast<const int32_t *>(slots)[i];
}
// Which vector a slot gets when several name it: the last.  Two passes over the norms: cleared, then the largest 2^31 | i.
static __global__ __launch_bounds__(256) void k_mx4_claim(Mx4Write W, int pass) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= W.m) return;
    const int64_t s = mx4_slot(W.slots, W.slots64, i, W.first);
    if (s < 0 || (uint64_t)s >= W.capacity) return;
    uint32_t *norm = reinterpret_cast<uint32_t *>(W.rows.at((uint64_t)s / 32) + W.rows.panel - 128) + (s & 31);
    if (pass == 0) __hip_atomic_store(norm, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else atomicMax(norm, 0x80000000u | (uint32_t)i);
}
// One workgroup takes 32 vectors, its waves every fourth k-step; a lane rounds one block (half, row) by itself, so neither the
// maximum nor the codes cross lanes.
template <int T, bool WIDE> static __global__ __launch_bounds__(256) void k_mx4_write(Mx4Write W) {
    __shared__ double part[4][64];
    __shared__ int64_t slot_s[32];
    __shared__ int lost_s[32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 31, half = lane >> 5;
    const uint64_t i0 = (uint64_t)blockIdx.x * 32;
    if (threadIdx.x < 32) {
        const uint64_t i = i0 + threadIdx.x;
        int64_t s = -1;
        if (i < W.m) s = mx4_slot(W.slots, W.slots64, i, W.first);
        if (s >= 0 && (uint64_t)s >= W.capacity) s = -1;
        if (s >= 0 && W.claimed) {
            const uint32_t *norm = reinterpret_cast<const uint32_t *>(W.rows.at((uint64_t)s / 32) + W.rows.panel - 128) + (s & 31);
            if (__hip_atomic_load(norm, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (0x80000000u | (uint32_t)i)) s = -1;
        }
        slot_s[threadIdx.x] = s;
        lost_s[threadIdx.x] = 0;
    }
    __syncthreads();
    if (W.slots && !W.claimed) {   // few vectors: a later vector with the same slot takes it
        for (uint64_t j = i0 + threadIdx.x; j < W.m; j += 256) {
            const int64_t s = mx4_slot(W.slots, W.slots64, j, W.first);
            if (s < 0) continue;
            for (int r = 0; r < 32 && i0 + r < j; r++)
                if (slot_s[r] == s) lost_s[r] = 1;
        }
        __syncthreads();
    }
    const int64_t slot = lost_s[row] ? -1 : slot_s[row];
    double ss = 0;
    if (slot >= 0) {
        const char *x = W.x + (i0 + row) * W.stride;
        char *panel = W.rows.at((uint64_t)slot / 32);
        const int at = (int)(slot & 31) + 32 * half;
        const int esz = T == MX4_F32 ? 4 : 2;
        for (uint32_t s = wave; s < W.rows.ks; s += 4) {
            const int have = (int)W.rows.dim - (int)(2 * s + half) * 32;
            float v[32], inv;
            if (have > 0) mx4_load32<T, WIDE>(x + (size_t)(2 * s + half) * 32 * esz, have, v);
            else {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = 0.f;
            }
            const int byte = mx4_scale(v, inv);
            mx4_u4 codes;
            const int sq = mx4_codes4(v, inv, byte == 255, codes);
            ss += byte == 255 ? __builtin_nan("") : (double)sq * mx4_pow2(2 * (byte - 128));   // (2x)^2 / 4
            *reinterpret_cast<mx4_u4 *>(panel + (size_t)s * 1024 + at * 16) = codes;
            panel[(size_t)W.rows.ks * 1024 + (s >> 2) * 256 + at * 4 + (s & 3)] = (char)byte;
        }
    }
    part[wave][lane] = ss;
    __syncthreads();
    if (threadIdx.x < 32 && slot >= 0) {
        double t = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) t += part[w][lane] + part[w][lane + 32];
        float nrm = (float)sqrt(t);
        if (!(nrm == nrm)) nrm = __uint_as_float(0x7FC00000u);
        *(reinterpret_cast<float *>(W.rows.at((uint64_t)slot / 32) + W.rows.panel - 128) + (slot & 31)) = nrm;
    }
}

// ---------------------------------------------------------------------------------------------------------------- read
struct Mx4Read {
    Mx4Rows rows;
    char *out;
    size_t stride;
    uint64_t m;
    const void *slots;
    int slots64;
    uint64_t first, capacity;
};
template <int T> __device__ __forceinline__ void mx4_store1(char *o, size_t i, float v) {
    if constexpr (T == MX4_F32) reinterpret_cast<float *>(o)[i] = v;
    else if constexpr (T == MX4_F16) reinterpret_cast<_Float16 *>(o)[i] = (_Float16)v;
    else {   // E2M1 values have two digits: bf16 holds them exactly, its subnormals the smallest blocks'
        reinterpret_cast<uint16_t *>(o)[i] = (uint16_t)(__float_as_uint(v) >> 16);
    }
}
// 2^(byte - 127) in fp32 (byte 0: subnormal; 255: NaN)
__device__ __forceinline__ float mx4_scale_value(uint32_t byte) {
    return byte == 255 ? __uint_as_float(0x7FC00000u) : (byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
}
__device__ __forceinline__ float mx4_code_value(uint32_t c) {   // c: 4 bits
    const uint32_t m = c & 7u;
    const float v = m < 2 ? 0.5f * (float)m : (float)((2u | (m & 1u)) << ((m >> 1) - 1)) * 0.5f;
    return c & 8u ? -v : v;
}
// A thread turns 8 codes (one dword) into 8 values; consecutive threads run along a row, so the stores of a wave are contiguous.
template <int T> static __global__ __launch_bounds__(256) void k_mx4_read(Mx4Read R) {
    const uint32_t per_row = (R.rows.dim + 7) / 8;
    const uint64_t total = R.m * per_row;
    for (uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (uint64_t)gridDim.x * 256) {
        const uint64_t i = t / per_row;
        const uint32_t piece = (uint32_t)(t - i * per_row), e = piece * 8;
        const int64_t s = mx4_slot(R.slots, R.slots64, i, R.first);
        float v[8];
        if (s < 0 || (uint64_t)s >= R.capacity) {
            const float f = s < 0 ? 0.f : __uint_as_float(0x7FC00000u);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = f;
        } else {
            const char *panel = R.rows.at((uint64_t)s / 32);
            const uint32_t step = e / 64, half = (e / 32) & 1, at = (uint32_t)(s & 31) + 32 * half;
            const uint32_t codes = *reinterpret_cast<const uint32_t *>(panel + (size_t)step * 1024 + at * 16 + (e & 31) / 2);
            const float sc = mx4_scale_value((uint8_t)panel[(size_t)R.rows.ks * 1024 + (step >> 2) * 256 + at * 4 + (step & 3)]);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = mx4_code_value((codes >> (4 * j)) & 15u) * sc;
        }
        char *o = R.out + i * R.stride;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (e + j < R.rows.dim) mx4_store1<T>(o, e + j, v[j]);
    }
}

// row src into row dst of one table (swap-delete)
static __global__ __launch_bounds__(256) void k_mx4_move(Mx4Rows R, uint64_t dst, uint64_t src) {
    char *d = R.at(dst / 32);
    const char *s = R.at(src / 32);
    const uint32_t dr = (uint32_t)(dst & 31), sr = (uint32_t)(src & 31);
    for (uint32_t i = threadIdx.x; i < R.ks * 2; i += 256)
        reinterpret_cast<mx4_u4 *>(d)[i * 32 + dr] = reinterpret_cast<const mx4_u4 *>(s)[i * 32 + sr];
    for (uint32_t i = threadIdx.x; i < R.kg * 2; i += 256)
        reinterpret_cast<uint32_t *>(d + (size_t)R.ks * 1024)[i * 32 + dr] = reinterpret_cast<const uint32_t *>(s + (size_t)R.ks * 1024)[i * 32 + sr];
    if (threadIdx.x == 0) reinterpret_cast<float *>(d + R.panel - 128)[dr] = reinterpret_cast<const float *>(s + R.panel - 128)[sr];
}

// ---------------------------------------------------------------------------------------------------------------- queries
// the query block: q_tiles operand tiles, then per query {norm fp32}, {|q|^2 fp64}
struct Mx4Queries {
    const char *x;
    size_t stride;
    uint32_t nq, dim, ks, kg;
    char *tiles;
    float *norm;         // [tiles * 32]
    double *sq;          // [tiles * 32]
    uint32_t *zero;      // words to clear for the kernels behind this one
    uint32_t zero_words;
};
template <int T, bool WIDE, int BITS> static __global__ __launch_bounds__(256) void k_mx4_queries(Mx4Queries Q) {
    __shared__ double part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 31, half = lane >> 5;
    const uint32_t q = blockIdx.x * 32 + row;
    char *tile = Q.tiles + (size_t)blockIdx.x * mx4_qtile(Q.dim, BITS);
    char *scales = tile + (size_t)Q.ks * (BITS == 6 ? 1536 : 1024);
    const int esz = T == MX4_F32 ? 4 : 2;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < Q.zero_words; i += gridDim.x * 256) Q.zero[i] = 0;
    double ss = 0;
    for (uint32_t s = wave; s < Q.kg * 4; s += 4) {
        char *sc = scales + (s >> 2) * 256 + lane * 4 + (s & 3);
        if (s >= Q.ks) {
            *sc = 0;
            continue;
        }
        const int have = q < Q.nq ? (int)Q.dim - (int)(2 * s + half) * 32 : 0;
        float v[32], inv;
        if (have > 0) mx4_load32<T, WIDE>(Q.x + q * Q.stride + (size_t)(2 * s + half) * 32 * esz, have, v);
        else {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = 0.f;
        }
        const int byte = mx4_scale(v, inv);
        int sq;
        if constexpr (BITS == 6) {
            uint32_t w[6];
            sq = mx4_codes6(v, inv, byte == 255, w);
            *reinterpret_cast<mx4_u4 *>(tile + (size_t)s * 1024 + lane * 16) = mx4_u4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<mx4_u2 *>(tile + (size_t)Q.ks * 1024 + (size_t)s * 512 + lane * 8) = mx4_u2{w[4], w[5]};
        } else {
            mx4_u4 w;
            sq = mx4_codes4(v, inv, byte == 255, w);
            *reinterpret_cast<mx4_u4 *>(tile + (size_t)s * 1024 + lane * 16) = w;
        }
        *sc = (char)byte;
        ss += byte == 255 ? __builtin_nan("") : (double)sq * mx4_pow2(2 * (byte - (BITS == 6 ? 130 : 128)));
    }
    part[wave][lane] = ss;
    __syncthreads();
    if (threadIdx.x < 32) {
        double t = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) t += part[w][lane] + part[w][lane + 32];
        Q.sq[q] = t;
        Q.norm[q] = (float)sqrt(t);
    }
}

// ---------------------------------------------------------------------------------------------------------------- scan
// How far a matrix-core dot may be from the exact one, over |q| |x|: each of the ks instructions adds its 64 products to the sum
// so far within 2^-22 of what it adds up (measured 2^-23.4); eight more of the same for the rounded norms and the comparison's own
// arithmetic, and twice all of it.
__host__ __device__ inline float mx4_slack(uint32_t ks) { return (float)(ks + 8) * 4.76837158203125e-7f; }
constexpr float MX4_EPS = 1.9073486328125e-6f;   // 2^-19, of |q|^2 + |x|^2 (L2): the same for sums of squares

enum { MX4_PROBE = 0, MX4_PROBE_ROWS = 1, MX4_FILTER = 2, MX4_DENSE = 3 };
struct Mx4Scan {
    Mx4Rows rows;
    const char *tiles;           // this launch's query tiles start at blockIdx.y * QT
    uint32_t qtile_bytes;
    uint32_t nq, metric;
    const float *qnorm;
    // which panels: n_take of them, number i is i * n_panels / n_take
    uint64_t n_panels, n_take;
    float *minima;               // PROBE: [nq][2 n_take] upper bounds of 16 rows each; PROBE_ROWS: [nq][n] of each row
    uint64_t minima_stride;
    const float2 *limit;         // FILTER: {alpha, beta} of each query
    uint32_t *counts;            // FILTER
    uint2 *cand;
    uint32_t cap;
    float *out;                  // DENSE: [nq][out_stride]
    uint64_t out_stride;
    float slack;
};

// one operand pair and its scales; the table is the A operand (results: a lane one query, its registers 16 rows) or, for dense
// scores, the B operand (a lane one row: stores along a query's line)
template <int BITS, bool SWAP, int I> __device__ __forceinline__ mx4_f16 mx4_mma(mx4_i8 t, mx4_i8 q, mx4_f16 c, int st, int sq) {
    constexpr int FQ = BITS == 6 ? 2 : 4;
    if constexpr (SWAP) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(q, t, c, FQ, 4, I, sq, I, st);
    else return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(t, q, c, 4, FQ, I, st, I, sq);
}
struct Mx4Chunk {   // four k-steps of a panel
    mx4_i4 a[4];
    int sc;
};
__device__ __forceinline__ void mx4_fetch(Mx4Chunk &c, const char *panel, uint32_t g, uint32_t ks, int lane) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t s = min(4 * g + i, ks - 1);   // (past the last step: the same bytes again, never used)
        c.a[i] = __builtin_nontemporal_load(reinterpret_cast<const mx4_i4 *>(panel + (size_t)s * 1024) + lane);
    }
    c.sc = __builtin_nontemporal_load(reinterpret_cast<const int *>(panel + (size_t)ks * 1024 + g * 256) + lane);
}
template <int BITS, bool SWAP, int QT, int I>
__device__ __forceinline__ void mx4_step(mx4_f16 *acc, const Mx4Chunk &c, const char *lds, uint32_t g, uint32_t ks, uint32_t qtile_bytes, const int *sq, int lane) {
    const uint32_t s = 4 * g + I;
    mx4_i8 t{c.a[I][0], c.a[I][1], c.a[I][2], c.a[I][3], 0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < QT; q++) {
        const char *b = lds + q * qtile_bytes;
        const mx4_i4 lo = reinterpret_cast<const mx4_i4 *>(b + s * 1024)[lane];
        mx4_i8 f{lo[0], lo[1], lo[2], lo[3], 0, 0, 0, 0};
        if constexpr (BITS == 6) {
            const mx4_u2 hi = reinterpret_cast<const mx4_u2 *>(b + ks * 1024 + s * 512)[lane];
            f[4] = (int)hi[0];
            f[5] = (int)hi[1];
        }
        acc[q] = mx4_mma<BITS, SWAP, I>(t, f, acc[q], c.sc, sq[q]);
    }
}

// A wave takes whole panels, one after the other, every wave of the grid in turn; the queries' operands stay in LDS.  NB chunks of
// the panel (256 elements each) are in flight: chunk g of the next panel is requested as soon as chunk g of this one has gone into
// the matrix cores.  Panels of more than 4 chunks go through the same four buffers several times.
template <int BITS, int QT, int MODE, int NB, bool GB> static __global__ __launch_bounds__(256) void k_mx4_scan(Mx4Scan P) {
    extern __shared__ char shared[];
    constexpr bool SWAP = MODE == MX4_DENSE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const uint32_t q0 = blockIdx.y * QT * 32;
    const uint32_t ks = P.rows.ks, kg = P.rows.kg;
    // (rows too wide for that, GB: the operands are read from the query block itself, through the caches)
    const char *lds = GB ? P.tiles + (size_t)blockIdx.y * QT * P.qtile_bytes : shared;
    float *yn_s = reinterpret_cast<float *>(shared + (GB ? 0 : QT * P.qtile_bytes));
    if constexpr (!GB) {
        const mx4_u4 *src = reinterpret_cast<const mx4_u4 *>(P.tiles + (size_t)blockIdx.y * QT * P.qtile_bytes);
        const uint32_t n16 = QT * P.qtile_bytes / 16;
        for (uint32_t i = threadIdx.x; i < n16; i += 256) reinterpret_cast<mx4_u4 *>(shared)[i] = src[i];
    }
    for (uint32_t i = threadIdx.x; i < QT * 32; i += 256) yn_s[i] = P.qnorm[q0 + i];   // (padded to whole tiles)
    __syncthreads();
    const uint32_t sc_at = ks * (BITS == 6 ? 1536 : 1024);
    float alpha[QT], beta[QT], qn[QT];
#pragma unroll
    for (int q = 0; q < QT; q++) {
        const uint32_t me = q0 + q * 32 + col;
        if constexpr (MODE == MX4_FILTER) {
            const float2 l = me < P.nq ? P.limit[me] : make_float2(0.f, __uint_as_float(0x7F800000u));
            alpha[q] = l.x;
            beta[q] = l.y;
        }
        qn[q] = yn_s[q * 32 + col];
    }
    const uint64_t W = (uint64_t)gridDim.x * 4;
    uint64_t w = (uint64_t)blockIdx.x * 4 + wave;
    if (w >= P.n_take) return;
    const auto panel_of = [&](uint64_t i) { return P.n_take == P.n_panels ? i : i * P.n_panels / P.n_take; };
    Mx4Chunk buf[NB];
    const char *panel = P.rows.at(panel_of(w));
#pragma unroll
    for (int g = 0; g < NB; g++)
        if (g < (int)kg) mx4_fetch(buf[g], panel, g, ks, lane);
    for (; w < P.n_take; w += W) {
        const uint64_t p = panel_of(w), wn = w + W;
        const char *next = wn < P.n_take ? P.rows.at(panel_of(wn)) : panel;   // (at the end: this panel again, never used)
        mx4_f16 acc[QT];
#pragma unroll
        for (int q = 0; q < QT; q++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[q][v] = 0.f;
        mx4_f4 nrm[4];
        float nx = 0.f;
        if constexpr (SWAP) nx = reinterpret_cast<const float *>(panel + P.rows.panel - 128)[col];
        else {
#pragma unroll
            for (int i = 0; i < 4; i++) nrm[i] = reinterpret_cast<const mx4_f4 *>(panel + P.rows.panel - 128)[2 * i + half];
        }
        for (uint32_t g0 = 0; g0 < kg; g0 += NB) {
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const uint32_t g = g0 + j;
                if (g >= kg) break;
                int sq[QT];
#pragma unroll
                for (int q = 0; q < QT; q++) sq[q] = reinterpret_cast<const int *>(lds + q * P.qtile_bytes + sc_at + g * 256)[lane];
                mx4_step<BITS, SWAP, QT, 0>(acc, buf[j], lds, g, ks, P.qtile_bytes, sq, lane);
                if (4 * g + 1 < ks) mx4_step<BITS, SWAP, QT, 1>(acc, buf[j], lds, g, ks, P.qtile_bytes, sq, lane);
                if (4 * g + 2 < ks) mx4_step<BITS, SWAP, QT, 2>(acc, buf[j], lds, g, ks, P.qtile_bytes, sq, lane);
                if (4 * g + 3 < ks) mx4_step<BITS, SWAP, QT, 3>(acc, buf[j], lds, g, ks, P.qtile_bytes, sq, lane);
                // the buffer's next contents: NB chunks on in this panel, or the chunk of the next panel that it takes
                if (g + NB < kg) mx4_fetch(buf[j], panel, g + NB, ks, lane);
                else mx4_fetch(buf[j], next, j, ks, lane);
            }
        }
        const uint64_t row0 = p * 32;
        if constexpr (MODE == MX4_DENSE) {
            const uint64_t row = row0 + col;
#pragma unroll
            for (int q = 0; q < QT; q++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const uint32_t me = q0 + q * 32 + 8 * (v >> 2) + 4 * half + (v & 3);
                    const float yn = yn_s[q * 32 + 8 * (v >> 2) + 4 * half + (v & 3)];
                    float s;
                    if (P.metric == MX4_L2) s = __fmaf_rn(-2.f, acc[q][v], __fmaf_rn(nx, nx, yn * yn));
                    else if (P.metric == MX4_IP) s = 1.f - acc[q][v];
                    else s = 1.f - acc[q][v] / nx / yn;
                    if (me < P.nq && row < P.rows.n) P.out[me * P.out_stride + row] = s;
                }
        } else if constexpr (MODE == MX4_FILTER) {
            // emitted when the score may be at or below the query's threshold: dot >= alpha |x| + beta + (L2: |x|^2 / 2)
            float base[16];
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const float x = nrm[v >> 2][v & 3];
                base[v] = P.metric == MX4_L2 ? 0.5f * (1.f - MX4_EPS) * x * x : 0.f;
                if (P.metric == MX4_COSINE && !(x > 0.f)) base[v] = __uint_as_float(0x7F800000u);   // no direction: score NaN
            }
#pragma unroll
            for (int q = 0; q < QT; q++) {
                bool any = false;
#pragma unroll
                for (int v = 0; v < 16; v++) any |= acc[q][v] >= __fmaf_rn(alpha[q], nrm[v >> 2][v & 3], base[v] + beta[q]);
                if (any) {
                    const uint32_t me = q0 + q * 32 + col;
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const uint64_t row = row0 + 8 * (v >> 2) + 4 * half + (v & 3);
                        if (acc[q][v] >= __fmaf_rn(alpha[q], nrm[v >> 2][v & 3], base[v] + beta[q]) && row < P.rows.n) {
                            const uint32_t at = atomicAdd(&P.counts[me], 1u);
                            if (at < P.cap) P.cand[(size_t)me * P.cap + at].x = (uint32_t)row;
                        }
                    }
                }
            }
        } else {
            const float inf = __uint_as_float(0x7F800000u);
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const uint32_t me = q0 + q * 32 + col;
                float best = inf;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const float x = nrm[v >> 2][v & 3], d = acc[q][v];
                    const uint64_t row = row0 + 8 * (v >> 2) + 4 * half + (v & 3);
                    float u;   // an upper bound of the score
                    if (P.metric == MX4_L2) u = __fmaf_rn(2.f * P.slack * qn[q], x, __fmaf_rn(-2.f, d, (1.f + MX4_EPS) * (x * x + qn[q] * qn[q])));
                    else if (P.metric == MX4_IP) u = __fmaf_rn(P.slack * qn[q], x, 1.f - d);
                    else u = 1.f - d / x / qn[q] + P.slack;
                    if (row >= P.rows.n || !(u == u)) u = inf;
                    if constexpr (MODE == MX4_PROBE_ROWS) {
                        if (me < P.nq && row < P.rows.n) P.minima[me * P.minima_stride + row] = u;
                    }
                    best = fminf(best, u);
                }
                if constexpr (MODE == MX4_PROBE) {
                    if (me < P.nq) P.minima[me * P.minima_stride + 2 * w + half] = best;
                }
            }
        }
        panel = next;
    }
}

// ---------------------------------------------------------------------------------------------------------------- threshold
__device__ __forceinline__ uint32_t mx4_key(float f) {   // order-preserving; NaN is never passed
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float mx4_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
struct Mx4Threshold {
    const float *minima;
    uint64_t stride, count;
    uint32_t k, metric;
    const float *qnorm;
    const double *qsq;
    float2 *limit;
    float slack;
};
// tau = the k-th smallest upper bound (each of different rows, so at least k rows are at or below it), then what the filter compares
// against.  The score of a row is rounded to fp32 before rows are compared: half a step of it more.
static __global__ __launch_bounds__(1024) void k_mx4_threshold(Mx4Threshold T) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t pick_s, left_s;
    const uint32_t q = blockIdx.x;
    const float *m = T.minima + q * T.stride;
    uint32_t prefix = 0, mask = 0, need = T.k;
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
    const bool all = T.k > T.count;
    for (int pass = 0; pass < 3 && !all; pass++) {
        const uint32_t bins = 1u << bits[pass];
        for (uint32_t i = threadIdx.x; i < bins; i += 1024) hist[i] = 0;
        __syncthreads();
        for (uint64_t i = threadIdx.x; i < T.count; i += 1024) {
            const uint32_t key = mx4_key(m[i]);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shifts[pass]) & (bins - 1)], 1u);
        }
        __syncthreads();
        if (threadIdx.x < 64) {   // one wave finds the bin of the need-th: bins / 64 each, then the lane's own
            const uint32_t each = bins / 64, b0 = threadIdx.x * each;
            uint32_t sum = 0;
            for (uint32_t i = 0; i < each; i++) sum += hist[b0 + i];
            uint32_t before = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t t = __shfl_up(before, o);
                if ((int)threadIdx.x >= o) before += t;
            }
            before -= sum;
            if (before < need && need <= before + sum) {
                uint32_t i = 0;
                while (before + hist[b0 + i] < need) before += hist[b0 + i++];
                pick_s = b0 + i;
                left_s = need - before;
            }
        }
        __syncthreads();
        prefix |= pick_s << shifts[pass];
        mask |= (bins - 1) << shifts[pass];
        need = left_s;
        __syncthreads();
    }
    if (threadIdx.x) return;
    const float inf = __uint_as_float(0x7F800000u);
    const float tau = all ? inf : mx4_unkey(prefix), yn = T.qnorm[q];
    float2 l;
    if (T.metric == MX4_L2) {
        l.x = -T.slack * yn;
        l.y = 0.5f * ((1.f - MX4_EPS) * yn * yn - (tau + MX4_EPS * fabsf(tau)));
    } else if (T.metric == MX4_IP) {
        l.x = -T.slack * yn;
        l.y = 1.f - tau - 9.5367431640625e-7f * fmaxf(1.f, fabsf(tau));   // 2^-20
    } else {
        l.x = ((1.f - tau) - T.slack - 9.5367431640625e-7f) * yn;
        l.y = 0.f;
    }
    if (tau == inf) l = make_float2(0.f, -inf);
    const double sq = T.qsq[q];
    if (!(sq == sq) || (T.metric == MX4_COSINE && sq == 0)) l = make_float2(0.f, inf);   // every score is NaN
    T.limit[q] = l;
}

// ---------------------------------------------------------------------------------------------------------------- exact scores
struct Mx4Exact {
    Mx4Rows rows;
    const char *tiles;
    uint32_t qtile_bytes, metric;
    const double *qsq;
};
__device__ __forceinline__ float mx4_code6(const uint32_t *w, int j) {   // element j of six dwords
    const int bit = 6 * j;
    uint32_t c = w[bit / 32] >> (bit % 32);
    if (bit % 32 > 26) c |= w[bit / 32 + 1] << (32 - bit % 32);
    const uint32_t m = c & 31u;
    const float v = m < 16 ? (float)m : (m < 24 ? (float)(2 * m - 16) : (float)(4 * m - 64));
    return (c & 32u ? -v : v) * 0.125f;
}
// this lane's share of a row's sums: blocks first, first + by, ...   In a block the sums are whole numbers (of 1/16): exact.
template <int BITS> __device__ __forceinline__ void mx4_row_sums(const Mx4Exact &E, const char *tile, uint32_t col, const char *panel, uint32_t r,
                                                                 uint32_t first, uint32_t by, double &dot, double &xx) {
    const uint32_t nb = E.rows.ks * 2;
    dot = 0;
    xx = 0;
    for (uint32_t b = first; b < nb; b += by) {
        const uint32_t s = b >> 1, half = b & 1, ra = r + 32 * half, qa = col + 32 * half;
        const mx4_u4 x = *reinterpret_cast<const mx4_u4 *>(panel + (size_t)s * 1024 + ra * 16);
        const uint32_t bx = (uint8_t)panel[(size_t)E.rows.ks * 1024 + (s >> 2) * 256 + ra * 4 + (s & 3)];
        const mx4_u4 lo = *reinterpret_cast<const mx4_u4 *>(tile + (size_t)s * 1024 + qa * 16);
        const uint32_t bq = (uint8_t)tile[(size_t)E.rows.ks * (BITS == 6 ? 1536 : 1024) + (s >> 2) * 256 + qa * 4 + (s & 3)];
        uint32_t w[6] = {lo[0], lo[1], lo[2], lo[3], 0, 0};
        if constexpr (BITS == 6) {
            const mx4_u2 hi = *reinterpret_cast<const mx4_u2 *>(tile + (size_t)E.rows.ks * 1024 + (size_t)s * 512 + qa * 8);
            w[4] = hi[0];
            w[5] = hi[1];
        }
        float d = 0, sq = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) {
            const float xv = mx4_code_value((x[j / 8] >> (4 * (j % 8))) & 15u);
            const float qv = BITS == 6 ? mx4_code6(w, j) : mx4_code_value((w[j / 8] >> (4 * (j % 8))) & 15u);
            d = __fmaf_rn(xv, qv, d);
            sq = __fmaf_rn(xv, xv, sq);
        }
        const double nan = __builtin_nan("");
        dot += bx == 255 || bq == 255 ? nan : (double)d * mx4_pow2((int)bx + (int)bq - 254);
        xx += bx == 255 ? nan : (double)sq * mx4_pow2(2 * (int)bx - 254);
    }
}
__device__ __forceinline__ float mx4_final(uint32_t metric, double dot, double xx, double qq) {
    if (metric == MX4_IP) return (float)(1.0 - dot);
    if (metric == MX4_L2) return (float)(qq + xx - 2.0 * dot);
    return (float)(1.0 - dot / (sqrt(qq) * sqrt(xx)));
}
constexpr int MX4_LANES = 16;   // lanes on one row in the exact kernels
template <int BITS> __device__ __forceinline__ float mx4_exact_score(const Mx4Exact &E, uint32_t q, uint64_t row) {
    double dot, xx;
    mx4_row_sums<BITS>(E, E.tiles + (size_t)(q >> 5) * E.qtile_bytes, q & 31, E.rows.at(row >> 5), (uint32_t)(row & 31), threadIdx.x % MX4_LANES, MX4_LANES, dot, xx);
#pragma unroll
    for (int o = MX4_LANES / 2; o; o >>= 1) {
        dot += __shfl_xor(dot, o);
        xx += __shfl_xor(xx, o);
    }
    return mx4_final(E.metric, dot, xx, E.qsq[q]);
}
// the filter's candidates, scored exactly in place
template <int BITS> static __global__ __launch_bounds__(256) void k_mx4_rerank(Mx4Exact E, const uint32_t *counts, uint2 *cand, uint32_t cap) {
    const uint32_t q = blockIdx.y, n = min(counts[q], cap);
    for (uint32_t i = (blockIdx.x * 256 + threadIdx.x) / MX4_LANES; i < n; i += gridDim.x * (256 / MX4_LANES)) {
        uint2 *c = cand + (size_t)q * cap + i;
        const float s = mx4_exact_score<BITS>(E, q, c->x);
        if (threadIdx.x % MX4_LANES == 0) c->y = __float_as_uint(s);
    }
}
// rows first .. first + m - 1, or ids[0 .. m)
template <int BITS> static __global__ __launch_bounds__(256) void k_mx4_exact_rows(Mx4Exact E, uint32_t nq, const uint32_t *ids, uint64_t first, uint64_t m, float *out) {
    const uint32_t q = blockIdx.y;
    for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / MX4_LANES; i < m; i += (uint64_t)gridDim.x * (256 / MX4_LANES)) {
        const float s = mx4_exact_score<BITS>(E, q, ids ? ids[i] : first + i);
        if (threadIdx.x % MX4_LANES == 0) out[q * m + i] = s;
    }
}

// ---------------------------------------------------------------------------------------------------------------- the k best
// order: (score, row), both ascending, as one 64-bit key; 0xFF.. = nothing (NaN scores become that)
constexpr uint64_t MX4_NONE = ~0ull;
__device__ __forceinline__ uint64_t mx4_pack(float s, uint32_t row) {
    if (!(s == s)) return MX4_NONE;
    return (uint64_t)mx4_key(s == 0.f ? 0.f : s) << 32 | row;   // (-0 and 0 are equal)
}
// ascending bitonic sort of n (a power of two) keys in LDS by the whole workgroup
__device__ __forceinline__ void mx4_sort(uint64_t *k, uint32_t n) {
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t stride = size >> 1; stride; stride >>= 1) {
            __syncthreads();
            for (uint32_t t = threadIdx.x; t < n / 2; t += blockDim.x) {
                const uint32_t lo = (t / stride) * stride * 2 + t % stride, hi = lo + stride;
                const bool up = (lo & size) == 0;
                const uint64_t a = k[lo], b = k[hi];
                if ((a > b) == up) {
                    k[lo] = b;
                    k[hi] = a;
                }
            }
        }
    __syncthreads();
}
constexpr uint32_t MX4_KEEP = 8192;      // keys in LDS (64 KiB)
constexpr uint32_t MX4_KMAX = 4096;      // largest k
// A running selection in LDS: keys below the k-th best so far are added; when the room is short, sorted and cut to k.
struct Mx4Keep {
    uint64_t *keys;      // [MX4_KEEP], shared
    uint32_t *n;         // shared
    uint64_t *limit;     // shared: nothing at or above it is wanted
    uint32_t k;
};
__device__ __forceinline__ void mx4_keep_cut(const Mx4Keep &K) {   // all threads; leaves the k best sorted
    __syncthreads();
    const uint32_t n = *K.n;
    uint32_t pow2 = 2;
    while (pow2 < n) pow2 <<= 1;
    for (uint32_t i = n + threadIdx.x; i < pow2; i += blockDim.x) K.keys[i] = MX4_NONE;
    mx4_sort(K.keys, pow2);
    if (threadIdx.x == 0) {
        *K.n = min(n, K.k);
        if (n >= K.k) *K.limit = min(*K.limit, K.keys[K.k - 1]);
    }
    __syncthreads();
}
// called by all threads, at most `room` of them with a key (MX4_NONE: none)
__device__ __forceinline__ void mx4_keep_add(const Mx4Keep &K, uint64_t key, uint32_t room) {
    __syncthreads();
    const bool full = *K.n + room > MX4_KEEP;   // (the same for all threads: nobody adds before the next barrier)
    __syncthreads();
    if (full) mx4_keep_cut(K);
    if (key < *K.limit) K.keys[atomicAdd(K.n, 1u)] = key;
}
struct Mx4Select {
    Mx4Exact E;
    uint32_t nq, k, cap;
    const uint32_t *counts;
    const uint2 *cand;
    uint32_t *again;            // [nq]: 1 = the list did not hold the answer: k_mx4_again
    uint64_t *again_limit;      // [nq] ... which then needs nothing above this
    int64_t *ids;               // [nq][k]
    float *scores;
    // k_mx4_again: slices of the table per query and their results
    uint32_t slices;
    uint64_t *part;             // [nq][slices][k]
    uint32_t *ticket;           // [nq]
};
__device__ __forceinline__ void mx4_emit(const Mx4Select &S, uint32_t q, const uint64_t *keys, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < S.k; i += blockDim.x) {
        const uint64_t key = i < n ? keys[i] : MX4_NONE;
        S.ids[(size_t)q * S.k + i] = key == MX4_NONE ? -1 : (int64_t)(uint32_t)key;
        S.scores[(size_t)q * S.k + i] = key == MX4_NONE ? -1.f : mx4_unkey((uint32_t)(key >> 32));
    }
}
static __global__ __launch_bounds__(512) void k_mx4_select(Mx4Select S) {
    __shared__ uint64_t keys[MX4_KEEP];
    __shared__ uint32_t n_s;
    __shared__ uint64_t limit_s;
    const uint32_t q = blockIdx.x, found = S.counts[q], n = min(found, S.cap);
    const Mx4Keep K{keys, &n_s, &limit_s, S.k};
    if (threadIdx.x == 0) {
        n_s = 0;
        limit_s = MX4_NONE;
    }
    for (uint32_t i0 = 0; i0 < n; i0 += 512) {
        const uint32_t i = i0 + threadIdx.x;
        uint64_t key = MX4_NONE;
        if (i < n) {
            const uint2 c = S.cand[(size_t)q * S.cap + i];
            key = mx4_pack(__uint_as_float(c.y), c.x);
        }
        mx4_keep_add(K, key, 512);
    }
    mx4_keep_cut(K);
    const uint32_t got = n_s;
    const double sq = S.E.qsq[q];
    const bool dead = !(sq == sq) || (S.E.metric == MX4_COSINE && sq == 0);   // every score is NaN
    const bool again = !dead && (found > S.cap || got < min((uint64_t)S.k, S.E.rows.n));
    if (threadIdx.x == 0) {
        S.again[q] = again;
        S.ticket[q] = 0;
        S.again_limit[q] = got >= S.k ? keys[S.k - 1] : MX4_NONE - 1;
    }
    mx4_emit(S, q, keys, got);
}
// Queries whose candidates overflowed (many rows as near as the k-th), or were fewer than k: every row scored exactly, `slices`
// workgroups a query, the last one joins their lists.  It only ever reads memory of its own query and waits for nobody.
template <int BITS> static __global__ __launch_bounds__(512) void k_mx4_again(Mx4Select S) {
    __shared__ uint64_t keys[MX4_KEEP];
    __shared__ uint32_t n_s, last_s;
    __shared__ uint64_t limit_s;
    const uint32_t q = blockIdx.y;
    if (!S.again[q]) return;
    const Mx4Keep K{keys, &n_s, &limit_s, S.k};
    if (threadIdx.x == 0) {
        n_s = 0;
        limit_s = S.again_limit[q] + 1;
    }
    const uint64_t n = S.E.rows.n, per = (n + S.slices - 1) / S.slices, a = min(n, per * blockIdx.x), b = min(n, a + per);
    const uint32_t at_once = 512 / MX4_LANES;
    for (uint64_t r0 = a; r0 < b; r0 += at_once) {
        const uint64_t row = r0 + threadIdx.x / MX4_LANES;
        const float s = mx4_exact_score<BITS>(S.E, q, min(row, n - 1));
        mx4_keep_add(K, threadIdx.x % MX4_LANES == 0 && row < b ? mx4_pack(s, (uint32_t)row) : MX4_NONE, at_once);
    }
    mx4_keep_cut(K);
    uint64_t *mine = S.part + ((size_t)q * S.slices + blockIdx.x) * S.k;
    for (uint32_t i = threadIdx.x; i < S.k; i += 512) __hip_atomic_store(&mine[i], i < n_s ? keys[i] : MX4_NONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last_s = atomicAdd(&S.ticket[q], 1u) == S.slices - 1;
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    if (threadIdx.x == 0) {
        n_s = 0;
        limit_s = MX4_NONE;
    }
    const uint64_t total = (uint64_t)S.slices * S.k;
    const uint64_t *all = S.part + (size_t)q * total;
    for (uint64_t i0 = 0; i0 < total; i0 += 512) {
        const uint64_t i = i0 + threadIdx.x;
        mx4_keep_add(K, i < total ? __hip_atomic_load(&all[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : MX4_NONE, 512);
    }
    mx4_keep_cut(K);
    mx4_emit(S, q, keys, n_s);
}

}  // namespace vsg
