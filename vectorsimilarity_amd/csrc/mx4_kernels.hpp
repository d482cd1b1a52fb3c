// mx4_kernels.hpp -- MXFP4 rows: writing, reading back, rounding queries, exact scores, the k best (mx4_common.hpp has the format;
// mx4_scan_kernels.hpp the passes over the table).
#pragma once
#include "mx4_common.hpp"
#include "mx4_read_plan.h"

#include <type_traits>

namespace vsg {

__device__ __forceinline__ double mx4_pow2(int e) {   // 2^e, |e| <= 1000
    return __longlong_as_double((long long)(e + 1023) << 52);
}

template <int T> __device__ __forceinline__ float mx4_widen(const void *p, size_t i) {
    if constexpr (T == MX4_F32) return static_cast<const float *>(p)[i];
    else if constexpr (T == MX4_F16) return (float)static_cast<const _Float16 *>(p)[i];
    else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
}
// 16 bytes of a caller's vectors, aligned to their elements only (the memory takes a wide access at any of their addresses)
typedef float mx4_f4_at __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t mx4_u4_at __attribute__((ext_vector_type(4), aligned(2)));
template <int T> constexpr int MX4_EACH = T == MX4_F32 ? 4 : 8;   // elements of such an access
template <int T> __device__ __forceinline__ void mx4_widen16(const void *x, int i, float v[32]) {   // the i-th
    if constexpr (T == MX4_F32) {
        const mx4_f4_at w = static_cast<const mx4_f4_at *>(x)[i];
#pragma unroll
        for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
    } else {
        const mx4_u4_at w = static_cast<const mx4_u4_at *>(x)[i];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint16_t h = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
            v[8 * i + j] = T == MX4_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
        }
    }
}
// 32 elements from x on, `have` of them in the row
template <int T> __device__ __forceinline__ void mx4_load32(const void *x, int have, float v[32]) {
    constexpr int EACH = MX4_EACH<T>;
    if (have >= 32) {   // (by itself: all of its loads are under way together)
#pragma unroll
        for (int i = 0; i < 32 / EACH; i++) mx4_widen16<T>(x, i, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 32 / EACH; i++) {
        if (EACH * (i + 1) <= have) {
            mx4_widen16<T>(x, i, v);
        } else {
#pragma unroll
            for (int j = EACH * i; j < EACH * (i + 1); j++) v[j] = j < have ? mx4_widen<T>(x, (size_t)j) : 0.f;
        }
    }
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
// four dwords of E2M1 codes; returns sum x^2 of the rounded elements (multiples of 1/4 below 2^11: exact).  The conversion rounds to
// nearest even and saturates, as the format asks (checked against the definition at every tie and border)
__device__ __forceinline__ float mx4_codes4(const float v[32], float inv, bool bad, mx4_u4 &out) {
    float ss = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        uint32_t d = 0;
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w] * inv, v[8 * w + 1] * inv, 1.f, 0);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w + 2] * inv, v[8 * w + 3] * inv, 1.f, 1);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w + 4] * inv, v[8 * w + 5] * inv, 1.f, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * w + 6] * inv, v[8 * w + 7] * inv, 1.f, 3);
        out[w] = bad ? 0u : d;
        const mx4_f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(out[w], 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(out[w], 1.f, 1);
        const mx4_f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(out[w], 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(out[w], 1.f, 3);
        ss = __fmaf_rn(a[0], a[0], __fmaf_rn(a[1], a[1], __fmaf_rn(b[0], b[0], __fmaf_rn(b[1], b[1], ss))));
        ss = __fmaf_rn(c[0], c[0], __fmaf_rn(c[1], c[1], __fmaf_rn(e[0], e[0], __fmaf_rn(e[1], e[1], ss))));
    }
    return ss;
}
// six dwords of E2M3 codes; returns sum x^2 (multiples of 1/64 below 2^11: exact).  The instruction interleaves its two sources;
// it is given the even and the odd elements, clamped to the largest value
__device__ __forceinline__ float mx4_codes6(const float v[32], float inv, bool bad, mx4_u6 &out) {
    mx4_f16 even, odd;
#pragma unroll
    for (int j = 0; j < 16; j++) {
        even[j] = bad ? 0.f : fminf(fmaxf(v[2 * j] * inv, -7.5f), 7.5f);
        odd[j] = bad ? 0.f : fminf(fmaxf(v[2 * j + 1] * inv, -7.5f), 7.5f);
    }
    out = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, 1.f);
    const mx4_f32 r = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(out, 1.f);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 32; j++) ss = __fmaf_rn(r[j], r[j], ss);
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
// Which vector a slot gets when several name it: the last.  Two passes over the norms: cleared, then the largest 2^31 | i (4097 slots
// 2.6 us each, 1M in order 5.0, 1M in any order 20 and 41; up to 4096 vectors k_mx4_write looks for later ones with its slots itself).
static __global__ __launch_bounds__(256) void k_mx4_claim(Mx4Write W, int pass) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= W.m) return;
    const int64_t s = mx4_slot(W.slots, W.slots64, i, W.first);
    if (s < 0 || (uint64_t)s >= W.capacity) return;
    uint32_t *norm = reinterpret_cast<uint32_t *>(W.rows.at((uint64_t)s / 32) + W.rows.panel - 128) + (s & 31);
    if (pass == 0) __hip_atomic_store(norm, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else atomicMax(norm, 0x80000000u | (uint32_t)i);
}
// One workgroup takes 32 vectors, its waves (up to 16) the k-steps in turn; a lane rounds one block (half, row) by itself, so neither
// the maximum nor the codes cross lanes.  Bound by memory where slots follow each other: 1M x 768 bf16 into the first rows 350-375 us
// (1.95 GB at 5.2 TB/s or more; a copy of the card's: 4.76), by slots in order 405.  In any order 1160: a row's codes are 16-byte pieces
// 512 bytes apart (the counters: 1.0 GB stored for 0.41).  4097 x 1000 fp16 9.7 us.
template <int T> static __global__ __launch_bounds__(1024) void k_mx4_write(Mx4Write W) {
    __shared__ double part[16][64];
    __shared__ int64_t slot_s[32];
    __shared__ int lost_s[32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, row = lane & 31, half = lane >> 5;
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
    if (W.slots && !W.claimed && W.m > 1) {   // few vectors: a later vector with the same slot takes it
        for (uint64_t j = i0 + threadIdx.x; j < W.m; j += blockDim.x) {
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
        for (uint32_t s = wave; s < W.rows.ks; s += waves) {
            const int have = (int)W.rows.dim - (int)(2 * s + half) * 32;
            float v[32], inv;
            if (have > 0) mx4_load32<T>(x + (size_t)(2 * s + half) * 32 * esz, have, v);
            else {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = 0.f;
            }
            const int byte = mx4_scale(v, inv);
            mx4_u4 codes;
            const float sq = mx4_codes4(v, inv, byte == 255, codes);
            ss += byte == 255 ? __builtin_nan("") : (double)sq * mx4_pow2(2 * (byte - 127));
            *reinterpret_cast<mx4_u4 *>(panel + (size_t)s * 1024 + at * 16) = codes;
            char *scale = panel + (size_t)W.rows.ks * 1024 + (s >> 2) * 256 + at * 4 + (s & 3);
            *scale = (char)byte;
            if (s + 1 == W.rows.ks)   // the group's bytes past the last step: zero (mx4_qtile)
                for (uint32_t i = (s & 3) + 1; i < 4; i++) *++scale = 0;
        }
    }
    part[wave][lane] = ss;
    __syncthreads();
    if (threadIdx.x < 32 && slot >= 0) {
        double t = 0;
        for (int w = 0; w < waves; w++) t += part[w][lane] + part[w][lane + 32];
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
// 2^(byte - 127) in fp32 (byte 0: subnormal; 255: NaN)
__device__ __forceinline__ float mx4_scale_value(uint32_t byte) {
    return byte == 255 ? __uint_as_float(0x7FC00000u) : (byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
}
// A thread turns 8 codes (one dword) into 8 values; consecutive threads run along a row, so a wave's stores are contiguous.  Rows in
// any order cost the 64 bytes around each of their 16-byte pieces: 700K of 1M x 1024 to bf16 710 us (1.43 GB written, 1.79 GB read:
// 4.5 TB/s), 1M x 768 765.  In order 700K x 1024 take 370 us and 1M x 768 520: ten rows of 768 are a workgroup's, which share panels
// with rows of workgroups on other XCDs (0.70 GB read for 0.41).  100 rows of 128 2.6 us.  A workgroup takes `rows` whole rows
// (mx4_read_plan.h).
template <int T> static __global__ __launch_bounds__(256) void k_mx4_read(Mx4Read R, uint32_t rows, uint32_t per_row, uint32_t reciprocal) {
    const uint64_t i0 = (uint64_t)blockIdx.x * rows;
    const uint32_t work = (uint32_t)min((uint64_t)rows, R.m - i0) * per_row;
    for (uint32_t t = threadIdx.x; t < work; t += 256) {
        const uint32_t r = mx4_quotient(t, reciprocal), piece = t - r * per_row, e = piece * 8;
        const uint64_t i = i0 + r;
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
            const mx4_f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1);
            const mx4_f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 3);
            v[0] = a[0] * sc, v[1] = a[1] * sc, v[2] = b[0] * sc, v[3] = b[1] * sc, v[4] = c[0] * sc, v[5] = c[1] * sc, v[6] = d[0] * sc, v[7] = d[1] * sc;
        }
        char *o = R.out + i * R.stride;
        if constexpr (T == MX4_F32) {
            float *of = reinterpret_cast<float *>(o) + e;
            if (e + 8 <= R.rows.dim) {
                *reinterpret_cast<mx4_f4_at *>(of) = mx4_f4_at{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<mx4_f4_at *>(of + 4) = mx4_f4_at{v[4], v[5], v[6], v[7]};
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (e + j < R.rows.dim) of[j] = v[j];
            }
        } else {
            // E2M1 values have two digits: bf16 holds them exactly, its subnormals the smallest blocks'
            uint16_t h[8];
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = T == MX4_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[j]) : (uint16_t)(__float_as_uint(v[j]) >> 16);
            uint16_t *oh = reinterpret_cast<uint16_t *>(o) + e;
            if (e + 8 <= R.rows.dim) {
                mx4_u4_at w;
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = (uint32_t)h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
                *reinterpret_cast<mx4_u4_at *>(oh) = w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (e + j < R.rows.dim) oh[j] = h[j];
            }
        }
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
// The query block: operand tiles, then per query {norm fp32}, {|q|^2 fp64}.  A workgroup rounds one tile of 32, as k_mx4_write does its
// vectors, its waves the k-steps in turn: latency (1 x 128 2.4 us, 64 x 768 6.5, 256 x 1024 5.9).
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
template <int T, int BITS> static __global__ __launch_bounds__(1024) void k_mx4_queries(Mx4Queries Q) {
    __shared__ double part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, row = lane & 31, half = lane >> 5;
    const uint32_t q = blockIdx.x * 32 + row;
    char *tile = Q.tiles + (size_t)blockIdx.x * mx4_qtile(Q.dim, BITS);
    char *scales = tile + (size_t)Q.kg * (BITS == 6 ? 4 * 1536 : 4 * 1024);
    const int esz = T == MX4_F32 ? 4 : 2;
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < Q.zero_words; i += gridDim.x * blockDim.x) Q.zero[i] = 0;
    double ss = 0;
    for (uint32_t s = wave; s < Q.kg * 4; s += waves) {
        char *sc = scales + (s >> 2) * 256 + lane * 4 + (s & 3);
        const int have = q < Q.nq ? (int)Q.dim - (int)(2 * s + half) * 32 : 0;
        float v[32], inv;
        if (have > 0) mx4_load32<T>(Q.x + q * Q.stride + (size_t)(2 * s + half) * 32 * esz, have, v);
        else {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = 0.f;
        }
        const int byte = mx4_scale(v, inv);
        float sq;
        if constexpr (BITS == 6) {
            mx4_u6 w;
            sq = mx4_codes6(v, inv, byte == 255, w);
            *reinterpret_cast<mx4_u4 *>(tile + (size_t)s * 1024 + lane * 16) = mx4_u4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<mx4_u2 *>(tile + (size_t)Q.kg * 4096 + (size_t)s * 512 + lane * 8) = mx4_u2{w[4], w[5]};
        } else {
            mx4_u4 w;
            sq = mx4_codes4(v, inv, byte == 255, w);
            *reinterpret_cast<mx4_u4 *>(tile + (size_t)s * 1024 + lane * 16) = w;
        }
        *sc = (char)byte;
        ss += byte == 255 ? __builtin_nan("") : (double)sq * mx4_pow2(2 * (byte - 127));
    }
    part[wave][lane] = ss;
    __syncthreads();
    if (threadIdx.x < 32) {
        double t = 0;
        for (int w = 0; w < waves; w++) t += part[w][lane] + part[w][lane + 32];
        Q.sq[q] = t;
        Q.norm[q] = (float)sqrt(t);
    }
}

// ---------------------------------------------------------------------------------------------------------------- threshold
__device__ __forceinline__ uint32_t mx4_key(float f) {   // order-preserving; NaN is never passed
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float mx4_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
constexpr uint32_t MX4_KEY_INF = 0xFF800000u;   // key of infinity: not counted
constexpr uint32_t MX4_BINS = 2048;
struct Mx4Bins {   // shared
    uint32_t hist[MX4_BINS + MX4_BINS / 32];   // (a word free after every 32: the scan's lanes read 32 bins each)
    __device__ __forceinline__ uint32_t &bin(uint32_t i) { return hist[i + (i >> 5)]; }
    uint32_t lo, hi, pick, left, in;
};
// A number at or above the k-th smallest of n keys, and close to it (MX4_KEY_INF: fewer than k of them are finite).  Bins of equal
// width between the smallest and the largest key, then inside the bin of the k-th; a bin of few keys is near enough.  All threads.
template <typename F> __device__ __forceinline__ uint32_t mx4_kth(Mx4Bins &B, uint64_t n, uint32_t k, F key_of) {
    __syncthreads();
    if (threadIdx.x == 0) {
        B.lo = 0xFFFFFFFFu;
        B.hi = 0;
    }
    __syncthreads();
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint32_t key = key_of(i);
        if (key < MX4_KEY_INF) {
            lo = min(lo, key);
            hi = max(hi, key);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor(lo, o));
        hi = max(hi, (uint32_t)__shfl_xor(hi, o));
    }
    if ((threadIdx.x & 63) == 0) {
        atomicMin(&B.lo, lo);
        atomicMax(&B.hi, hi);
    }
    __syncthreads();
    lo = B.lo;
    hi = B.hi;
    if (lo > hi) return MX4_KEY_INF;
    uint32_t need = k;
    for (int pass = 0; pass < 4; pass++) {
        // bins of 2^shift keys from lo on
        const uint32_t range = hi - lo;
        const int shift = range < MX4_BINS ? 0 : 32 - __builtin_clz(range) - 11;
        for (uint32_t i = threadIdx.x; i < MX4_BINS + MX4_BINS / 32; i += blockDim.x) B.hist[i] = 0;
        if (threadIdx.x == 0) B.pick = 0xFFFFFFFFu;
        __syncthreads();
        for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t key = key_of(i);
            if (key >= lo && key <= hi && key < MX4_KEY_INF) atomicAdd(&B.bin((key - lo) >> shift), 1u);
        }
        __syncthreads();
        if (threadIdx.x < 64) {   // one wave: 32 bins a lane, then the lane's own
            const uint32_t b0 = threadIdx.x * (MX4_BINS / 64);
            uint32_t sum = 0, own[MX4_BINS / 64];
#pragma unroll
            for (uint32_t i = 0; i < MX4_BINS / 64; i++) sum += own[i] = B.bin(b0 + i);
            uint32_t before = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t t = __shfl_up(before, o);
                if ((int)threadIdx.x >= o) before += t;
            }
            before -= sum;
            if (before < need && need <= before + sum) {
                uint32_t pick = 0, left = 0, in = 0;
#pragma unroll
                for (uint32_t i = 0; i < MX4_BINS / 64; i++) {
                    if (before < need) pick = b0 + i, left = need - before, in = own[i];
                    before += own[i];
                }
                B.pick = pick;
                B.left = left;
                B.in = in;
            }
        }
        __syncthreads();
        const uint32_t pick = B.pick, left = B.left, in = B.in;
        __syncthreads();
        if (pick == 0xFFFFFFFFu) return MX4_KEY_INF;   // fewer than k finite keys
        hi = min(hi, lo + (pick << shift) + ((1u << shift) - 1));
        lo = lo + (pick << shift);
        need = left;
        if (shift == 0 || in <= 8 + k / 16) break;
    }
    return hi;
}
// The ranks of n <= room keys (MX4_NONE: none, without a rank) by counting: bins of equal width between the least and the largest score,
// keys in their bins' order, and a key's place in its bin by comparison with the others there.  False, and nothing done, when a bin
// holds too many (scores that crowd): then they are sorted.  All threads; emit(rank, key).
constexpr uint32_t MX4_CROWD = 128;
template <typename F> __device__ __forceinline__ bool mx4_ranked(Mx4Bins &B, const uint64_t *keys, uint32_t n, uint64_t *binned, F emit) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < MX4_BINS + MX4_BINS / 32; i += blockDim.x) B.hist[i] = 0;
    if (threadIdx.x == 0) {
        B.lo = 0xFFFFFFFFu;
        B.hi = 0;
        B.in = 0;
    }
    __syncthreads();
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
        if (keys[i] != ~0ull) {
            lo = min(lo, (uint32_t)(keys[i] >> 32));
            hi = max(hi, (uint32_t)(keys[i] >> 32));
        }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor(lo, o));
        hi = max(hi, (uint32_t)__shfl_xor(hi, o));
    }
    if ((threadIdx.x & 63) == 0) {
        atomicMin(&B.lo, lo);
        atomicMax(&B.hi, hi);
    }
    __syncthreads();
    lo = B.lo;
    hi = B.hi;
    if (lo > hi) return true;   // no key
    // (by the scores and not by their bits, which spread an exact match and the rest over all the powers of two between them)
    const float least = mx4_unkey(lo), range = mx4_unkey(hi) - least, per = range > 0 ? (float)MX4_BINS / range : 0.f;
    if (!(range < 3e38f) || !(per < 3e38f)) return false;
    const auto bin_of = [&](uint64_t key) { return min((uint32_t)((mx4_unkey((uint32_t)(key >> 32)) - least) * per), MX4_BINS - 1); };
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
        if (keys[i] != ~0ull) atomicAdd(&B.bin(bin_of(keys[i])), 1u);
    __syncthreads();
    if (threadIdx.x < 64) {   // counts -> first places
        const uint32_t b0 = threadIdx.x * (MX4_BINS / 64);
        uint32_t sum = 0, most = 0, own[MX4_BINS / 64];
#pragma unroll
        for (uint32_t i = 0; i < MX4_BINS / 64; i++) {
            sum += own[i] = B.bin(b0 + i);
            most = max(most, own[i]);
        }
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = __shfl_up(before, o);
            if ((int)threadIdx.x >= o) before += t;
        }
        before -= sum;
#pragma unroll
        for (uint32_t i = 0; i < MX4_BINS / 64; i++) {
            B.bin(b0 + i) = before;
            before += own[i];
        }
        atomicMax(&B.in, most);
    }
    __syncthreads();
    if (B.in > MX4_CROWD) return false;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
        if (keys[i] != ~0ull) binned[atomicAdd(&B.bin(bin_of(keys[i])), 1u)] = keys[i];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t key = keys[i];
        if (key == ~0ull) continue;
        const uint32_t bin = bin_of(key), first = bin ? B.bin(bin - 1) : 0, last = B.bin(bin);   // (a bin's place is now its end)
        uint32_t rank = first;
        for (uint32_t j = first; j < last; j++) rank += binned[j] < key;
        emit(rank, key);
    }
    return true;
}
struct Mx4Threshold {
    const float *minima;
    uint64_t stride, count;
    uint32_t k, metric;
    const float *qnorm;
    const double *qsq;
    float2 *limit;
    float *tau;
    float slack;
};
// a Cosine query of norm zero, or one that holds an infinity or a NaN: every score is NaN
__device__ __forceinline__ bool mx4_dead(uint32_t metric, double sq) { return !(sq == sq) || (metric == MX4_COSINE && sq == 0); }
// One workgroup a query, latency of a few passes over LDS: 256 queries of 7800 bounds 10.8 us, 1 of 400 4.2 us.
// tau = a little above the k-th smallest upper bound (each of different rows, so at least k rows are at or below it), then what the
// filter compares against
constexpr uint32_t MX4_STAGED = 16384;
static __global__ __launch_bounds__(1024) void k_mx4_threshold(Mx4Threshold T) {
    __shared__ Mx4Bins bins;
    __shared__ uint32_t staged[MX4_STAGED];   // (up to 2^14 bounds are read once)
    const uint32_t q = blockIdx.x;
    const float *m = T.minima + q * T.stride;
    uint32_t key = MX4_KEY_INF;
    if (T.k <= T.count) {
        if (T.count <= MX4_STAGED) {
            for (uint32_t i = threadIdx.x; i < T.count; i += 1024) staged[i] = mx4_key(m[i]);
            key = mx4_kth(bins, T.count, T.k, [&](uint64_t i) { return staged[i]; });
        } else {
            key = mx4_kth(bins, T.count, T.k, [&](uint64_t i) { return mx4_key(m[i]); });
        }
    }
    if (threadIdx.x) return;
    const float inf = __uint_as_float(0x7F800000u);
    const float yn = T.qnorm[q], tau = yn > MX4_LONG ? inf : mx4_unkey(key);
    T.tau[q] = tau;
    float2 l;
    if (T.metric == MX4_L2) {
        l.x = -T.slack * yn;
        l.y = 0.5f * ((1.f - MX4_EPS) * yn * yn - (tau + MX4_EPS * fabsf(tau)) - 2.f * MX4_TINY);
    } else if (T.metric == MX4_IP) {
        l.x = -T.slack * yn;
        l.y = 1.f - tau - MX4_STEP * fmaxf(1.f, fabsf(tau));
    } else {
        l.x = ((1.f - tau) - T.slack - MX4_STEP) * yn;
        l.y = yn < MX4_SHORT ? -inf : 1e-42f;   // (0: a zero vector's dot is 0, and its score NaN)
    }
    if (tau == inf) l = make_float2(0.f, -inf);
    if (mx4_dead(T.metric, T.qsq[q])) l = make_float2(0.f, inf);
    T.limit[q] = l;
}

// ---------------------------------------------------------------------------------------------------------------- exact scores
struct Mx4Exact {
    Mx4Rows rows;
    const char *tiles;
    uint32_t qtile_bytes, metric;
    const double *qsq;
};
template <typename F> __device__ __forceinline__ void mx4_unpack8(uint32_t codes, F use) {   // eight E2M1 elements
    const mx4_f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1);
    const mx4_f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 3);
    use(0, a[0]), use(1, a[1]), use(2, b[0]), use(3, b[1]), use(4, c[0]), use(5, c[1]), use(6, d[0]), use(7, d[1]);
}
// this lane's share of R rows' sums: blocks first, first + by, ...   In a block the sums are whole numbers (of 1/16): exact.
template <int BITS, int R> __device__ __forceinline__ void mx4_row_sums(const Mx4Exact &E, const char *tile, uint32_t col, const uint32_t (&row)[R],
                                                                        uint32_t first, uint32_t by, double (&dot)[R], double (&xx)[R]) {
    const uint32_t nb = E.rows.ks * 2;
    const char *panel[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        panel[i] = E.rows.at(row[i] >> 5);
        dot[i] = 0;
        xx[i] = 0;
    }
    for (uint32_t b = first; b < nb; b += by) {
        const uint32_t s = b >> 1, half = b & 1, qa = col + 32 * half;
        mx4_u4 x[R];
        uint32_t bx[R];
#pragma unroll
        for (int i = 0; i < R; i++) {   // (all rows' loads are under way before the first is used)
            const uint32_t ra = (row[i] & 31) + 32 * half;
            x[i] = *reinterpret_cast<const mx4_u4 *>(panel[i] + (size_t)s * 1024 + ra * 16);
            bx[i] = (uint8_t)panel[i][(size_t)E.rows.ks * 1024 + (s >> 2) * 256 + ra * 4 + (s & 3)];
        }
        const mx4_u4 lo = *reinterpret_cast<const mx4_u4 *>(tile + (size_t)s * 1024 + qa * 16);
        const uint32_t bq = (uint8_t)tile[(size_t)E.rows.kg * (BITS == 6 ? 4 * 1536 : 4 * 1024) + (s >> 2) * 256 + qa * 4 + (s & 3)];
        mx4_f32 qv;
        if constexpr (BITS == 6) {
            const mx4_u2 hi = *reinterpret_cast<const mx4_u2 *>(tile + (size_t)E.rows.kg * 4096 + (size_t)s * 512 + qa * 8);
            qv = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(mx4_u6{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1]}, 1.f);
        } else {
#pragma unroll
            for (int w = 0; w < 4; w++) mx4_unpack8(lo[w], [&](int j, float v) { qv[8 * w + j] = v; });
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            float d = 0, sq = 0;
#pragma unroll
            for (int w = 0; w < 4; w++)
                mx4_unpack8(x[i][w], [&](int j, float v) {
                    d = __fmaf_rn(v, qv[8 * w + j], d);
                    sq = __fmaf_rn(v, v, sq);
                });
            const double nan = __builtin_nan("");
            dot[i] += bx[i] == 255 || bq == 255 ? nan : (double)d * mx4_pow2((int)bx[i] + (int)bq - 254);
            xx[i] += bx[i] == 255 ? nan : (double)sq * mx4_pow2(2 * (int)bx[i] - 254);
        }
    }
}
__device__ __forceinline__ float mx4_final(uint32_t metric, double dot, double xx, double qq) {
    if (metric == MX4_IP) return (float)(1.0 - dot);
    if (metric == MX4_L2) return (float)(qq + xx - 2.0 * dot);
    return (float)(1.0 - dot / (sqrt(qq) * sqrt(xx)));
}
// lanes on one row: one for each of its blocks, 2 to 32
__host__ __device__ inline uint32_t mx4_row_lanes(uint32_t ks) { return ks <= 1 ? 2u : ks <= 2 ? 4u : (ks <= 4 ? 8u : (ks <= 8 ? 16u : 32u)); }
template <int BITS, int R> __device__ __forceinline__ void mx4_exact_scores(const Mx4Exact &E, uint32_t q, const uint32_t (&row)[R], uint32_t lanes, float (&score)[R]) {
    double dot[R], xx[R];
    mx4_row_sums<BITS, R>(E, E.tiles + (size_t)(q >> 5) * E.qtile_bytes, q & 31, row, threadIdx.x & (lanes - 1), lanes, dot, xx);
    const double qq = E.qsq[q];
#pragma unroll
    for (int i = 0; i < R; i++) {
        for (int o = (int)lanes / 2; o; o >>= 1) {
            dot[i] += __shfl_xor(dot[i], o);
            xx[i] += __shfl_xor(xx[i], o);
        }
        score[i] = mx4_final(E.metric, dot[i], xx[i], qq);
    }
}
template <int BITS> __device__ __forceinline__ float mx4_exact_score(const Mx4Exact &E, uint32_t q, uint32_t row, uint32_t lanes) {
    const uint32_t rows[1] = {row};
    float s[1];
    mx4_exact_scores<BITS, 1>(E, q, rows, lanes, s);
    return s[0];
}
// rows first .. first + m - 1, or ids[0 .. m)
template <int BITS> static __global__ __launch_bounds__(256) void k_mx4_exact_rows(Mx4Exact E, const uint32_t *ids, uint64_t first, uint64_t m, float *out) {
    const uint32_t lanes = mx4_row_lanes(E.rows.ks), at_once = 256 / lanes, me = threadIdx.x / lanes;
    for (uint64_t i = (uint64_t)blockIdx.x * at_once + me; i < m; i += (uint64_t)gridDim.x * at_once) {
        const float s = mx4_exact_score<BITS>(E, 0, ids ? ids[i] : (uint32_t)(first + i), lanes);
        if ((threadIdx.x & (lanes - 1)) == 0) out[i] = s;
    }
}

// ---------------------------------------------------------------------------------------------------------------- the k best
// order: (score, row), both ascending, as one 64-bit key; 0xFF.. = nothing (NaN scores become that)
constexpr uint64_t MX4_NONE = ~0ull;
__device__ __forceinline__ uint64_t mx4_pack(float s, uint32_t row) {
    if (!(s == s)) return MX4_NONE;
    return (uint64_t)mx4_key(s == 0.f ? 0.f : s) << 32 | row;   // (-0 and 0 are equal)
}
// ascending bitonic sort of n (a power of two) keys in LDS by the whole workgroup.  Thread t takes pair t: with strides to 64 a wave's
// pairs are 128 keys that nobody else touches, so that only longer strides need the workgroup's barrier.
__device__ __forceinline__ void mx4_sort(uint64_t *k, uint32_t n) {
    __syncthreads();
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (int s = 30 - __builtin_clz(size); s >= 0; s--) {
            const uint32_t stride = 1u << s;
            for (uint32_t t = threadIdx.x; t < n / 2; t += blockDim.x) {
                const uint32_t lo = (t >> s << (s + 1)) + (t & (stride - 1)), hi = lo + stride;
                const bool up = (lo & size) == 0;
                const uint64_t a = k[lo], b = k[hi];
                if ((a > b) == up) {
                    k[lo] = b;
                    k[hi] = a;
                }
            }
            if (stride > 64 || (stride == 1 && size >= 128)) __syncthreads();   // (the next stride is above 64, or this one was)
            else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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
// called by all threads, with at most `room` keys in all (MX4_NONE: none)
template <int R> __device__ __forceinline__ void mx4_keep_add(const Mx4Keep &K, const uint64_t (&key)[R], uint32_t room) {
    __syncthreads();
    const bool full = *K.n + room > MX4_KEEP || *K.n >= 2 * K.k + 512;   // (the same for all threads: nobody adds before the next barrier)
    __syncthreads();
    if (full) mx4_keep_cut(K);
#pragma unroll
    for (int i = 0; i < R; i++)
        if (key[i] < *K.limit) K.keys[atomicAdd(K.n, 1u)] = key[i];
}
struct Mx4Select {
    Mx4Exact E;
    uint32_t nq, k, segments, segment;
    const uint32_t *counts;     // [nq][segments]
    const Mx4Cand *cand;
    const float *minima, *qnorm;   // DENSE: [nq][n] upper bounds
    const float *tau;           // others: what the filter took rows by: k scores at least are at or below it
    float slack;
    uint32_t *again;            // [nq]: 1 = the list did not hold the answer: k_mx4_again
    uint64_t *again_limit;      // [nq] ... which then needs nothing above this
    int64_t *ids;               // [nq][k]
    float *scores;
    // k_mx4_finish: workgroups a query, what each of them leaves for the last one, and how many of them have
    uint32_t shares, room;
    uint64_t *share;            // [nq][shares][room]
    uint32_t *share_n;          // [nq][shares]
    uint32_t *done;             // [nq]
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
// Of a query's candidates only those whose lower bound is at or below the k-th smallest upper bound (little more than k) are scored
// exactly, a lane a block; then sorted.  DENSE: the candidates are all rows of a small table, their upper bounds the probe's
// (without a probe none, and every row is scored).  Few
// queries with many rows to score: `shares` workgroups a query, each with every shares-th 64 candidates; the last one to end joins them.
// Steps of latency, then the gather: 1 query, k 10 9.1 us (lists 2, bounds and their k-th 3.5, scores 1.1, ranks 0.9); 256 queries
// against 1M x 1024, k 100 34 us, of which 20 the 26 K rows' pieces (64 bytes of memory each); 7 queries, k 1000 27 us (one workgroup
// a query 52, with a bitonic sort of the k).
constexpr uint32_t MX4_FINISH = 1024;
constexpr uint32_t MX4_SHARES = 16;     // most workgroups a query
constexpr uint32_t MX4_LISTED = 6144;   // candidates kept in LDS; more are read from memory every time
template <int BITS, bool DENSE> static __global__ __launch_bounds__(1024) void k_mx4_finish(Mx4Select S) {
    __shared__ uint64_t keys[MX4_KEEP];
    __shared__ Mx4Bins bins;
    __shared__ __attribute__((aligned(8))) uint32_t up_s[MX4_LISTED];   // keys of the upper bounds
    __shared__ uint16_t segment_s[DENSE ? 1 : MX4_LISTED];   // where a candidate is listed
    __shared__ uint32_t rows_s[2 * MX4_FINISH];
    __shared__ uint32_t first_s[MX4_SEGMENTS + 1], n_s, rows_n, last_s;
    __shared__ uint64_t limit_s;
    __shared__ int over_s;
    const uint32_t q = blockIdx.x, me = blockIdx.y;
    const Mx4Keep K{keys, &n_s, &limit_s, S.k};
    static_assert(MX4_SEGMENTS == MX4_FINISH, "");
    const uint32_t have = !DENSE && threadIdx.x < S.segments ? S.counts[(size_t)q * S.segments + threadIdx.x] : 0;   // a segment a thread
    const float y = S.qnorm[q];
    if (threadIdx.x == 0) {
        first_s[0] = 0;
        n_s = 0;
        rows_n = 0;
        limit_s = MX4_NONE;
        over_s = 0;
    }
    __syncthreads();
    if constexpr (!DENSE) {
        if (have > S.segment || y > MX4_LONG) over_s = 1;   // (a long query's dots may be NaN where the scores are not)
        uint32_t sum = have;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = __shfl_up(sum, o);
            if ((int)(threadIdx.x & 63) >= o) sum += t;
        }
        if ((threadIdx.x & 63) == 63) up_s[threadIdx.x >> 6] = sum;
        __syncthreads();
        uint32_t waves = up_s[threadIdx.x & 15];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const uint32_t t = __shfl_up(waves, o);
            if ((int)(threadIdx.x & 15) >= o) waves += t;
        }
        if (threadIdx.x >= 64) sum += __shfl(waves, (int)(threadIdx.x >> 6) - 1);
        first_s[threadIdx.x + 1] = sum;
        for (uint32_t i = sum - have; i < min(sum, MX4_LISTED); i++) segment_s[i] = (uint16_t)threadIdx.x;
        __syncthreads();
        if (over_s) {   // part of the list is lost: every row is looked at (k_mx4_again)
            if (threadIdx.x == 0 && me == 0) {
                const bool dead = mx4_dead(S.E.metric, S.E.qsq[q]);
                S.again[q] = !dead;
                S.ticket[q] = 0;
                S.again_limit[q] = (uint64_t)mx4_key(S.tau[q]) << 32 | 0xFFFFFFFFu;
            }
            return;
        }
    }
    const uint32_t n = DENSE ? (uint32_t)S.E.rows.n : first_s[MX4_SEGMENTS];
    const auto listed = [&](uint32_t i) -> const Mx4Cand & {   // candidate i of all segments
        uint32_t seg = 0;
        if (i < MX4_LISTED) {
            seg = segment_s[i];
        } else {
#pragma unroll
            for (uint32_t step = MX4_SEGMENTS / 2; step; step >>= 1)
                if (first_s[seg + step] <= i) seg += step;
        }
        return S.cand[((size_t)q * S.segments + seg) * S.segment + (i - first_s[seg])];
    };
    const auto bounds = [&](const Mx4Cand &c, float &low, float &up) { mx4_bounds(S.E.metric, c.dot, c.x, y, S.slack, low, up); };
    const auto up_key = [&](uint64_t i) {
        float up, low;
        if constexpr (DENSE) up = y > MX4_LONG ? __uint_as_float(0x7F800000u) : S.minima[(size_t)q * S.E.rows.n + i];
        else bounds(listed((uint32_t)i), low, up);
        return up == up ? mx4_key(up) : MX4_KEY_INF;
    };
    const uint32_t lanes = mx4_row_lanes(S.E.rows.ks), at_once = MX4_FINISH / lanes;
    uint32_t key = MX4_KEY_INF;
    const bool all = DENSE && !S.minima;   // a table of few rows: every one of them
    if (n > S.k && !all) {
        if (n <= MX4_LISTED) {
            for (uint32_t i = threadIdx.x; i < n; i += MX4_FINISH) up_s[i] = up_key(i);
            key = mx4_kth(bins, n, S.k, [&](uint64_t i) { return up_s[i]; });
        } else {
            key = mx4_kth(bins, n, S.k, up_key);
        }
    }
    const float most = mx4_unkey(key);
    // rows worth an exact score, collected and scored MX4_FINISH or more at a time
    const uint32_t mine = (((n + 63) / 64 + S.shares - 1 - me) / S.shares) * 64;   // this workgroup's candidates, the last 64 perhaps fewer
    for (uint32_t j0 = 0; j0 < mine; j0 += MX4_FINISH) {
        const uint32_t j = j0 + threadIdx.x, i = ((j >> 6) * S.shares + me) * 64 + (j & 63);
        if (j < mine && i < n) {
            uint32_t row = i;
            float low;
            if (all) {
                low = -__uint_as_float(0x7F800000u);
            } else if constexpr (DENSE) {
                const float up = S.minima[(size_t)q * S.E.rows.n + i];
                const float x = reinterpret_cast<const float *>(S.E.rows.at(i / 32) + S.E.rows.panel - 128)[i & 31];
                low = mx4_low(S.E.metric, up, x, y, S.slack);
            } else {
                const Mx4Cand &c = listed(i);
                float up;
                row = c.row;
                bounds(c, low, up);
            }
            if (!(low > most)) rows_s[atomicAdd(&rows_n, 1u)] = row;
        }
        __syncthreads();
        const uint32_t m = rows_n;
        if (m <= MX4_FINISH && j0 + MX4_FINISH < mine) {   // (the same for all threads)
            __syncthreads();
            continue;
        }
        if (n_s + m > MX4_KEEP) mx4_keep_cut(K);
        const uint32_t base = n_s;
        const auto score = [&](auto each) {
            constexpr int R = decltype(each)::value;
            for (uint32_t r0 = threadIdx.x / lanes; r0 < m; r0 += R * at_once) {
                uint32_t row[R];
                float s[R];
#pragma unroll
                for (int i = 0; i < R; i++) row[i] = rows_s[min(r0 + i * at_once, m - 1)];
                mx4_exact_scores<BITS, R>(S.E, q, row, lanes, s);
#pragma unroll
                for (int i = 0; i < R; i++)
                    if ((threadIdx.x & (lanes - 1)) == 0 && r0 + i * at_once < m) keys[base + r0 + i * at_once] = mx4_pack(s[i], row[i]);
            }
        };
        if (m <= at_once) score(std::integral_constant<int, 1>{});
        else score(std::integral_constant<int, 2>{});
        __syncthreads();
        if (threadIdx.x == 0) {
            n_s = base + m;
            rows_n = 0;
        }
        __syncthreads();
    }
    if (S.shares > 1) {
        __syncthreads();
        if (n_s > S.room) mx4_keep_cut(K);   // (room >= k)
        uint64_t *to = S.share + ((size_t)q * S.shares + me) * S.room;
        for (uint32_t i = threadIdx.x; i < n_s; i += MX4_FINISH) __hip_atomic_store(&to[i], keys[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (threadIdx.x == 0) __hip_atomic_store(&S.share_n[q * S.shares + me], n_s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (threadIdx.x == 0) {   // (one thread's fences, on both sides, hold for the workgroup: the barriers are between)
            __threadfence();
            last_s = atomicAdd(&S.done[q], 1u) == S.shares - 1;
            __threadfence();
            n_s = 0;
            limit_s = MX4_NONE;
        }
        __syncthreads();
        if (!last_s) return;
        if (threadIdx.x <= MX4_SHARES) first_s[threadIdx.x] = 0;
        __syncthreads();
        if (threadIdx.x < S.shares) {
            const uint32_t m = __hip_atomic_load(&S.share_n[q * S.shares + threadIdx.x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            for (uint32_t w = threadIdx.x + 1; w <= S.shares; w++) atomicAdd(&first_s[w], m);
        }
        __syncthreads();
        const uint32_t total = first_s[S.shares];
        const uint64_t *from = S.share + (size_t)q * S.shares * S.room;
        for (uint32_t i0 = 0; i0 < total; i0 += MX4_FINISH) {
            const uint32_t i = i0 + threadIdx.x;
            uint32_t w = 0;
            while (w + 1 < S.shares && first_s[w + 1] <= i) w++;
            const bool have = i < total;
            const uint64_t key[1] = {have ? __hip_atomic_load(&from[(size_t)w * S.room + (i - first_s[w])], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : MX4_NONE};
            mx4_keep_add(K, key, MX4_FINISH);
        }
    }
    __syncthreads();
    const uint32_t scored = n_s;
    const auto conclude = [&](uint32_t got, uint64_t kth) {   // one thread
        S.again[q] = !DENSE && !mx4_dead(S.E.metric, S.E.qsq[q]) && got < min((uint64_t)S.k, S.E.rows.n);
        S.ticket[q] = 0;
        S.again_limit[q] = got >= S.k ? kth : MX4_NONE - 1;
    };
    if (2 * scored <= MX4_LISTED) {   // (up_s is free by now)
        if (threadIdx.x == 0) {
            rows_n = 0;
            limit_s = MX4_NONE;
        }
        __syncthreads();
        const auto emit = [&](uint32_t rank, uint64_t key) {
            if (rank < S.k) {
                S.ids[(size_t)q * S.k + rank] = (int64_t)(uint32_t)key;
                S.scores[(size_t)q * S.k + rank] = mx4_unkey((uint32_t)(key >> 32));
                if (rank == S.k - 1) limit_s = key;
            }
            atomicAdd(&rows_n, 1u);
        };
        bool done = true;
        if (scored > 256) {
            done = mx4_ranked(bins, keys, scored, reinterpret_cast<uint64_t *>(up_s), emit);
        } else if (threadIdx.x < scored && keys[threadIdx.x] != MX4_NONE) {   // few: against each of the others
            const uint64_t key = keys[threadIdx.x];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < scored; j++) rank += keys[j] < key;
            emit(rank, key);
        }
        __syncthreads();
        if (done) {
            const uint32_t got = rows_n;
            for (uint32_t i = got + threadIdx.x; i < S.k; i += MX4_FINISH) {
                S.ids[(size_t)q * S.k + i] = -1;
                S.scores[(size_t)q * S.k + i] = -1.f;
            }
            if (threadIdx.x == 0) conclude(got, limit_s);
            return;
        }
    }
    mx4_keep_cut(K);
    uint32_t got = n_s;
    while (got && keys[got - 1] == MX4_NONE) got--;   // NaN scores
    if (threadIdx.x == 0) conclude(got, keys[S.k - 1]);
    mx4_emit(S, q, keys, got);
}
// Queries whose candidates overflowed (many rows as near as the k-th, or beyond fp32), or were fewer than k: every row scored exactly,
// `slices` workgroups a query, the last one joins their lists.  It only ever reads memory of its own query and waits for nobody.  The
// grid is slices x groups: a group takes every groups-th query, so that the usual case -- nobody's list overflowed -- is a short launch
// (2.9 us).  41 queries, half of 67 K rows with one score: 288 us, most of it the slices' sorts.
template <int BITS> static __global__ __launch_bounds__(512, 4) void k_mx4_again(Mx4Select S) {
    __shared__ uint64_t keys[MX4_KEEP];
    __shared__ uint32_t n_s, last_s;
    __shared__ uint64_t limit_s;
    constexpr int EACH = 4;   // rows under way to a lane
    const uint32_t ask = blockIdx.y + threadIdx.x * gridDim.y;   // (all of a group's queries at once: a batch has fewer than threads)
    if (!__syncthreads_or(ask < S.nq && S.again[ask])) return;
    for (uint32_t q = blockIdx.y; q < S.nq; q += gridDim.y) {
        if (!S.again[q]) continue;
        const Mx4Keep K{keys, &n_s, &limit_s, S.k};
        __syncthreads();
        if (threadIdx.x == 0) {
            n_s = 0;
            limit_s = S.again_limit[q] + 1;
        }
        const uint64_t n = S.E.rows.n, per = (n + S.slices - 1) / S.slices, a = min(n, per * blockIdx.x), b = min(n, a + per);
        const uint32_t lanes = mx4_row_lanes(S.E.rows.ks), at_once = 512 / lanes;
        for (uint64_t r0 = a; r0 < b; r0 += EACH * at_once) {
            uint32_t row[EACH];
            float score[EACH];
            uint64_t key[EACH];
#pragma unroll
            for (int i = 0; i < EACH; i++) row[i] = (uint32_t)min(r0 + i * at_once + threadIdx.x / lanes, n - 1);
            mx4_exact_scores<BITS, EACH>(S.E, q, row, lanes, score);
#pragma unroll
            for (int i = 0; i < EACH; i++)
                key[i] = (threadIdx.x & (lanes - 1)) == 0 && r0 + i * at_once + threadIdx.x / lanes < b ? mx4_pack(score[i], row[i]) : MX4_NONE;
            mx4_keep_add(K, key, EACH * at_once);
        }
        mx4_keep_cut(K);
        uint64_t *mine = S.part + ((size_t)q * S.slices + blockIdx.x) * S.k;
        for (uint32_t i = threadIdx.x; i < S.k; i += 512) __hip_atomic_store(&mine[i], i < n_s ? keys[i] : MX4_NONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (threadIdx.x == 0) {   // (as in k_mx4_finish)
            __threadfence();
            last_s = atomicAdd(&S.ticket[q], 1u) == S.slices - 1;
            __threadfence();
            n_s = 0;
            limit_s = MX4_NONE;
        }
        __syncthreads();
        if (!last_s) continue;
        const uint64_t total = (uint64_t)S.slices * S.k;
        const uint64_t *all = S.part + (size_t)q * total;
        for (uint64_t i0 = 0; i0 < total; i0 += EACH * 512) {
            uint64_t key[EACH];
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                const uint64_t i = i0 + j * 512 + threadIdx.x;
                key[j] = i < total ? __hip_atomic_load(&all[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : MX4_NONE;
            }
            mx4_keep_add(K, key, EACH * 512);
        }
        mx4_keep_cut(K);
        mx4_emit(S, q, keys, n_s);
    }
}

}  // namespace vsg
