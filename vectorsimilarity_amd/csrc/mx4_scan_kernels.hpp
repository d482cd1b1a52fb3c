// mx4_scan_kernels.hpp -- the passes over a table of MXFP4 rows: every row's dot with every query on the matrix cores, then the
// scores themselves (DENSE), upper bounds of a sample (PROBE, PROBE_ROWS) or the rows that may be among the k best (FILTER).
#pragma once
#include "mx4_common.hpp"

#include <type_traits>

namespace vsg {

// one operand pair and its scales; the table is the A operand (results: a lane one query, its registers 16 rows) or, for dense
// scores, the B operand (a lane one row: stores along a query's line)
template <int BITS, bool SWAP, int I> __device__ __forceinline__ mx4_f16 mx4_mma(mx4_i8 t, mx4_i8 q, mx4_f16 c, int st, int sq) {
    constexpr int FQ = BITS == 6 ? 2 : 4;
    if constexpr (SWAP) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(q, t, c, FQ, 4, I, sq, I, st);
    else return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(t, q, c, 4, FQ, I, st, I, sq);
}
template <typename T> __device__ __forceinline__ const __attribute__((address_space(1))) T *mx4_in_memory(uint64_t address) {
    return (const __attribute__((address_space(1))) T *)address;
}
struct Mx4Chunk {   // four k-steps of a panel
    mx4_i4 a[4];
    int sc;
};
template <bool ONCE> __device__ __forceinline__ void mx4_fetch(Mx4Chunk &c, uint64_t panel, uint32_t g, uint32_t ks, int lane) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t s = min(4 * g + i, ks - 1);   // (past the last step: the last one again, against zeros)
        const auto p = mx4_in_memory<mx4_i4>(panel + (size_t)s * 1024) + lane;
        c.a[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
    }
    const auto sc = mx4_in_memory<int>(panel + (size_t)ks * 1024 + g * 256) + lane;
    c.sc = ONCE ? __builtin_nontemporal_load(sc) : *sc;
}
// QT query tiles' operands of k-step s = 4 g + i
template <int BITS> struct Mx4Operand {
    mx4_i4 lo;
    mx4_i2 hi;   // BITS == 6
    __device__ __forceinline__ void load(const char *tile, uint32_t s, uint32_t kg, int lane) {
        lo = reinterpret_cast<const mx4_i4 *>(tile + s * 1024)[lane];
        if constexpr (BITS == 6) hi = reinterpret_cast<const mx4_i2 *>(tile + kg * 4096 + s * 512)[lane];
    }
    __device__ __forceinline__ mx4_i8 get() const {
        if constexpr (BITS == 6) return mx4_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], 0, 0};
        else return mx4_i8{lo[0], lo[1], lo[2], lo[3], 0, 0, 0, 0};
    }
};
// a candidate into its query's list (segments of counters: one counter would make all waves wait in line for it)
__device__ __forceinline__ void mx4_admit(const Mx4Scan &P, uint32_t q, uint32_t row, float d, float x, float y) {
    const uint32_t seg = q * MX4_SEGMENTS + ((row >> 5) & (MX4_SEGMENTS - 1));
    const uint32_t at = atomicAdd(&P.counts[seg], 1u);
    if (at < P.segment) {
        Mx4Cand c{row, 0.f, 0.f, 0u};
        mx4_bounds(P.metric, d, x, y, P.slack, c.low, c.up);
        P.cand[(size_t)seg * P.segment + at] = c;
    }
}

// registers of a wave, about: what its operands, sums and panel in flight need
constexpr int mx4_scan_waves(int bits, int qt, int mode, int nb, int src) {
    const int regs = (src == MX4_REGS ? qt * nb * (bits == 6 ? 25 : 17) : qt * 12) + qt * 16 + nb * 17 + (mode == MX4_DENSE ? 60 : 105);
    return regs <= 128 ? 4 : (regs <= 168 ? 3 : (regs <= 256 ? 2 : 1));
}
// A wave takes whole panels, one after the other, every wave of the grid in turn.  NB chunks of the panel (256 elements each) are in
// flight: chunk g of the next panel is requested as soon as chunk g of this one has gone into the matrix cores.  Panels of more than
// 4 chunks go through the same four buffers several times.  The queries' operands (SRC) are
//   up to 64 queries          in LDS, read per k-step: the registers hold more of the table in flight instead
//   more, rows to 1024        in registers: LDS could not feed the matrix cores (1.5 KiB a tile and step against 32 cycles of matrix
//                             work on each of four SIMDs), so a wave keeps two tiles and `groups` waves take the same panels, which
//                             then come from the CU's own cache
//   rows beyond the LDS       in global memory, through the caches
template <int BITS, int QT, int MODE, int NB, int SRC>
static __global__ __launch_bounds__(256, mx4_scan_waves(BITS, QT, MODE, NB, SRC)) void k_mx4_scan(Mx4Scan P) {
    extern __shared__ char shared[];
    constexpr bool SWAP = MODE == MX4_DENSE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const uint32_t groups = SRC == MX4_REGS ? P.groups : 1, group = SRC == MX4_REGS ? wave % groups : 0;
    const uint32_t block_q0 = blockIdx.y * groups * QT * 32, q0 = block_q0 + group * QT * 32;
    const uint32_t ks = P.rows.ks, kg = SRC == MX4_REGS ? NB : P.rows.kg;
    const char *tiles = P.tiles + (size_t)(q0 / 32) * P.qtile_bytes;
    const char *lds = SRC == MX4_SHARED ? shared : tiles;
    const uint32_t block_q = groups * QT * 32;
    float *yn_b = reinterpret_cast<float *>(shared + (SRC == MX4_SHARED ? QT * P.qtile_bytes : 0));   // |q|, 1 / |q| of the workgroup's queries
    mx4_u4 *queue = reinterpret_cast<mx4_u4 *>(yn_b + 2 * block_q) + wave * MX4_QUEUE;   // FILTER: {query, row, dot, |x|}
    uint32_t queued = 0;
    if constexpr (SRC == MX4_SHARED) {
        const mx4_u4 *src = reinterpret_cast<const mx4_u4 *>(tiles);
        const uint32_t n16 = QT * P.qtile_bytes / 16;
        for (uint32_t i = threadIdx.x; i < n16; i += blockDim.x) reinterpret_cast<mx4_u4 *>(shared)[i] = src[i];
    }
    for (uint32_t i = threadIdx.x; i < block_q; i += blockDim.x) {
        const float y = P.qnorm[block_q0 + i];   // (padded to whole tiles)
        yn_b[i] = y;
        yn_b[block_q + i] = 1.f / y;
    }
    __syncthreads();
    const float *yn_s = yn_b + group * QT * 32, *yr_s = yn_s + block_q;
    const uint32_t sc_at = kg * (BITS == 6 ? 4 * 1536 : 4 * 1024);
    Mx4Operand<BITS> op[SRC == MX4_REGS ? QT * 4 * NB : 1];
    int opsc[SRC == MX4_REGS ? QT * NB : 1];
    if constexpr (SRC == MX4_REGS) {
#pragma unroll
        for (int q = 0; q < QT; q++) {
            const char *tile = tiles + q * P.qtile_bytes;
#pragma unroll
            for (int s = 0; s < 4 * NB; s++) op[q * 4 * NB + s].load(tile, s, NB, lane);
#pragma unroll
            for (int g = 0; g < NB; g++) opsc[q * NB + g] = reinterpret_cast<const int *>(tile + sc_at + g * 256)[lane];
        }
    }
    // FILTER: what a row's dot is held against (k_mx4_threshold); PROBE: |q|, 1 / |q|
    float alpha[QT], beta[QT];
#pragma unroll
    for (int q = 0; q < QT; q++) {
        const uint32_t me = q0 + q * 32 + col;
        if constexpr (MODE == MX4_FILTER) {
            const float2 l = me < P.nq ? P.limit[me] : make_float2(0.f, __uint_as_float(0x7F800000u));
            alpha[q] = l.x;
            beta[q] = l.y;
        } else {
            alpha[q] = yn_s[q * 32 + col];
            beta[q] = yr_s[q * 32 + col];
        }
    }
    bool shorts = false;   // DENSE, Cosine: queries whose reciprocal norm is no use
    if constexpr (MODE == MX4_DENSE) {
        for (int i = lane; i < QT * 32; i += 64) shorts |= yn_s[i] < MX4_SHORT && yn_s[i] > 0.f;
        shorts = __any(shorts);
    }
    const uint32_t abreast = (blockDim.x / 64) / groups;   // panels that a workgroup's waves take at a time
    const uint32_t W = gridDim.x * abreast, n_take = (uint32_t)P.n_take;
    uint32_t w = blockIdx.x * abreast + wave / groups;
    if (w >= n_take) return;
    const auto panel_of = [&](uint32_t i) -> uint64_t { return MODE == MX4_PROBE ? (i * P.every) >> 24 : i; };
    // the wave's queue, 64 survivors at a time
    const auto flush = [&]() {
        for (uint32_t i = lane; i < queued; i += 64) {
            const mx4_u4 e = queue[i];
            mx4_admit(P, e[0], e[1], __uint_as_float(e[2]), __uint_as_float(e[3]), yn_s[e[0] - q0]);
        }
        queued = 0;
    };
    Mx4Chunk buf[NB];
    mx4_f4 nrm[4];   // |x| of this lane's 16 rows (DENSE: nx, its one row), loaded with the panel's first chunks
    float nx = 0.f;
    const auto fetch_norms = [&](uint64_t of) {
        if constexpr (SWAP) nx = mx4_in_memory<float>(of + P.rows.panel - 128)[col];
        else {
#pragma unroll
            for (int i = 0; i < 4; i++) nrm[i] = mx4_in_memory<mx4_f4>(of + P.rows.panel - 128)[2 * i + half];
        }
    };
    uint64_t panel = P.rows.uniform_at(panel_of(w));
    fetch_norms(panel);
#pragma unroll
    for (int g = 0; g < NB; g++)
        if (g < (int)kg) mx4_fetch<SRC != MX4_REGS>(buf[g], panel, g, ks, lane);
    for (; w < n_take; w += W) {
        const uint64_t p = panel_of(w);
        const uint32_t wn = w + W;
        const uint64_t next = wn < n_take ? P.rows.uniform_at(panel_of(wn)) : panel;   // (at the end: this panel again, never used)
        mx4_f16 acc[QT];
#pragma unroll
        for (int q = 0; q < QT; q++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[q][v] = 0.f;
        for (uint32_t g0 = 0; g0 < kg; g0 += NB) {
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const uint32_t g = g0 + j;
                if (g >= kg) break;
                int sq[QT];
#pragma unroll
                for (int q = 0; q < QT; q++) sq[q] = SRC == MX4_REGS ? opsc[q * NB + j] : reinterpret_cast<const int *>(lds + q * P.qtile_bytes + sc_at + g * 256)[lane];
                const auto step = [&](auto index) {
                    constexpr int I = decltype(index)::value;
                    const mx4_i8 t{buf[j].a[I][0], buf[j].a[I][1], buf[j].a[I][2], buf[j].a[I][3], 0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < QT; q++) {
                        Mx4Operand<BITS> o;
                        if constexpr (SRC == MX4_REGS) o = op[q * 4 * NB + 4 * j + I];
                        else o.load(lds + q * P.qtile_bytes, 4 * g + I, kg, lane);
                        acc[q] = mx4_mma<BITS, SWAP, I>(t, o.get(), acc[q], buf[j].sc, sq[q]);
                    }
                };
                step(std::integral_constant<int, 0>{});
                step(std::integral_constant<int, 1>{});
                step(std::integral_constant<int, 2>{});
                step(std::integral_constant<int, 3>{});
                // the buffer's next contents: NB chunks on in this panel, or the chunk of the next panel that it takes
                if (SRC != MX4_REGS && g + NB < kg) mx4_fetch<true>(buf[j], panel, g + NB, ks, lane);
                else mx4_fetch<SRC != MX4_REGS>(buf[j], next, j, ks, lane);
            }
        }
        // this panel's norms, and the next one's on their way
        mx4_f16 xn;
        const float xrow = nx;
#pragma unroll
        for (int v = 0; v < 16; v++) xn[v] = nrm[v >> 2][v & 3];
        fetch_norms(next);
        const uint64_t row0 = p * 32;
        const bool tail = row0 + 32 > P.rows.n;
        const float inf = __uint_as_float(0x7F800000u), nan = __uint_as_float(0x7FC00000u);
        const auto row_of = [&](int v) { return row0 + 8 * (v >> 2) + 4 * half + (v & 3); };
        const auto dense = [&](auto metric, auto whole, auto divide) {
            constexpr int M = decltype(metric)::value;
            const uint64_t row = row0 + col;
            float *line = P.out + (q0 + 4 * half) * P.out_stride + row;
            const float c0 = xrow * xrow, rx = 1.f / xrow;
#pragma unroll
            for (int q = 0; q < QT; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const mx4_f4 y4 = *reinterpret_cast<const mx4_f4 *>(yn_s + 4 * half + q * 32 + 8 * i);
                    const mx4_f4 r4 = *reinterpret_cast<const mx4_f4 *>(yr_s + 4 * half + q * 32 + 8 * i);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float d = acc[q][4 * i + j], y = y4[j];
                        float s;
                        if constexpr (M == MX4_L2) s = __fmaf_rn(-2.f, d, __fmaf_rn(y, y, c0));
                        else if constexpr (M == MX4_IP) s = 1.f - d;
                        else if constexpr (decltype(divide)::value) s = 1.f - d / xrow / y;
                        else s = 1.f - d * rx * r4[j];
                        if (decltype(whole)::value || (q0 + q * 32 + 8 * i + 4 * half + j < P.nq && row < P.rows.n)) __builtin_nontemporal_store(s, line);
                        line += j < 3 ? P.out_stride : 5 * P.out_stride;
                    }
                }
        };
        // a survivor when its score may be at or below the query's threshold.  f is the dot less what its row asks for, and is held
        // against one number a query:  L2 dot + slack |q| |x| - |x|^2 / 2,  IP dot + slack |q| |x|,  Cosine dot / |x|
        const auto filter = [&](auto metric) {
            constexpr int M = decltype(metric)::value;
            mx4_f16 h;
            bool odd = false;   // Cosine: vectors too short for this arithmetic go on to the exact one
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const float x = xn[v];
                if constexpr (M == MX4_L2) h[v] = 0.5f * (1.f - MX4_EPS) * x * x;
                if constexpr (M == MX4_COSINE) {
                    h[v] = __builtin_amdgcn_rcpf(x);   // (zero: 0 x infinity is NaN, never a survivor)
                    odd |= x < MX4_SHORT && x > 0.f;
                }
            }
            odd = M == MX4_COSINE && __any(odd);
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const float bound = M == MX4_COSINE && beta[q] == 0.f ? alpha[q] : beta[q];
                const auto f = [&](int v) {
                    const float x = xn[v], d = acc[q][v];
                    if constexpr (M == MX4_L2) return __fmaf_rn(-alpha[q], x, d) - h[v];
                    else if constexpr (M == MX4_IP) return __fmaf_rn(-alpha[q], x, d);
                    else return d * h[v];
                };
                float most = f(0);
#pragma unroll
                for (int v = 1; v < 16; v++) most = fmaxf(most, f(v));
                if (!__any(most >= bound) && !odd) continue;
                if (queued > MX4_QUEUE - 128) flush();
                const uint32_t me = q0 + q * 32 + col, before = queued;
                bool spilt = false;
                const auto hit = [&](int v) {
                    const float x = xn[v];
                    return (f(v) >= bound || (M == MX4_COSINE && x < MX4_SHORT && x > 0.f && bound < inf)) && row_of(v) < P.rows.n;
                };
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const bool mine = hit(v);
                    const uint64_t b = __ballot(mine);
                    if (b == 0) continue;
                    const uint32_t at = queued + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0u));
                    queued += __builtin_popcountll(b);
                    spilt |= queued > MX4_QUEUE;
                    if (mine && at < MX4_QUEUE) queue[at] = mx4_u4{me, (uint32_t)row_of(v), __float_as_uint(acc[q][v]), __float_as_uint(xn[v])};
                }
                if (spilt) {   // a panel full of survivors: this tile's again, straight to the lists
                    queued = before;
#pragma unroll 1
                    for (int v = 0; v < 16; v++)
                        if (hit(v)) mx4_admit(P, me, (uint32_t)row_of(v), acc[q][v], xn[v], yn_s[q * 32 + col]);
                }
            }
        };
        // the smallest upper bound (mx4_bounds, with a reciprocal's rounding in the slack) of this lane's 16 rows
        const auto probe = [&](auto metric) {
            constexpr int M = decltype(metric)::value;
            float h[16];
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const float x = xn[v];
                const bool none = tail && row_of(v) >= P.rows.n;
                if constexpr (M == MX4_L2) h[v] = none ? inf : (1.f + MX4_EPS) * x * x;
                else if constexpr (M == MX4_IP) h[v] = none ? inf : 0.f;
                else h[v] = none || x < MX4_SHORT ? nan : __builtin_amdgcn_rcpf(x);
            }
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const uint32_t me = q0 + q * 32 + col;
                const float y = alpha[q], c = P.slack * y;
                const auto up = [&](float best) {
                    float u;
                    if constexpr (M == MX4_L2) u = best + __fmaf_rn((1.f + MX4_EPS) * y, y, MX4_TINY);
                    else if constexpr (M == MX4_IP) u = 1.f + best, u = u + MX4_STEP * fmaxf(1.f, fabsf(u));
                    else u = y < MX4_SHORT ? inf : __fmaf_rn(best, beta[q], 1.f + P.slack + MX4_STEP);
                    return u == u ? u : inf;
                };
                const auto g = [&](int v) {   // smaller is nearer
                    const float x = xn[v], d = acc[q][v];
                    if constexpr (M == MX4_L2) return __fmaf_rn(2.f * c, x, __fmaf_rn(-2.f, d, h[v]));
                    else if constexpr (M == MX4_IP) return __fmaf_rn(c, x, h[v] - d);
                    else return -d * h[v];
                };
                if constexpr (MODE == MX4_PROBE_ROWS) {
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (me < P.nq && row_of(v) < P.rows.n) P.minima[me * P.minima_stride + row_of(v)] = up(g(v));
                } else {
                    float best = g(0);
#pragma unroll
                    for (int v = 1; v < 16; v++) best = fminf(best, g(v));
                    if (me < P.nq) P.minima[me * P.minima_stride + 2 * w + half] = up(best);
                }
            }
        };
        constexpr std::integral_constant<int, MX4_L2> l2{};
        constexpr std::integral_constant<int, MX4_IP> ip{};
        constexpr std::integral_constant<int, MX4_COSINE> cosine{};
        if constexpr (MODE == MX4_DENSE) {
            const bool whole = !tail && q0 + QT * 32 <= P.nq;
            if (P.metric == MX4_L2) {
                if (whole) dense(l2, std::true_type{}, std::false_type{});
                else dense(l2, std::false_type{}, std::false_type{});
            } else if (P.metric == MX4_IP) {
                if (whole) dense(ip, std::true_type{}, std::false_type{});
                else dense(ip, std::false_type{}, std::false_type{});
            } else if (shorts || __any(xrow < MX4_SHORT && xrow > 0.f)) {
                dense(cosine, std::false_type{}, std::true_type{});
            } else if (whole) {
                dense(cosine, std::true_type{}, std::false_type{});
            } else {
                dense(cosine, std::false_type{}, std::false_type{});
            }
        } else if constexpr (MODE == MX4_FILTER) {
            if (P.metric == MX4_L2) filter(l2);
            else if (P.metric == MX4_IP) filter(ip);
            else filter(cosine);
        } else {
            if (P.metric == MX4_L2) probe(l2);
            else if (P.metric == MX4_IP) probe(ip);
            else probe(cosine);
        }
        panel = next;
    }
    if constexpr (MODE == MX4_FILTER) flush();
}

}  // namespace vsg
