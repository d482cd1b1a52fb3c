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
struct Mx4Chunk {   // four k-steps of a panel
    mx4_i4 a[4];
    int sc;
};
template <bool ONCE> __device__ __forceinline__ void mx4_fetch(Mx4Chunk &c, const char *panel, uint32_t g, uint32_t ks, int lane) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t s = min(4 * g + i, ks - 1);   // (past the last step: the same bytes again, never used)
        const mx4_i4 *p = reinterpret_cast<const mx4_i4 *>(panel + (size_t)s * 1024) + lane;
        c.a[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
    }
    const int *sc = reinterpret_cast<const int *>(panel + (size_t)ks * 1024 + g * 256) + lane;
    c.sc = ONCE ? __builtin_nontemporal_load(sc) : *sc;
}
// QT query tiles' operands of k-step s = 4 g + i
template <int BITS> struct Mx4Operand {
    mx4_i4 lo;
    mx4_i2 hi;   // BITS == 6
    __device__ __forceinline__ void load(const char *tile, uint32_t s, uint32_t ks, int lane) {
        lo = reinterpret_cast<const mx4_i4 *>(tile + s * 1024)[lane];
        if constexpr (BITS == 6) hi = reinterpret_cast<const mx4_i2 *>(tile + ks * 1024 + s * 512)[lane];
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
constexpr int mx4_scan_waves(int bits, int qt, int nb, int src) {
    const int regs = (src == MX4_REGS ? qt * nb * (bits == 6 ? 25 : 17) : qt * 12) + qt * 16 + nb * 17 + 80;
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
static __global__ __launch_bounds__(256, mx4_scan_waves(BITS, QT, NB, SRC)) void k_mx4_scan(Mx4Scan P) {
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
    const uint32_t sc_at = ks * (BITS == 6 ? 1536 : 1024);
    Mx4Operand<BITS> op[SRC == MX4_REGS ? QT * 4 * NB : 1];
    int opsc[SRC == MX4_REGS ? QT * NB : 1];
    if constexpr (SRC == MX4_REGS) {
#pragma unroll
        for (int q = 0; q < QT; q++) {
            const char *tile = tiles + q * P.qtile_bytes;
#pragma unroll
            for (int s = 0; s < 4 * NB; s++) op[q * 4 * NB + s].load(tile, min((uint32_t)s, ks - 1), ks, lane);
#pragma unroll
            for (int g = 0; g < NB; g++) opsc[q * NB + g] = reinterpret_cast<const int *>(tile + sc_at + g * 256)[lane];
        }
    }
    float alpha[QT], beta[QT], qn[QT], qr[QT];
#pragma unroll
    for (int q = 0; q < QT; q++) {
        const uint32_t me = q0 + q * 32 + col;
        if constexpr (MODE == MX4_FILTER) {
            const float2 l = me < P.nq ? P.limit[me] : make_float2(0.f, __uint_as_float(0x7F800000u));
            alpha[q] = l.x;
            beta[q] = l.y;
        }
        qn[q] = yn_s[q * 32 + col];
        if constexpr (MODE == MX4_PROBE || MODE == MX4_PROBE_ROWS) qr[q] = yr_s[q * 32 + col];
    }
    bool shorts = false;   // DENSE, Cosine: queries whose reciprocal norm is no use
    if constexpr (MODE == MX4_DENSE) {
        for (int i = 0; i < QT * 32; i++) shorts |= yn_s[i] < MX4_SHORT && yn_s[i] > 0.f;
    }
    const uint32_t abreast = (blockDim.x / 64) / groups;   // panels that a workgroup's waves take at a time
    const uint64_t W = (uint64_t)gridDim.x * abreast;
    uint64_t w = (uint64_t)blockIdx.x * abreast + wave / groups;
    if (w >= P.n_take) return;
    const auto panel_of = [&](uint64_t i) { return P.n_take == P.n_panels ? i : i * P.n_panels / P.n_take; };
    // the wave's queue, 64 survivors at a time
    const auto flush = [&]() {
        for (uint32_t i = lane; i < queued; i += 64) {
            const mx4_u4 e = queue[i];
            mx4_admit(P, e[0], e[1], __uint_as_float(e[2]), __uint_as_float(e[3]), yn_s[e[0] - q0]);
        }
        queued = 0;
    };
    Mx4Chunk buf[NB];
    const char *panel = P.rows.at(panel_of(w));
#pragma unroll
    for (int g = 0; g < NB; g++)
        if (g < (int)kg) mx4_fetch<SRC != MX4_REGS>(buf[g], panel, g, ks, lane);
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
                for (int q = 0; q < QT; q++) sq[q] = SRC == MX4_REGS ? opsc[q * NB + j] : reinterpret_cast<const int *>(lds + q * P.qtile_bytes + sc_at + g * 256)[lane];
                const auto step = [&](auto index) {
                    constexpr int I = decltype(index)::value;
                    if (4 * g + I >= ks) return;
                    const mx4_i8 t{buf[j].a[I][0], buf[j].a[I][1], buf[j].a[I][2], buf[j].a[I][3], 0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < QT; q++) {
                        Mx4Operand<BITS> o;
                        if constexpr (SRC == MX4_REGS) o = op[q * 4 * NB + 4 * j + I];
                        else o.load(lds + q * P.qtile_bytes, 4 * g + I, ks, lane);
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
        const uint64_t row0 = p * 32;
        if constexpr (MODE == MX4_DENSE) {
            const uint64_t row = row0 + col;
            float *line = P.out + (q0 + 4 * half) * P.out_stride + row;
            const float *yl = yn_s + 4 * half;
            const float c0 = P.metric == MX4_L2 ? nx * nx : 1.f, rx = 1.f / nx;
            const bool divide = P.metric == MX4_COSINE && (shorts || __any(nx < MX4_SHORT && nx > 0.f));
            const bool whole = row0 + 32 <= P.rows.n && q0 + QT * 32 <= P.nq;
#pragma unroll
            for (int q = 0; q < QT; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const mx4_f4 y4 = *reinterpret_cast<const mx4_f4 *>(yl + q * 32 + 8 * i), r4 = *reinterpret_cast<const mx4_f4 *>(yl + block_q + q * 32 + 8 * i);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float d = acc[q][4 * i + j], y = y4[j];
                        float s;
                        if (P.metric == MX4_L2) s = __fmaf_rn(-2.f, d, __fmaf_rn(y, y, c0));
                        else if (P.metric == MX4_IP) s = 1.f - d;
                        else if (!divide) s = 1.f - d * rx * r4[j];
                        else s = 1.f - d / nx / y;
                        const uint32_t me = q * 32 + 8 * i + j;
                        if (whole || (q0 + me + 4 * half < P.nq && row < P.rows.n)) __builtin_nontemporal_store(s, line);
                        line += j < 3 ? P.out_stride : 5 * P.out_stride;
                    }
                }
        } else if constexpr (MODE == MX4_FILTER) {
            // a survivor when its score may be at or below the query's threshold: dot >= alpha |x| + beta + (L2: |x|^2 / 2)
            float base[16];
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const float x = nrm[v >> 2][v & 3];
                base[v] = P.metric == MX4_L2 ? 0.5f * (1.f - MX4_EPS) * x * x : 0.f;
                if (P.metric == MX4_COSINE && x < MX4_SHORT) base[v] = x > 0.f ? -__uint_as_float(0x7F800000u) : __uint_as_float(0x7F800000u);   // (zero: score NaN)
            }
#pragma unroll
            for (int q = 0; q < QT; q++) {
                bool any = false;
#pragma unroll
                for (int v = 0; v < 16; v++) any |= acc[q][v] >= __fmaf_rn(alpha[q], nrm[v >> 2][v & 3], base[v] + beta[q]);
                if (__any(any)) {
                    const uint32_t me = q0 + q * 32 + col;
                    uint32_t total = 0;
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const bool hit = acc[q][v] >= __fmaf_rn(alpha[q], nrm[v >> 2][v & 3], base[v] + beta[q]);
                        total += __builtin_popcountll(__ballot(hit));
                    }
                    if (queued + total > MX4_QUEUE) flush();
                    const bool direct = total > MX4_QUEUE;   // a panel full of survivors
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const float x = nrm[v >> 2][v & 3], d = acc[q][v];
                        const uint64_t row = row0 + 8 * (v >> 2) + 4 * half + (v & 3);
                        const bool hit = d >= __fmaf_rn(alpha[q], x, base[v] + beta[q]) && row < P.rows.n;
                        const uint64_t b = __ballot(hit);
                        if (b == 0) continue;
                        if (direct) {
                            if (hit) mx4_admit(P, me, (uint32_t)row, d, x, qn[q]);
                        } else {
                            if (hit) queue[queued + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0u))] =
                                mx4_u4{me, (uint32_t)row, __float_as_uint(d), __float_as_uint(x)};
                            queued += __builtin_popcountll(b);
                        }
                    }
                }
            }
        } else {
            const float inf = __uint_as_float(0x7F800000u);
            float rx[16];
            if (P.metric == MX4_COSINE) {
#pragma unroll
                for (int v = 0; v < 16; v++) rx[v] = __builtin_amdgcn_rcpf(nrm[v >> 2][v & 3]);
            }
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const uint32_t me = q0 + q * 32 + col;
                float best = inf;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const float x = nrm[v >> 2][v & 3], d = acc[q][v];
                    const uint64_t row = row0 + 8 * (v >> 2) + 4 * half + (v & 3);
                    float u;   // an upper bound of the score (mx4_bounds, with reciprocals: two more roundings, in the slack)
                    if (P.metric == MX4_L2) u = __fmaf_rn(2.f * P.slack * qn[q], x, __fmaf_rn(-2.f, d, __fmaf_rn(1.f + MX4_EPS, __fmaf_rn(x, x, qn[q] * qn[q]), MX4_TINY)));
                    else if (P.metric == MX4_IP) u = __fmaf_rn(P.slack * qn[q], x, 1.f - d) + MX4_STEP * fmaxf(1.f, fabsf(1.f - d));
                    else {
                        u = 1.f - d * rx[v] * qr[q] + (P.slack + MX4_STEP);
                        if (x < MX4_SHORT || qn[q] < MX4_SHORT) u = x > 0.f ? 2.001f : inf;
                    }
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
    if constexpr (MODE == MX4_FILTER) flush();
}

}  // namespace vsg
