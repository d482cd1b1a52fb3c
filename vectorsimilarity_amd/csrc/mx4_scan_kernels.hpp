// mx4_scan_kernels.hpp -- the passes over a table of MXFP4 rows: every row's dot with every query on the matrix cores, then the
// scores themselves (DENSE), upper bounds of a sample (PROBE, PROBE_ROWS) or the rows that may be among the k best (FILTER).
#pragma once
#include "mx4_host.hpp"

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
// What a row's dot is held against: f(dot, row) >= beta when the row's score may be at or below the query's threshold
// (k_mx4_threshold).  L2 dot + slack |q| |x| - |x|^2 / 2,  IP dot + slack |q| |x|,  Cosine dot - least cosine x |q| |x|
template <int M> __device__ __forceinline__ float mx4_held(float d, float x, float alpha) {
    const float f = __fmaf_rn(-alpha, x, d);
    if constexpr (M == MX4_L2) return __fmaf_rn(x * (-0.5f * (1.f - MX4_EPS)), x, f);
    else return f;
}
// rows that fp32 arithmetic says nothing about: they go on to the exact one (zero vectors, whose Cosine is NaN, need not)
template <int M> __device__ __forceinline__ bool mx4_beyond(float x) { return x > MX4_LONG || (M == MX4_COSINE && x < MX4_SHORT && x > 0.f); }
// this lane's survivors
template <int M> __device__ __forceinline__ uint32_t mx4_survivors(const mx4_f16 &d, const mx4_f16 &x, float alpha, float beta) {
    uint32_t mask = 0;
#pragma unroll
    for (int v = 0; v < 16; v++) {
        bool hit = mx4_held<M>(d[v], x[v], alpha) >= beta;
        hit |= mx4_beyond<M>(x[v]) && beta < __uint_as_float(0x7F800000u);
        mask |= hit ? 1u << v : 0u;
    }
    return mask;
}
// rows at or behind n do not count: bit v is row first + 8 (v / 4) + v % 4
__device__ __forceinline__ uint32_t mx4_rows_below(uint64_t first, uint64_t n) {
    uint32_t mask = 0;
#pragma unroll
    for (int v = 0; v < 16; v++) mask |= first + 8 * (v >> 2) + (v & 3) < n ? 1u << v : 0u;
    return mask;
}
// A panel's survivors for one query tile go straight to the workgroup's own part of their query's list: a counter in LDS, stores that
// nobody waits for.  (Lists that workgroups share want a returning atomic each, which takes microseconds, and where many rows crowd
// around a threshold all wait for the same few: 1.4 M survivors, 580 us.)  taken, list: this lane's query's.  odd: see its callers
template <int M> __device__ __forceinline__ void mx4_survive(const Mx4Scan &P, uint32_t *taken, Mx4Cand *list, const mx4_f16 &d, const mx4_f16 &x, float alpha,
                                                             float beta, uint64_t row0, int half, bool odd) {
    uint32_t rows = 0, mask = 0;   // rows with a survivor in some lane, this lane's: without branches, which would cost more
#pragma unroll
    for (int v = 0; v < 16; v++) {
        const bool hit = mx4_held<M>(d[v], x[v], alpha) >= beta;
        mask |= hit ? 1u << v : 0u;
        rows |= __ballot(hit) ? 1u << v : 0u;
    }
    if (odd) {
        asm volatile("");   // (or the compiler computes it every time)
        rows = 0xFFFFu;
        mask = mx4_survivors<M>(d, x, alpha, beta) & mx4_rows_below(row0 + 4 * half, P.rows.n);
    }
    uint32_t at = mask ? atomicAdd(taken, (uint32_t)__builtin_popcount(mask)) : 0;
    while (rows) {
        const int v = __builtin_ctz(rows);
        rows &= rows - 1;
        if (mask >> v & 1 && at < P.segment) list[at] = Mx4Cand{(uint32_t)row0 + 8 * (v >> 2) + 4 * half + (v & 3), d[v], x[v]};
        at += mask >> v & 1;
    }
}
// PROBE: smaller is nearer, then the upper bound (mx4_bounds, a reciprocal's rounding in the slack) of the smallest.  h is per row
template <int M> __device__ __forceinline__ float mx4_probe_row(float x, bool none) {
    const float inf = __uint_as_float(0x7F800000u), nan = __uint_as_float(0x7FC00000u);
    none |= x > MX4_LONG;
    if constexpr (M == MX4_L2) return none ? inf : (1.f + MX4_EPS) * x * x;
    else if constexpr (M == MX4_IP) return none ? inf : 0.f;
    else return none || x < MX4_SHORT ? nan : __builtin_amdgcn_rcpf(x);
}
template <int M> __device__ __forceinline__ float mx4_probe_value(float d, float x, float h, float c) {   // c = slack |q|
    if constexpr (M == MX4_L2) return __fmaf_rn(2.f * c, x, __fmaf_rn(-2.f, d, h));
    else if constexpr (M == MX4_IP) return __fmaf_rn(c, x, h - d);
    else return -d * h;
}
template <int M> __device__ __forceinline__ float mx4_probe_bound(float best, float y, float ry, float slack) {
    const float inf = __uint_as_float(0x7F800000u);
    float u;
    if constexpr (M == MX4_L2) u = best + __fmaf_rn((1.f + MX4_EPS) * y, y, MX4_TINY);
    else if constexpr (M == MX4_IP) u = 1.f + best, u = u + MX4_STEP * fmaxf(1.f, fabsf(u));
    else u = y < MX4_SHORT ? inf : __fmaf_rn(best, ry, 1.f + slack + MX4_STEP);
    return u == u ? u : inf;
}

// The ring of k_mx4_ring: the workgroup's waves bring every panel into LDS together, a KiB at a time in turn, and `stages` panels
// are under way or in use.  Constants by the chunks of a panel (codes, scales, norms in whole KiB); the stages fill the LDS.
constexpr int mx4_ring_pieces(int nb) { return (4 * nb * 1024 + nb * 256 + 128 + 1023) / 1024; }
constexpr int mx4_ring_stages(int nb) { return nb == 2 ? 15 : (nb == 3 ? 10 : 7); }
constexpr int mx4_ring_bytes(int nb) { return mx4_ring_stages(nb) * mx4_ring_pieces(nb) * 1024; }
constexpr int MX4_RING_WAVES = 4;
// 16 bytes a lane from base + offset to LDS (lds: the wave's first byte), without passing through registers
__device__ __forceinline__ void mx4_to_lds(uint32_t lds, uint32_t offset, uint64_t base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void mx4_wait_loads() {   // until at most N of the wave's memory operations are under way
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// The same two for some of the waves (wave < first), the branches inside: to the compiler they are one straight line, and what
// stands before and behind them may be mixed.
template <int N> __device__ __forceinline__ void mx4_to_lds_first(int wave, uint32_t lds, uint32_t offset, uint64_t base) {
    asm volatile("s_cmp_lt_i32 %0, %1\n\ts_cbranch_scc0 .Lmx4_none_%=\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %4\n.Lmx4_none_%=:"
                 ::"s"(wave), "n"(N), "s"(lds), "v"(offset), "s"(base) : "memory", "scc", "m0");
}
template <int FIRST, int MANY, int FEW> __device__ __forceinline__ void mx4_wait_loads_first(int wave) {   // at most MANY or FEW
    asm volatile("s_cmp_lt_i32 %0, %1\n\ts_cbranch_scc0 .Lmx4_few_%=\n\ts_waitcnt vmcnt(%2)\n\ts_branch .Lmx4_there_%=\n.Lmx4_few_%=:\n\ts_waitcnt vmcnt(%3)\n.Lmx4_there_%=:"
                 ::"s"(wave), "n"(FIRST), "n"(MANY), "n"(FEW) : "memory", "scc");
}
// A wave takes whole panels, one after the other, every wave of the grid in turn.  NB chunks of the panel (256 elements each) are in
// flight: chunk g of the next panel is requested as soon as chunk g of this one has gone into the matrix cores.  Panels of more than
// 4 chunks go through the same four buffers several times.  The queries' operands (SRC) are
//   up to 64 queries          in LDS, read per k-step: the registers hold more of the table in flight instead
//   more, rows to 1024        in registers for scores and bounds of every row: a wave keeps two tiles, and the waves take the same
//                             panels through the CU's cache; LDS would be read 1.5 KiB a tile and step against 32 cycles of matrix
//                             work on each of four SIMDs.  Probe and filter: LDS too, or k_mx4_ring
//   rows beyond the LDS       in global memory, through the caches
// 64 queries x 4M x 768, top-10: filter 255 us, 1.65 GB at 6.5 TB/s.  Scores: 256 x 1M x 1024 335-350 us, 1.57 GB at 4.6 TB/s, two thirds
// of it stores; 33 x 200K x 1000 (4 bits) 37 us, 136 MB; 1 x 100K x 128 5.2 us, where a launch is most of it.
template <int BITS, int QT, int MODE, int NB, int SRC>
static __global__ __launch_bounds__(256, mx4_scan_waves(BITS, QT, MODE, NB, SRC)) void k_mx4_scan(Mx4Scan P) {
    extern __shared__ char shared[];
    constexpr bool SWAP = MODE == MX4_DENSE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    constexpr bool HELD = SRC == MX4_REGS;   // operands in registers
    const uint32_t groups = HELD ? P.groups : 1, group = HELD ? wave % groups : 0;
    const uint32_t block_q0 = blockIdx.y * groups * QT * 32, q0 = block_q0 + group * QT * 32;
    const uint32_t ks = P.rows.ks, kg = HELD ? NB : P.rows.kg;
    const char *tiles = P.tiles + (size_t)(q0 / 32) * P.qtile_bytes;
    const char *lds = SRC == MX4_SHARED ? shared : tiles;
    const uint32_t block_q = groups * QT * 32;
    float *yn_b = reinterpret_cast<float *>(shared + (SRC == MX4_SHARED ? QT * P.qtile_bytes : 0));   // |q|, 1 / |q| of the workgroup's queries (L2 scores: |q|, |q|^2)
    uint32_t *taken = reinterpret_cast<uint32_t *>(yn_b);   // FILTER: candidates of each of them so far
    if constexpr (SRC == MX4_SHARED) {
        const mx4_u4 *src = reinterpret_cast<const mx4_u4 *>(tiles);
        const uint32_t n16 = QT * P.qtile_bytes / 16;
        for (uint32_t i = threadIdx.x; i < n16; i += blockDim.x) reinterpret_cast<mx4_u4 *>(shared)[i] = src[i];
    }
    for (uint32_t i = threadIdx.x; i < block_q; i += blockDim.x) {
        if constexpr (MODE == MX4_FILTER) {
            taken[i] = 0;
        } else {
            const float y = P.qnorm[block_q0 + i];   // (padded to whole tiles)
            yn_b[i] = y;
            yn_b[block_q + i] = MODE == MX4_DENSE && P.metric == MX4_L2 ? (float)P.qsq[block_q0 + i] : 1.f / y;
        }
    }
    __syncthreads();
    const float *yn_s = yn_b + group * QT * 32, *yr_s = yn_s + block_q;
    const uint32_t sc_at = kg * (BITS == 6 ? 4 * 1536 : 4 * 1024);
    Mx4Operand<BITS> op[HELD ? QT * 4 * NB : 1];
    int opsc[HELD ? QT * NB : 1];
    if constexpr (HELD) {
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
    // FILTER: neighbouring panels go to different workgroups, so that rows that crowd together fill no part of a list
    uint32_t w = MODE == MX4_FILTER ? wave * gridDim.x + blockIdx.x : blockIdx.x * abreast + wave / groups;
    if (MODE != MX4_FILTER && w >= n_take) return;
    const auto panel_of = [&](uint32_t i) -> uint64_t { return MODE == MX4_PROBE ? (i * P.every) >> 24 : i; };
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
    uint64_t panel = P.rows.uniform_at(panel_of(min(w, n_take - 1)));
    fetch_norms(panel);
#pragma unroll
    for (int g = 0; g < NB; g++)
        if (g < (int)kg) mx4_fetch<!HELD>(buf[g], panel, g, ks, lane);
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
                for (int q = 0; q < QT; q++) sq[q] = HELD ? opsc[q * NB + j] : reinterpret_cast<const int *>(lds + q * P.qtile_bytes + sc_at + g * 256)[lane];
                const Mx4Chunk &c = buf[j];
                const auto step = [&](auto index) {
                    constexpr int I = decltype(index)::value;
                    const mx4_i8 t{c.a[I][0], c.a[I][1], c.a[I][2], c.a[I][3], 0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < QT; q++) {
                        Mx4Operand<BITS> o;
                        if constexpr (HELD) o = op[q * 4 * NB + 4 * j + I];
                        else o.load(lds + q * P.qtile_bytes, 4 * g + I, kg, lane);
                        acc[q] = mx4_mma<BITS, SWAP, I>(t, o.get(), acc[q], c.sc, sq[q]);
                    }
                };
                step(std::integral_constant<int, 0>{});
                step(std::integral_constant<int, 1>{});
                step(std::integral_constant<int, 2>{});
                step(std::integral_constant<int, 3>{});
                // the buffer's next contents: NB chunks on in this panel, or the chunk of the next panel that it takes
                if (!HELD && g + NB < kg) mx4_fetch<true>(buf[j], panel, g + NB, ks, lane);
                else mx4_fetch<!HELD>(buf[j], next, j, ks, lane);
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
                        if constexpr (M == MX4_L2) s = __fmaf_rn(-2.f, d, r4[j] + c0);
                        else if constexpr (M == MX4_IP) s = 1.f - d;
                        else if constexpr (decltype(divide)::value) s = 1.f - d / xrow / y;
                        else s = 1.f - d * rx * r4[j];
                        if (decltype(whole)::value || (q0 + q * 32 + 8 * i + 4 * half + j < P.nq && row < P.rows.n)) __builtin_nontemporal_store(s, line);
                        line += j < 3 ? P.out_stride : 5 * P.out_stride;
                    }
                }
        };
        const auto filter = [&](auto metric) {
            constexpr int M = decltype(metric)::value;
            float least = xn[0], longest = xn[0];
#pragma unroll
            for (int v = 1; v < 16; v++) {
                least = fminf(least, xn[v]);
                longest = fmaxf(longest, xn[v]);
            }
            const bool odd = tail || __any(longest > MX4_LONG || (M == MX4_COSINE && least < MX4_SHORT));
#pragma unroll
            for (int q = 0; q < QT; q++) {
                float most = mx4_held<M>(acc[q][0], xn[0], alpha[q]);
#pragma unroll
                for (int v = 1; v < 16; v++) most = fmaxf(most, mx4_held<M>(acc[q][v], xn[v], alpha[q]));
                if (!__any(most >= beta[q]) && !odd) continue;
                const uint32_t me = q * 32 + col;
                mx4_survive<M>(P, taken + me, P.cand + ((size_t)(q0 + me) * P.segments + blockIdx.x) * P.segment, acc[q], xn, alpha[q], beta[q], row0, half, odd);
            }
        };
        const auto probe = [&](auto metric) {
            constexpr int M = decltype(metric)::value;
            mx4_f16 h;
#pragma unroll
            for (int v = 0; v < 16; v++) h[v] = mx4_probe_row<M>(xn[v], tail && row_of(v) >= P.rows.n);
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const uint32_t me = q0 + q * 32 + col;
                const float c = P.slack * alpha[q];
                if constexpr (MODE == MX4_PROBE_ROWS) {
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (me < P.nq && row_of(v) < P.rows.n)
                            P.minima[me * P.minima_stride + row_of(v)] = mx4_probe_bound<M>(mx4_probe_value<M>(acc[q][v], xn[v], h[v], c), alpha[q], beta[q], P.slack);
                } else {
                    float best = mx4_probe_value<M>(acc[q][0], xn[0], h[0], c);
#pragma unroll
                    for (int v = 1; v < 16; v++) best = fminf(best, mx4_probe_value<M>(acc[q][v], xn[v], h[v], c));
                    if (me < P.nq) P.minima[me * P.minima_stride + 2 * w + half] = mx4_probe_bound<M>(best, alpha[q], beta[q], P.slack);
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
    if constexpr (MODE == MX4_FILTER) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < block_q && block_q0 + i < P.nq; i += blockDim.x) P.counts[(size_t)(block_q0 + i) * P.segments + blockIdx.x] = taken[i];
    }
}

// The same passes for 65 to 256 queries against rows of at most 1024 elements.  Four waves, QT tiles each, take every panel together; it
// comes through LDS, so that the memory's latency is covered by a ring of panels and not by registers, which hold the operands.  One
// wave a SIMD: the comparisons of the panel before are made between the matrix instructions of this one, whose last chunk covers the
// barrier and the first reads of the next.
// Filter of 1M x 1024 (549 MB): 128 queries, the nearest one 140 us; 256 queries, 1 | 10 | 100 nearest 190 | 210 | 250 us (524 GFLOP at
// 2.8 | 2.5 | 2.1 PFLOP/s): each panel with survivors costs its wave some 800 cycles.  Eight waves of one tile each read the LDS twice
// as often (without survivors 207 us against 160).
template <int BITS, int QT, int MODE, int NB, int M> static __global__ __launch_bounds__(256, 1) void k_mx4_ring(Mx4Scan P) {
    extern __shared__ char shared[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    constexpr int PIECES = mx4_ring_pieces(NB), STAGES = mx4_ring_stages(NB), STAGE = PIECES * 1024;
    constexpr int EACH = PIECES / MX4_RING_WAVES, OVER = PIECES % MX4_RING_WAVES;   // waves below OVER take one piece more
    constexpr uint32_t BLOCK_Q = MX4_RING_WAVES * QT * 32;
    const uint32_t block_q0 = blockIdx.y * BLOCK_Q, q0 = block_q0 + wave * QT * 32, ks = P.rows.ks;
    const char *tiles = P.tiles + (size_t)(q0 / 32) * P.qtile_bytes;
    float *yn_b = reinterpret_cast<float *>(shared + mx4_ring_bytes(NB));      // PROBE: |q|, 1 / |q|
    uint32_t *taken = reinterpret_cast<uint32_t *>(yn_b);                      // FILTER: candidates of each query so far
    for (uint32_t i = threadIdx.x; i < BLOCK_Q; i += 256) {
        if constexpr (MODE == MX4_FILTER) taken[i] = 0;
        else {
            const float y = P.qnorm[block_q0 + i];   // (padded to whole tiles)
            yn_b[i] = y;
            yn_b[BLOCK_Q + i] = 1.f / y;
        }
    }
    __syncthreads();
    Mx4Operand<BITS> op[QT][4 * NB];
    int opsc[QT][NB];
    float alpha[QT], beta[QT];   // FILTER: the threshold; PROBE: |q|, 1 / |q|
#pragma unroll
    for (int q = 0; q < QT; q++) {
        const char *tile = tiles + q * P.qtile_bytes;
#pragma unroll
        for (int s = 0; s < 4 * NB; s++) op[q][s].load(tile, s, NB, lane);
#pragma unroll
        for (int g = 0; g < NB; g++) opsc[q][g] = reinterpret_cast<const int *>(tile + NB * (BITS == 6 ? 4 * 1536 : 4 * 1024) + g * 256)[lane];
        const uint32_t me = q0 + q * 32 + col;
        if constexpr (MODE == MX4_FILTER) {
            const float2 l = me < P.nq ? P.limit[me] : make_float2(0.f, __uint_as_float(0x7F800000u));
            alpha[q] = l.x;
            beta[q] = l.y;
        } else {
            alpha[q] = yn_b[me - block_q0];
            beta[q] = yn_b[BLOCK_Q + me - block_q0];
        }
    }
    const uint32_t n_take = (uint32_t)P.n_take;
    uint32_t w = blockIdx.x;
    if (w >= n_take) return;
    const auto panel_of = [&](uint32_t i) -> uint64_t { return MODE == MX4_PROBE ? (i * P.every) >> 24 : i; };
    uint32_t ahead = w, fill = 0, use = 0;   // the panel to request next, the stage it goes to, the stage in use
    // (past the end the last panel again, so that the count of what is under way stays the same)
    const auto requested = [&]() -> uint64_t { return P.rows.uniform_at(panel_of(min(ahead, n_take - 1))); };
    const auto request = [&](uint64_t from) {
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)shared + fill * STAGE;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const uint32_t offset = (i * MX4_RING_WAVES + wave) * 1024;
            mx4_to_lds(to + offset, min(offset + lane * 16, P.rows.panel - 16), from);
        }
        if constexpr (OVER != 0) {
            const uint32_t offset = (EACH * MX4_RING_WAVES + wave) * 1024;
            mx4_to_lds_first<OVER>(wave, to + offset, min(offset + lane * 16, P.rows.panel - 16), from);
        }
        ahead += gridDim.x;
        fill = fill + 1 == STAGES ? 0 : fill + 1;
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; i++) request(requested());

    struct Panel {
        mx4_f16 acc[QT], x;   // dots, |x|
        uint32_t w;
    };
    const auto row0_of = [&](const Panel &p) { return panel_of(p.w) * 32; };
    // a panel's comparisons, v-th of its rows
    float most[QT], least, longest;
    mx4_f16 h;
    const auto compare = [&](const Panel &p, int v) {
        if constexpr (MODE == MX4_FILTER) {
            if (M == MX4_COSINE) least = v ? fminf(least, p.x[v]) : p.x[0];
            longest = v ? fmaxf(longest, p.x[v]) : p.x[0];
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const float f = mx4_held<M>(p.acc[q][v], p.x[v], alpha[q]);
                most[q] = v ? fmaxf(most[q], f) : f;
            }
        } else {
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const float f = mx4_probe_value<M>(p.acc[q][v], p.x[v], h[v], P.slack * alpha[q]);
                most[q] = v ? fminf(most[q], f) : f;
            }
        }
    };
    const auto conclude = [&](const Panel &p) {
        if constexpr (MODE == MX4_FILTER) {
            const uint64_t row0 = row0_of(p);
            uint64_t any[QT], all = 0;
#pragma unroll
            for (int q = 0; q < QT; q++) all |= any[q] = __ballot(most[q] >= beta[q]);
            bool odd = row0 + 32 > P.rows.n;   // the last panel's padding
            if (__any(longest > MX4_LONG || (M == MX4_COSINE && least < MX4_SHORT))) {
                asm volatile("");   // (or the compiler computes it every time)
                bool some = false;
#pragma unroll
                for (int v = 0; v < 16; v++) some |= mx4_beyond<M>(p.x[v]);
                odd |= __any(some);
            }
            if (all == 0 && !odd) return;
#pragma unroll
            for (int q = 0; q < QT; q++) {
                if (any[q] == 0 && !odd) continue;
                const uint32_t me = wave * QT * 32 + q * 32 + col;
                mx4_survive<M>(P, taken + me, P.cand + ((size_t)(block_q0 + me) * P.segments + blockIdx.x) * P.segment, p.acc[q], p.x, alpha[q], beta[q], row0, half, odd);
            }
        } else {
#pragma unroll
            for (int q = 0; q < QT; q++) {
                const uint32_t me = q0 + q * 32 + col;
                if (me < P.nq) P.minima[me * P.minima_stride + 2 * p.w + half] = mx4_probe_bound<M>(most[q], alpha[q], beta[q], P.slack);
            }
        }
    };
    const auto prepare = [&](Panel &p) {   // PROBE: what is per row
        if constexpr (MODE == MX4_PROBE) {
            const uint64_t row0 = row0_of(p);
#pragma unroll
            for (int v = 0; v < 16; v++) h[v] = mx4_probe_row<M>(p.x[v], row0 + 8 * (v >> 2) + 4 * half + (v & 3) >= P.rows.n);
        }
    };
    Mx4Chunk buf[2];
    const char *stage = shared;
    const auto take = [&](Mx4Chunk &c, int j) {
#pragma unroll
        for (int i = 0; i < 4; i++) c.a[i] = reinterpret_cast<const mx4_i4 *>(stage + min(4u * j + i, ks - 1) * 1024)[lane];
        c.sc = reinterpret_cast<const int *>(stage + ks * 1024 + j * 256)[lane];
    };
    // this wave's part of the next panel is there, with AFTER panels behind it under way; beyond the barrier everybody's is, and
    // nobody reads the panel before this one any more: what comes next goes into its stage
    const auto arrive = [&](auto after) {
        constexpr int AFTER = decltype(after)::value;
        mx4_wait_loads_first<OVER, AFTER *(EACH + 1), AFTER * EACH>(wave);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    arrive(std::integral_constant<int, STAGES - 2>{});
    take(buf[0], 0);
    // one panel: its dots into p, and q's comparisons.  Its first chunk is in buf[FIRST], its last one's matrix instructions cover the
    // wait for the next panel's first
    const auto round = [&](Panel &p, Panel &q, auto parity) {
        constexpr int FIRST = decltype(parity)::value;
        const uint64_t from = requested();
        prepare(q);
        mx4_f4 nrm[4];
#pragma unroll
        for (int i = 0; i < 4; i++) nrm[i] = reinterpret_cast<const mx4_f4 *>(stage + P.rows.panel - 128)[2 * i + half];
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
            for (int v = 0; v < 16; v++) p.acc[t][v] = 0.f;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            Mx4Chunk &c = buf[(FIRST + j) & 1], &next = buf[(FIRST + j + 1) & 1];
            if (j + 1 < NB) {
                take(next, j + 1);
            } else {
                arrive(std::integral_constant<int, STAGES - 3>{});
                request(from);
                use = use + 1 == STAGES ? 0 : use + 1;
                stage = shared + use * STAGE;
                take(next, 0);
            }
            const auto step = [&](auto index) {
                constexpr int I = decltype(index)::value;
                const mx4_i8 t{c.a[I][0], c.a[I][1], c.a[I][2], c.a[I][3], 0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < QT; i++) p.acc[i] = mx4_mma<BITS, false, I>(t, op[i][4 * j + I].get(), p.acc[i], c.sc, opsc[i][j]);
                // 16 rows of the panel before, over 4 NB steps
                const int s = 4 * j + I;
#pragma unroll
                for (int v = s * 16 / (4 * NB); v < (s + 1) * 16 / (4 * NB); v++) compare(q, v);
                __builtin_amdgcn_sched_barrier(0);   // (left to itself the compiler puts them all behind the matrix instructions)
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        }
#pragma unroll
        for (int v = 0; v < 16; v++) p.x[v] = nrm[v >> 2][v & 3];
        p.w = w;
#pragma unroll
        for (int i = 0; i < QT; i++) asm volatile("" : "+a"(p.acc[i]), "+v"(most[i]));   // (... or behind the branches of the rare case)
        conclude(q);
    };
    Panel a, b;   // b: a panel before the first one, without survivors at any threshold
#pragma unroll
    for (int v = 0; v < 16; v++) {
        b.x[v] = 1.f;
#pragma unroll
        for (int q = 0; q < QT; q++) b.acc[q][v] = __uint_as_float(0x7FC00000u);
    }
    b.w = w;   // (PROBE: overwritten with the panel's own result)
    const auto last = [&](Panel &p) {
        prepare(p);
#pragma unroll
        for (int v = 0; v < 16; v++) compare(p, v);
        conclude(p);
    };
    for (;;) {
        round(a, b, std::integral_constant<int, 0>{});
        w += gridDim.x;
        if (w >= n_take) {
            last(a);
            break;
        }
        round(b, a, std::integral_constant<int, NB & 1>{});
        w += gridDim.x;
        if (w >= n_take) {
            last(b);
            break;
        }
    }
    mx4_wait_loads<0>();   // (what is under way writes this workgroup's LDS)
    if constexpr (MODE == MX4_FILTER) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < BLOCK_Q && block_q0 + i < P.nq; i += 256) P.counts[(size_t)(block_q0 + i) * P.segments + blockIdx.x] = taken[i];
    }
}

}  // namespace vsg
