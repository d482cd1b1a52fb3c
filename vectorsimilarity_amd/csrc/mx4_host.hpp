// mx4_host.hpp -- what the MXFP4 translation unit gives the table code in vsgpu.hip.
#pragma once
#include "mx4_common.hpp"

namespace vsg {
struct Mx4Write;
struct Mx4Read;
enum { MX4_SHARED = 0, MX4_GLOBAL = 1, MX4_REGS = 2 };   // where k_mx4_scan has the queries' operands (REGS: in passes that keep every row's result; the others SHARED)
struct Mx4ScanShape {
    int src, cus;
    bool ring;        // the probe and the filter are k_mx4_ring
    uint32_t qt, y;   // query tiles a wave, workgroups side by side (each with groups x qt tiles)
};
// registers of a wave of k_mx4_scan, about: what its operands, sums and panel in flight need
constexpr int mx4_scan_waves(int bits, int qt, int mode, int nb, int src) {
    const int regs = (src == MX4_REGS ? qt * nb * (bits == 6 ? 25 : 17) : qt * 12) + qt * 16 + nb * 17 + (mode == MX4_DENSE ? 60 : 105);
    return regs <= 128 ? 4 : (regs <= 168 ? 3 : (regs <= 256 ? 2 : 1));
}
// ... its workgroups along the table: as many as stay resident; few panels: fewer, so that a wave's start is not most of its work.
// y > 1: workgroups side by side take the same panels, each with its own queries.  They are on one XCD (workgroups are dealt over eight)
// and share its L2, which holds what they read while it is one workgroup a CU; for scores, and where panels are large (400K x 1536,
// 256 queries: scores 285 -> 228 us, top-10 232 -> 224; 300K x 2048 with 4 bits: 266 -> 194, 218 -> 197; but top-10 of
// 400K x 1100 179 -> 203, of 2M x 128 225 -> 329).
inline uint64_t mx4_scan_grid(int bits, int qt, int mode, int nb, int src, size_t lds, uint64_t n_take, uint32_t kg, uint32_t abreast, int cus, uint32_t y) {
    const bool alone = lds + 512 > 160 * 1024 || (src == MX4_SHARED && y > 1 && (mode == MX4_DENSE || kg > 5));
    const uint64_t fit = alone ? 1 : (160 * 1024) / (lds + 512), waves = (uint64_t)mx4_scan_waves(bits, qt, mode, nb, src);
    uint64_t all = (uint64_t)cus * (fit < waves ? fit : waves) / y;
    if (y > 1 && all >= 16) all &= ~(uint64_t)7;
    const uint64_t need = (n_take + abreast - 1) / abreast;
    return all < need ? (all ? all : 1) : need;
}
inline int mx4_scan_chunks(uint32_t kg) { return kg == 1 ? 1 : 4; }   // SHARED: a panel's chunks in flight
inline size_t mx4_scan_lds(int src, uint32_t qt, uint32_t groups, uint32_t qtile_bytes) { return (src == MX4_SHARED ? (size_t)qt * qtile_bytes : 0) + groups * qt * 256; }
int mx4_scan4(hipStream_t s, int mode, const Mx4Scan &P, const Mx4ScanShape &shape);
int mx4_scan6(hipStream_t s, int mode, const Mx4Scan &P, const Mx4ScanShape &shape);
Mx4Rows mx4_rows_of(const void *base, size_t n, size_t dim);
int mx4_launch_write(hipStream_t s, const Mx4Write &W, int type);
int mx4_launch_read(hipStream_t s, const Mx4Read &R, int type, int cus);
int mx4_launch_queries(hipStream_t s, const void *x, int type, size_t stride, size_t nq, const Mx4Rows &R, int bits, uint32_t tiles, char *block,
                       float *norm, double *sq, uint32_t *zero, size_t zero_words);
// the one pass of a top-k over every row, for the statistics: marked by these events, made by this kernel
struct Mx4Pass {
    hipEvent_t begin = nullptr, end = nullptr;
    const char *kernel = "";
};
size_t mx4_topk_bytes(size_t n, size_t dim, size_t nq, size_t k, int bits);
int mx4_topk_batch(hipStream_t s, int device, const Mx4Rows &R, const void *queries, int type, size_t nq, size_t qstride, size_t k, int metric,
                   int bits, int64_t *ids, float *scores, void *ws, size_t ws_bytes, Mx4Pass *pass = nullptr);
}  // namespace vsg

// a vsgpu_table of MXFP4 rows; host pointers, every call ends with its stream drained
struct vsgpu_table;
int mx4_table_store(vsgpu_table *t, const void *vectors, size_t first, size_t n);   // rounds n vectors into rows first ..
int mx4_table_move(vsgpu_table *t, size_t dst, size_t src);
int mx4_table_values(vsgpu_table *t, size_t first, size_t n, float *out);
int mx4_table_scores(vsgpu_table *t, const void *query, const uint32_t *ids, size_t first, size_t n, double *scores);
int mx4_table_topk(vsgpu_table *t, const void *queries, size_t nq, size_t qstride, size_t k, size_t cap, uint32_t *ids, double *scores, uint32_t *counts);
