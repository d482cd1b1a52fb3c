// vsgpu_mx4.hip -- the MXFP4 row store of include/vsgpu.h: checks, plans and launches around mx4_kernels.hpp (gfx950).
//
// Nothing here allocates, waits or keeps state: every call works on the caller's device memory and stream (a captured stream
// included), its scratch is the caller's workspace.
#include "vsgpu_internal.hpp"
#include "mx4_host.hpp"
#include "mx4_kernels.hpp"

using namespace vsg;

namespace {

// the calling thread's device, put back on every way out
struct DeviceScope {
    int before = -1;
    bool ok = false;
    explicit DeviceScope(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        ok = before == device || hipSetDevice(device) == hipSuccess;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

constexpr size_t MAX_DIM = 65536, MAX_ROWS = 0xFFFFFFE0ull, QUERY_BATCH = 256;
constexpr int PLAN_CUS = 256;   // what sizes a workspace: it does not depend on the device that will be given it
constexpr size_t LDS_BUDGET = 160 * 1024 - 1024;   // for the queries' operands

int elem_size(int type) { return type == VSGPU_F32 ? 4 : (type == VSGPU_F16 || type == VSGPU_BF16 ? 2 : 0); }

int compute_units(int device) {
    static std::atomic<int> seen[64];
    if (device < 0 || device >= 64) return 256;
    int n = seen[device].load(std::memory_order_relaxed);
    if (!n) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) n = 256;
        seen[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

bool bad_shape(size_t n, size_t dim) { return dim == 0 || dim > MAX_DIM || n > MAX_ROWS; }

}  // namespace

namespace vsg {

Mx4Rows mx4_rows_of(const void *base, size_t n, size_t dim) {
    Mx4Rows r{};
    r.base = static_cast<char *>(const_cast<void *>(base));
    r.dim = (uint32_t)dim;
    r.ks = mx4_steps(r.dim);
    r.kg = mx4_groups(r.dim);
    r.panel = mx4_panel(r.dim);
    r.n = n;
    return r;
}

// how a batch of at most QUERY_BATCH queries runs
struct Plan {
    uint32_t tiles;              // 32-query tiles, padded to what the workgroups take
    uint32_t groups;             // waves that share a panel
    Mx4ScanShape shape;
    uint32_t qtile_bytes;
    uint64_t panels, take;       // panels of the table / of the probe
    bool by_row;                 // the probe keeps every row's bound, not one of 16 rows
    bool dense;                  // ... and those bounds are the candidate list: no threshold, no second pass
    bool all;                    // ... or there are no bounds: every row is scored exactly, no pass at all
    uint64_t minima;             // floats per query
    uint32_t segments, segment;  // parts of a candidate list and what each holds
    uint32_t shares, room;       // workgroups per query that k_mx4_finish takes, candidates each may leave
    uint32_t slices;             // ... that k_mx4_again may need
};
static Plan plan_scan(size_t dim, size_t nq, int bits, int cus) {
    Plan p{};
    const uint32_t nt = (uint32_t)((nq + 31) / 32);
    p.qtile_bytes = mx4_qtile((uint32_t)dim, bits);
    p.shape.cus = cus;
    p.groups = 1;
    if (nt > 2 && dim <= 1024) {
        // Scores and bounds of every row: operands in registers.  The probe and the filter: the ring where a panel's matrix work
        // outweighs its barrier and comparisons, queries in LDS and panels by wave below that (2M rows, top-10, 128 queries: 256
        // elements 150 us against the ring's 202, 512 221 : 228, 1024 406 : 285; 256 queries: 256 elements 260 : 267, 512 402 : 310)
        const uint32_t kg = mx4_groups((uint32_t)dim);
        p.shape.src = MX4_REGS;
        p.shape.ring = kg > (nt <= 4 ? 2u : 1u);
        p.shape.qt = p.shape.ring && nt <= 4 ? 1 : 2;
        p.groups = (nt + 1) / 2;   // (REGS: two tiles a wave)
        p.shape.y = (nt + 1) / 2;
        p.tiles = p.shape.ring ? 4 * p.shape.qt : 2 * p.shape.y;
        return p;
    } else if (p.qtile_bytes + 256 > LDS_BUDGET) {
        p.shape.src = MX4_GLOBAL;
        p.shape.qt = 1;
    } else {
        p.shape.src = MX4_SHARED;
        p.shape.qt = nt >= 2 && 2 * (p.qtile_bytes + 256) <= LDS_BUDGET ? 2 : 1;
    }
    p.shape.y = (nt + p.shape.qt - 1) / p.shape.qt;
    p.tiles = p.shape.y * p.shape.qt;
    return p;
}
static Plan plan_topk(size_t n, size_t dim, size_t nq, size_t k, int bits, int cus) {
    Plan p = plan_scan(dim, nq, bits, cus);
    p.panels = (n + 31) / 32;
    // Small tables for their k: the probe covers every row.  One bound per 16 rows would put the threshold far above the k-th score.
    p.dense = n <= MX4_LISTED;
    p.by_row = p.dense || n < 64 * k;
    // Very small ones: two rounds of exact scores (mx4_row_lanes) cost less than the pass that would save some of them (whole calls,
    // 64 rows of 1024: 16.6 -> 13.7 us, 16 queries 18.6 -> 13.9; 512 rows of 128: 16.6 -> 13.7; four rounds, 128 rows of 4096: 27 -> 35)
    p.all = n * mx4_row_lanes(mx4_steps((uint32_t)dim)) <= 2048;
    uint64_t expected;   // candidates
    if (p.by_row) {
        p.take = p.panels;
        p.minima = p.all ? 0 : n;
        expected = k;
    } else {
        // a probe of n / div rows leaves about k div candidates per query: div balances its bytes against what they cost.  Whole
        // calls at div 8 | 16 | 32 | 64: 64 queries x 4M x 768, k 10: 356 | 324 | 315 | 312 us, k 100: 381 | 357 | 350 | 357;
        // 256 x 1M x 1024, k 10: 255 | 250 | 264 | 279, k 100: 313 | 338 | 362 | 406
        const double div = std::min(64.0, std::max(8.0, std::sqrt((double)n / ((double)nq * (double)k))));
        p.take = std::min<uint64_t>(p.panels, std::max<uint64_t>((uint64_t)((double)p.panels / div), 4 * k));
        p.minima = 2 * p.take;
        expected = k * ((p.panels + p.take - 1) / p.take);
    }
    // A segment for each workgroup of the filter.  Panels are dealt over them in turn, so that only rows crowded around the threshold
    // fill one: twice its share and two panels
    if (p.shape.ring) p.segments = (uint32_t)std::min<uint64_t>(PLAN_CUS, p.panels);
    else p.segments = (uint32_t)mx4_scan_grid(bits, p.shape.qt, MX4_FILTER, p.shape.src == MX4_GLOBAL ? 4 : mx4_scan_chunks(mx4_groups((uint32_t)dim)),
                                              p.shape.src == MX4_GLOBAL ? MX4_GLOBAL : MX4_SHARED,
                                              mx4_scan_lds(p.shape.src == MX4_GLOBAL ? MX4_GLOBAL : MX4_SHARED, p.shape.qt, 1, p.qtile_bytes), p.panels, mx4_groups((uint32_t)dim), 4, PLAN_CUS, p.shape.y);
    p.segment = p.dense ? 0 : (uint32_t)std::min<uint64_t>((p.panels + p.segments - 1) / p.segments * 32, expected * 2 / p.segments + 72);
    // k rows or more are scored exactly, a workgroup 1024 / lanes of them at once: several of these rounds are worth a second workgroup
    const size_t rounds = k * mx4_row_lanes(mx4_steps((uint32_t)dim)) / 1024;
    p.shares = (uint32_t)std::max<size_t>(1, std::min<size_t>({MX4_SHARES, rounds / 2, (size_t)PLAN_CUS / nq}));
    p.room = (uint32_t)std::max<size_t>(k, 1024);
    p.slices = k <= 128 ? 32 : 8;
    return p;
}

struct Layout {   // of the workspace
    size_t at = 0;
    char *base = nullptr;
    template <typename T> T *take(size_t count) {
        char *p = base + at;
        at = (at + count * sizeof(T) + 255) & ~(size_t)255;
        return reinterpret_cast<T *>(p);
    }
};
struct QueryBlock {
    char *tiles;
    float *norm;
    double *sq;
};
static QueryBlock take_queries(Layout &L, const Plan &p) {
    QueryBlock b;
    b.tiles = L.take<char>((size_t)p.tiles * p.qtile_bytes);
    b.norm = L.take<float>((size_t)p.tiles * 32);
    b.sq = L.take<double>((size_t)p.tiles * 32);
    return b;
}
struct TopkBlock {
    QueryBlock q;
    float2 *limit;
    float *tau;
    uint32_t *done, *counts, *share_n, *again, *ticket;
    uint64_t *again_limit, *share;
    float *minima;
    Mx4Cand *cand;
    uint64_t *part;
};
static TopkBlock take_topk(Layout &L, const Plan &p, size_t nq, size_t k) {
    TopkBlock b;
    b.q = take_queries(L, p);
    b.limit = L.take<float2>(nq);
    b.tau = L.take<float>(nq);
    b.done = L.take<uint32_t>(nq);
    b.counts = L.take<uint32_t>(p.dense ? 0 : nq * (size_t)p.segments);
    b.share_n = L.take<uint32_t>(p.shares > 1 ? nq * p.shares : 0);
    b.share = L.take<uint64_t>(p.shares > 1 ? nq * p.shares * (size_t)p.room : 0);
    b.again = L.take<uint32_t>(nq);
    b.ticket = L.take<uint32_t>(nq);
    b.again_limit = L.take<uint64_t>(nq);
    b.minima = L.take<float>(nq * p.minima);
    b.cand = L.take<Mx4Cand>(nq * (size_t)p.segment * p.segments);
    b.part = L.take<uint64_t>(nq * p.slices * k);
    return b;
}

template <int BITS> static int launch_queries(hipStream_t s, const Mx4Queries &Q, uint32_t tiles, int type) {
    const dim3 g(tiles), b(64 * std::min(16u, Q.kg * 4));
#define MX4_CASE(T)                                                                                       \
    hipLaunchKernelGGL((k_mx4_queries<T, BITS>), g, b, 0, s, Q);
    if (type == VSGPU_F32) { MX4_CASE(MX4_F32) }
    else if (type == VSGPU_F16) { MX4_CASE(MX4_F16) }
    else { MX4_CASE(MX4_BF16) }
#undef MX4_CASE
    HIPCHK(hipGetLastError());
    return VSGPU_OK;
}
int mx4_launch_queries(hipStream_t s, const void *x, int type, size_t stride, size_t nq, const Mx4Rows &R, int bits, uint32_t tiles,
                       char *block, float *norm, double *sq, uint32_t *zero, size_t zero_words) {
    Mx4Queries Q{static_cast<const char *>(x), stride, (uint32_t)nq, R.dim, R.ks, R.kg, block, norm, sq, zero, (uint32_t)zero_words};
    return bits == 6 ? launch_queries<6>(s, Q, tiles, type) : launch_queries<4>(s, Q, tiles, type);
}

static int launch_scan(hipStream_t s, int mode, const Mx4Scan &P, const Plan &p, int bits) {
    return bits == 6 ? mx4_scan6(s, mode, P, p.shape) : mx4_scan4(s, mode, P, p.shape);
}

int mx4_launch_write(hipStream_t s, const Mx4Write &W0, int type) {
    Mx4Write W = W0;
    if (W.m == 0) return VSGPU_OK;
    if (W.slots && W.m > 4096) {   // (up to there every workgroup looks for later owners of its slots itself)
        const dim3 g((unsigned)((W.m + 255) / 256));
        hipLaunchKernelGGL(k_mx4_claim, g, dim3(256), 0, s, W, 0);
        hipLaunchKernelGGL(k_mx4_claim, g, dim3(256), 0, s, W, 1);
        W.claimed = 1;
    }
    // (waves beyond the rows' steps only help in that search)
    const unsigned search = W.slots && !W.claimed ? (unsigned)std::min<uint64_t>(16, (W.m + 127) / 128) : 1;
    const dim3 g((unsigned)((W.m + 31) / 32)), b(64 * std::max(search, std::min(16u, W.rows.ks)));
#define MX4_CASE(T)                                                                \
    hipLaunchKernelGGL((k_mx4_write<T>), g, b, 0, s, W);
    if (type == VSGPU_F32) { MX4_CASE(MX4_F32) }
    else if (type == VSGPU_F16) { MX4_CASE(MX4_F16) }
    else { MX4_CASE(MX4_BF16) }
#undef MX4_CASE
    HIPCHK(hipGetLastError());
    return VSGPU_OK;
}
int mx4_launch_read(hipStream_t s, const Mx4Read &R, int type, int cus) {
    if (R.m == 0) return VSGPU_OK;
    const uint32_t per_row = mx4_read_pieces(R.rows.dim), rows = mx4_read_rows(R.m, per_row, (uint32_t)cus), reciprocal = mx4_reciprocal(per_row);
    const dim3 g((unsigned)((R.m + rows - 1) / rows)), b(256);
#define MX4_CASE(T)                                                                                                           \
    hipLaunchKernelGGL((k_mx4_read<T>), g, b, 0, s, R, rows, per_row, reciprocal);
    if (type == VSGPU_F32) { MX4_CASE(MX4_F32) }
    else if (type == VSGPU_F16) { MX4_CASE(MX4_F16) }
    else { MX4_CASE(MX4_BF16) }
#undef MX4_CASE
    HIPCHK(hipGetLastError());
    return VSGPU_OK;
}

size_t mx4_topk_bytes(size_t n, size_t dim, size_t nq, size_t k, int bits) {
    const auto bytes = [&](size_t m) {
        Layout L;
        take_topk(L, plan_topk(n, dim, m, k, bits, PLAN_CUS), m, k);
        return L.at;
    };
    // (a last batch of fewer queries may plan a wider probe)
    return nq > QUERY_BATCH && nq % QUERY_BATCH ? std::max(bytes(QUERY_BATCH), bytes(nq % QUERY_BATCH)) : bytes(std::min(nq, QUERY_BATCH));
}

// queries of one batch -> ids / scores [nq][k] on the device
int mx4_topk_batch(hipStream_t s, int device, const Mx4Rows &R, const void *queries, int type, size_t nq, size_t qstride, size_t k, int metric,
                   int bits, int64_t *ids, float *scores, void *ws, size_t ws_bytes, Mx4Pass *pass) {
    const int cus = compute_units(device);
    const Plan p = plan_topk(R.n, R.dim, nq, k, bits, cus);
    Layout L;
    L.base = static_cast<char *>(ws);
    const TopkBlock b = take_topk(L, p, nq, k);
    if (L.at > ws_bytes) return fail(VSGPU_ERR_ARG, "workspace of %zu bytes, %zu needed", ws_bytes, L.at);
    int rc = mx4_launch_queries(s, queries, type, qstride, nq, R, bits, p.tiles, b.q.tiles, b.q.norm, b.q.sq, b.done, nq);
    if (rc) return rc;
    Mx4Scan P{};
    P.rows = R;
    P.tiles = b.q.tiles;
    P.qtile_bytes = p.qtile_bytes;
    P.groups = p.groups;
    P.nq = (uint32_t)nq;
    P.metric = (uint32_t)metric;
    P.qnorm = b.q.norm;
    P.n_take = p.take;
    P.every = (p.panels << 24) / p.take;   // (2^27 panels at most)
    P.minima = b.minima;
    P.minima_stride = p.minima;
    P.limit = b.limit;
    P.counts = b.counts;
    P.cand = b.cand;
    P.segments = p.segments;
    P.segment = p.segment;
    P.slack = mx4_slack(R.ks);
    // the pass over every row: the filter, the probe of a small table, the exact scores of a very small one
    if (pass) pass->kernel = p.all ? "k_mx4_finish" : (!p.dense && p.shape.ring ? "k_mx4_ring" : "k_mx4_scan");
    const auto mark = [&](hipEvent_t event) { return event ? hipEventRecord(event, s) : hipSuccess; };
    const hipEvent_t begin = pass ? pass->begin : nullptr, end = pass ? pass->end : nullptr;
    if (p.dense) HIPCHK(mark(begin));
    if (!p.all) rc = launch_scan(s, p.by_row ? MX4_PROBE_ROWS : MX4_PROBE, P, p, bits);
    if (rc) return rc;
    if (!p.dense) {
        const Mx4Threshold T{b.minima, p.minima, p.minima, (uint32_t)k, (uint32_t)metric, b.q.norm, b.q.sq, b.limit, b.tau, P.slack};
        hipLaunchKernelGGL(k_mx4_threshold, dim3((unsigned)nq), dim3(1024), 0, s, T);
        HIPCHK(hipGetLastError());
        P.n_take = p.panels;
        HIPCHK(mark(begin));
        rc = launch_scan(s, MX4_FILTER, P, p, bits);
        if (rc) return rc;
    }
    if (!p.all) HIPCHK(mark(end));
    Mx4Select S{};
    S.E = Mx4Exact{R, b.q.tiles, p.qtile_bytes, (uint32_t)metric, b.q.sq};
    S.nq = (uint32_t)nq;
    S.k = (uint32_t)k;
    S.segments = p.segments;
    S.segment = p.segment;
    S.shares = p.shares;
    S.room = p.room;
    S.share = b.share;
    S.share_n = b.share_n;
    S.done = b.done;
    S.counts = b.counts;
    S.cand = b.cand;
    S.again = b.again;
    S.again_limit = b.again_limit;
    S.ids = ids;
    S.scores = scores;
    S.slices = p.slices;
    S.part = b.part;
    S.ticket = b.ticket;
    S.minima = p.all ? nullptr : b.minima;
    S.qnorm = b.q.norm;
    S.tau = b.tau;
    S.slack = P.slack;
    const dim3 fg((unsigned)nq, p.shares), ag(p.slices, (unsigned)std::max<size_t>(1, std::min<size_t>(nq, (size_t)cus / p.slices)));
    if (p.dense) {
        if (bits == 6) hipLaunchKernelGGL((k_mx4_finish<6, true>), fg, dim3(MX4_FINISH), 0, s, S);
        else hipLaunchKernelGGL((k_mx4_finish<4, true>), fg, dim3(MX4_FINISH), 0, s, S);
    } else if (bits == 6) {
        hipLaunchKernelGGL((k_mx4_finish<6, false>), fg, dim3(MX4_FINISH), 0, s, S);
        hipLaunchKernelGGL((k_mx4_again<6>), ag, dim3(512), 0, s, S);
    } else {
        hipLaunchKernelGGL((k_mx4_finish<4, false>), fg, dim3(MX4_FINISH), 0, s, S);
        hipLaunchKernelGGL((k_mx4_again<4>), ag, dim3(512), 0, s, S);
    }
    HIPCHK(hipGetLastError());
    if (p.all) HIPCHK(mark(end));
    return VSGPU_OK;
}

int mx4_scores_batch(hipStream_t s, int device, const Mx4Rows &R, const void *queries, int type, size_t nq, size_t qstride, int metric, int bits,
                     float *out, size_t out_stride, void *ws, size_t ws_bytes) {
    const Plan p = plan_scan(R.dim, nq, bits, compute_units(device));
    Layout L;
    L.base = static_cast<char *>(ws);
    const QueryBlock b = take_queries(L, p);
    if (L.at > ws_bytes) return fail(VSGPU_ERR_ARG, "workspace of %zu bytes, %zu needed", ws_bytes, L.at);
    const int rc = mx4_launch_queries(s, queries, type, qstride, nq, R, bits, p.tiles, b.tiles, b.norm, b.sq, nullptr, 0);
    if (rc) return rc;
    Mx4Scan P{};
    P.rows = R;
    P.tiles = b.tiles;
    P.qtile_bytes = p.qtile_bytes;
    P.groups = p.groups;
    P.nq = (uint32_t)nq;
    P.metric = (uint32_t)metric;
    P.qnorm = b.norm;
    P.qsq = b.sq;
    P.n_take = (R.n + 31) / 32;
    P.out = out;
    P.out_stride = out_stride;
    P.slack = mx4_slack(R.ks);
    return launch_scan(s, MX4_DENSE, P, p, bits);
}

}  // namespace vsg

// ---------------------------------------------------------------------------------------------------------------- tables
static Mx4Rows rows_of(const vsgpu_table *t) {
    Mx4Rows r = mx4_rows_of(nullptr, t->n, t->dim);
    r.slabs = t->d_slabs;
    r.shift = t->slab_shift - 5;
    return r;
}
static size_t in_bytes(const vsgpu_table *t) { return t->dim * (size_t)elem_size(t->mx4_in); }
constexpr size_t STAGE_BYTES = (size_t)64 << 20;

int mx4_table_store(vsgpu_table *t, const void *vectors, size_t first, size_t n) {
    vsgpu_ctx *c = t->ctx;
    const size_t row = in_bytes(t), piece = std::max<size_t>(1, STAGE_BYTES / row);
    for (size_t i = 0; i < n; i += piece) {
        const size_t m = std::min(piece, n - i);
        const int rc = ensure(c, c->dense, m * row);
        if (rc) return rc;
        HIPCHK(hipMemcpyAsync(c->dense.p, static_cast<const char *>(vectors) + i * row, m * row, hipMemcpyHostToDevice, c->stream));
        Mx4Write W{};
        W.rows = rows_of(t);
        W.x = static_cast<const char *>(c->dense.p);
        W.stride = row;
        W.m = m;
        W.first = first + i;
        W.capacity = t->slabs.size() << t->slab_shift;
        const int rl = mx4_launch_write(c->stream, W, t->mx4_in);
        if (rl) return rl;
        HIPCHK(hipStreamSynchronize(c->stream));   // (the caller's buffer is borrowed; reader lanes query on their own streams)
    }
    return VSGPU_OK;
}
int mx4_table_move(vsgpu_table *t, size_t dst, size_t src) {
    hipLaunchKernelGGL(k_mx4_move, dim3(1), dim3(256), 0, t->ctx->stream, rows_of(t), (uint64_t)dst, (uint64_t)src);
    HIPCHK(hipGetLastError());
    HIPCHK(hipStreamSynchronize(t->ctx->stream));
    return VSGPU_OK;
}
int mx4_table_values(vsgpu_table *t, size_t first, size_t n, float *out) {
    vsgpu_ctx *c = t->ctx;
    const size_t row = t->dim * 4, piece = std::max<size_t>(1, STAGE_BYTES / row);
    for (size_t i = 0; i < n; i += piece) {
        const size_t m = std::min(piece, n - i);
        const int rc = ensure(c, c->dense, m * row);
        if (rc) return rc;
        Mx4Read R{};
        R.rows = rows_of(t);
        R.out = static_cast<char *>(c->dense.p);
        R.stride = row;
        R.m = m;
        R.first = first + i;
        R.capacity = t->n;
        const int rl = mx4_launch_read(c->stream, R, VSGPU_F32, c->n_cu);
        if (rl) return rl;
        HIPCHK(hipMemcpyAsync(out + i * t->dim, c->dense.p, m * row, hipMemcpyDeviceToHost, c->stream));
        HIPCHK(hipStreamSynchronize(c->stream));
    }
    return VSGPU_OK;
}
// the host's queries, packed on the device (ctx->qfrag)
static int upload_queries(vsgpu_table *t, const void *queries, size_t nq, size_t qstride) {
    vsgpu_ctx *c = t->ctx;
    const size_t row = in_bytes(t), bytes = (nq * row + 15) & ~(size_t)15;
    int rc = ensure(c, c->qfrag, bytes);
    if (!rc) rc = ensure_pin_up(c, bytes);
    if (rc) return rc;
    for (size_t q = 0; q < nq; q++) memcpy(static_cast<char *>(c->pin_up) + q * row, static_cast<const char *>(queries) + q * qstride, row);
    return upload_block(c, c->qfrag.p, c->pin_up, bytes);
}
int mx4_table_scores(vsgpu_table *t, const void *query, const uint32_t *ids, size_t first, size_t n, double *scores) {
    vsgpu_ctx *c = t->ctx;
    int rc = upload_queries(t, query, 1, 0);
    if (rc) return rc;
    const Mx4Rows R = rows_of(t);
    const Plan p = plan_scan(t->dim, 1, t->mx4_bits, c->n_cu);
    Layout size;
    take_queries(size, p);
    rc = ensure(c, c->qfrag2, size.at);
    if (rc) return rc;
    Layout L;
    L.base = static_cast<char *>(c->qfrag2.p);
    const QueryBlock b = take_queries(L, p);
    rc = mx4_launch_queries(c->stream, c->qfrag.p, t->mx4_in, in_bytes(t), 1, R, t->mx4_bits, p.tiles, b.tiles, b.norm, b.sq, nullptr, 0);
    if (rc) return rc;
    const Mx4Exact E{R, b.tiles, p.qtile_bytes, (uint32_t)t->metric, b.sq};
    const size_t piece = (size_t)1 << 24;
    for (size_t i = 0; i < n; i += piece) {
        const size_t m = std::min(piece, n - i);
        rc = ensure(c, c->dense, m * 4);
        if (!rc) rc = ensure_pinned(c, m * 4);
        if (!rc && ids) rc = ensure(c, c->ids, m * 4);
        if (rc) return rc;
        if (ids) HIPCHK(hipMemcpyAsync(c->ids.p, ids + i, m * 4, hipMemcpyHostToDevice, c->stream));
        const uint32_t *d_ids = ids ? static_cast<const uint32_t *>(c->ids.p) : nullptr;
        const dim3 g((unsigned)std::min<size_t>((m + 15) / 16, (size_t)c->n_cu * 16));
        if (t->mx4_bits == 6) hipLaunchKernelGGL((k_mx4_exact_rows<6>), g, dim3(256), 0, c->stream, E, d_ids, (uint64_t)(first + i), (uint64_t)m, (float *)c->dense.p);
        else hipLaunchKernelGGL((k_mx4_exact_rows<4>), g, dim3(256), 0, c->stream, E, d_ids, (uint64_t)(first + i), (uint64_t)m, (float *)c->dense.p);
        HIPCHK(hipGetLastError());
        HIPCHK(hipMemcpyAsync(c->pinned, c->dense.p, m * 4, hipMemcpyDeviceToHost, c->stream));
        HIPCHK(hipStreamSynchronize(c->stream));
        const float *src = static_cast<const float *>(c->pinned);
        for (size_t j = 0; j < m; j++) scores[i + j] = (double)src[j];
    }
    return VSGPU_OK;
}
// vsgpu_topk's contract: every row at or below the k-th smallest score, ascending by id.  The device returns the best `take` >= k rows;
// only when all of them are at or below the k-th score may there be more.
int mx4_table_topk(vsgpu_table *t, const void *queries, size_t nq, size_t qstride, size_t k, size_t cap, uint32_t *ids, double *scores, uint32_t *counts) {
    vsgpu_ctx *c = t->ctx;
    const size_t n = t->n, kk = std::min(k, n), take = std::min(std::min(cap, n), (size_t)MX4_KMAX);
    if (take < kk) {   // k beyond the device's lists: the caller scores every row
        for (size_t q = 0; q < nq; q++) counts[q] = VSGPU_COUNT_OVERFLOW;
        return VSGPU_OK;
    }
    const Mx4Rows R = rows_of(t);
    const size_t row = in_bytes(t), batch = std::min(nq, QUERY_BATCH), ws = mx4_topk_bytes(n, t->dim, nq, take, t->mx4_bits);
    const size_t ids_bytes = (batch * take * 8 + 255) & ~(size_t)255, out_bytes = ids_bytes + batch * take * 4;
    int rc = ensure(c, c->dense, ws);
    if (!rc) rc = ensure(c, c->sel, out_bytes);
    if (!rc) rc = ensure_pinned(c, out_bytes);
    if (rc) return rc;
    for (size_t q0 = 0; q0 < nq; q0 += QUERY_BATCH) {
        const size_t m = std::min(QUERY_BATCH, nq - q0);
        ScanChainGuard chain(t);
        rc = upload_queries(t, static_cast<const char *>(queries) + q0 * qstride, m, qstride);
        if (rc) return rc;
        chain.before_scan();
        Mx4Pass pass;
        if (c->opt_events & 1) pass.begin = c->ev_a, pass.end = c->ev_b;
        rc = mx4_topk_batch(c->stream, c->device, R, c->qfrag.p, t->mx4_in, m, row, take, t->metric, t->mx4_bits, static_cast<int64_t *>(c->sel.p),
                            reinterpret_cast<float *>(static_cast<char *>(c->sel.p) + ids_bytes), c->dense.p, c->dense.cap, &pass);
        if (rc) return rc;
        chain.submitted();
        HIPCHK(hipMemcpyAsync(c->pinned, c->sel.p, out_bytes, hipMemcpyDeviceToHost, c->stream));
        HIPCHK(hipStreamSynchronize(c->stream));
        if (c->poll && c->poll(c->poll_user)) return VSGPU_ERR_TIMEOUT;
        account_scan(c, t, n, 1, pass.kernel);
        const int64_t *rid = static_cast<const int64_t *>(c->pinned);
        const float *rsc = reinterpret_cast<const float *>(static_cast<const char *>(c->pinned) + ids_bytes);
        std::vector<std::pair<uint32_t, double>> hits;
        for (size_t q = 0; q < m; q++) {
            hits.clear();
            for (size_t i = 0; i < take && rid[q * take + i] >= 0; i++) hits.emplace_back((uint32_t)rid[q * take + i], (double)rsc[q * take + i]);
            c->stats.candidates += hits.size();
            size_t keep = hits.size();
            if (hits.size() > kk) {
                const double T = hits[kk - 1].second;
                keep = kk;
                while (keep < hits.size() && hits[keep].second <= T) keep++;
            }
            if (keep == take && take < n && keep > 0 && hits[keep - 1].second <= hits[std::min(kk, keep) - 1].second) {
                counts[q0 + q] = VSGPU_COUNT_OVERFLOW;   // ties may go on behind the list
                continue;
            }
            hits.resize(keep);
            std::sort(hits.begin(), hits.end());
            counts[q0 + q] = (uint32_t)keep;
            for (size_t i = 0; i < keep; i++) {
                ids[(q0 + q) * cap + i] = hits[i].first;
                scores[(q0 + q) * cap + i] = hits[i].second;
            }
        }
    }
    return VSGPU_OK;
}

// ---------------------------------------------------------------------------------------------------------------- the C entries
static int check_table(const void *table, size_t rows, size_t dim, const char *what) {
    if (bad_shape(rows, dim)) return fail(VSGPU_ERR_ARG, "%s: %zu rows of %zu elements (1..%zu elements, at most %zu rows)", what, rows, dim, MAX_DIM, MAX_ROWS);
    if (rows && (!table || ((uintptr_t)table & 15))) return fail(VSGPU_ERR_ARG, "%s: the table must be 16-byte aligned device memory", what);
    return VSGPU_OK;
}
static int check_device(int device) {
    const int n = vsgpu_device_count();
    if (n <= 0) return fail(VSGPU_ERR_NO_DEVICE, "no HIP device visible: the gfx950 kernels are the only compute path");
    if (device < 0 || device >= n) return fail(VSGPU_ERR_ARG, "device %d out of range (0..%d)", device, n - 1);
    return VSGPU_OK;
}
static int check_vectors(const void *x, int type, size_t m, size_t stride, size_t dim, const char *what) {
    const size_t es = (size_t)elem_size(type);
    if (!es) return fail(VSGPU_ERR_UNSUPPORTED, "%s: vectors of type %d (fp32, fp16 and bf16 only)", what, type);
    if (m && (!x || ((uintptr_t)x & (es - 1)) || (stride & (es - 1)) || (m > 1 && stride < dim * es)))
        return fail(VSGPU_ERR_ARG, "%s: vectors must be aligned to their elements, rows at least %zu bytes apart (stride %zu)", what, dim * es, stride);
    return VSGPU_OK;
}
static int check_queries(size_t nq, int metric, int bits) {
    if (metric < VSGPU_L2 || metric > VSGPU_COSINE) return fail(VSGPU_ERR_ARG, "metric %d", metric);
    if (bits != 4 && bits != 6) return fail(VSGPU_ERR_ARG, "queries of %d bits (4 or 6)", bits);
    if (nq > ((size_t)1 << 24)) return fail(VSGPU_ERR_ARG, "%zu queries in one call", nq);
    return VSGPU_OK;
}
static int check_slots(const void *slots, int slot_bytes, size_t first, size_t m, size_t capacity, const char *what) {
    if (m > 0x7FFFFFFFull) return fail(VSGPU_ERR_ARG, "%s: %zu vectors in one call", what, m);
    if (slots ? (slot_bytes != 4 && slot_bytes != 8) || ((uintptr_t)slots & (slot_bytes - 1)) : first > capacity || m > capacity - first)
        return fail(VSGPU_ERR_ARG, "%s: rows %zu..%zu of %zu, or slots that are not aligned 4- or 8-byte integers", what, first, first + m, capacity);
    return VSGPU_OK;
}

extern "C" size_t vsgpu_mx4_panel_bytes(size_t dim) { return dim == 0 || dim > MAX_DIM ? 0 : mx4_panel((uint32_t)dim); }

extern "C" int vsgpu_mx4_write(int device, void *stream, void *table, size_t capacity, size_t dim, const void *vectors, int type, size_t m,
                               size_t stride, const void *slots, int slot_bytes, size_t first) {
    int rc = check_table(table, capacity, dim, "mx4_write");
    if (!rc) rc = check_vectors(vectors, type, m, stride, dim, "mx4_write");
    if (!rc) rc = check_slots(slots, slot_bytes, first, m, capacity, "mx4_write");
    if (rc || m == 0 || capacity == 0) return rc;
    if ((rc = check_device(device))) return rc;
    DeviceScope scope(device);
    if (!scope.ok) return fail(VSGPU_ERR_HIP, "hipSetDevice(%d) failed", device);
    Mx4Write W{};
    W.rows = mx4_rows_of(table, capacity, dim);
    W.x = static_cast<const char *>(vectors);
    W.stride = stride;
    W.m = m;
    W.slots = slots;
    W.slots64 = slot_bytes == 8;
    W.first = first;
    W.capacity = capacity;
    return mx4_launch_write(static_cast<hipStream_t>(stream), W, type);
}

extern "C" int vsgpu_mx4_read(int device, void *stream, const void *table, size_t capacity, size_t dim, const void *slots, int slot_bytes, size_t first,
                              size_t m, void *out, int type, size_t stride) {
    int rc = check_table(table, capacity, dim, "mx4_read");
    if (!rc) rc = check_vectors(out, type, m, stride, dim, "mx4_read");
    if (!rc) rc = check_slots(slots, slot_bytes, first, m, capacity, "mx4_read");
    if (rc || m == 0) return rc;
    if ((rc = check_device(device))) return rc;
    DeviceScope scope(device);
    if (!scope.ok) return fail(VSGPU_ERR_HIP, "hipSetDevice(%d) failed", device);
    Mx4Read R{};
    R.rows = mx4_rows_of(table, capacity, dim);
    R.out = static_cast<char *>(out);
    R.stride = stride;
    R.m = m;
    R.slots = slots;
    R.slots64 = slot_bytes == 8;
    R.first = first;
    R.capacity = capacity;
    return mx4_launch_read(static_cast<hipStream_t>(stream), R, type, compute_units(device));
}

extern "C" size_t vsgpu_mx4_scores_workspace(size_t dim, size_t nq, int bits) {
    if (bad_shape(0, dim) || (bits != 4 && bits != 6) || nq == 0) return 0;
    Layout L;
    take_queries(L, plan_scan(dim, std::min(nq, QUERY_BATCH), bits, PLAN_CUS));
    return L.at;
}
extern "C" int vsgpu_mx4_scores(int device, void *stream, const void *table, size_t n, size_t dim, const void *queries, int type, size_t nq,
                                size_t qstride, int metric, int bits, float *scores, size_t scores_stride, void *workspace, size_t workspace_bytes) {
    int rc = check_table(table, n, dim, "mx4_scores");
    if (!rc) rc = check_vectors(queries, type, nq, qstride, dim, "mx4_scores");
    if (!rc) rc = check_queries(nq, metric, bits);
    if (rc || nq == 0 || n == 0) return rc;
    if (!scores || (nq > 1 && scores_stride < n) || !workspace || ((uintptr_t)workspace & 255))
        return fail(VSGPU_ERR_ARG, "mx4_scores: no output, a stride below %zu, or a workspace that is not 256-byte aligned", n);
    if ((rc = check_device(device))) return rc;
    DeviceScope scope(device);
    if (!scope.ok) return fail(VSGPU_ERR_HIP, "hipSetDevice(%d) failed", device);
    const Mx4Rows R = mx4_rows_of(table, n, dim);
    for (size_t q = 0; q < nq; q += QUERY_BATCH) {
        rc = mx4_scores_batch(static_cast<hipStream_t>(stream), device, R, static_cast<const char *>(queries) + q * qstride, type,
                              std::min(QUERY_BATCH, nq - q), qstride, metric, bits, scores + q * scores_stride, scores_stride, workspace, workspace_bytes);
        if (rc) return rc;
    }
    return VSGPU_OK;
}

extern "C" size_t vsgpu_mx4_topk_workspace(size_t n, size_t dim, size_t nq, size_t k, int bits) {
    if (bad_shape(n, dim) || (bits != 4 && bits != 6) || k == 0 || k > MX4_KMAX || nq == 0) return 0;
    return mx4_topk_bytes(n, dim, nq, k, bits);
}
extern "C" int vsgpu_mx4_topk(int device, void *stream, const void *table, size_t n, size_t dim, const void *queries, int type, size_t nq, size_t qstride,
                              size_t k, int metric, int bits, int64_t *ids, float *scores, void *workspace, size_t workspace_bytes) {
    int rc = check_table(table, n, dim, "mx4_topk");
    if (!rc) rc = check_vectors(queries, type, nq, qstride, dim, "mx4_topk");
    if (!rc) rc = check_queries(nq, metric, bits);
    if (rc) return rc;
    if (k == 0 || k > MX4_KMAX) return fail(VSGPU_ERR_UNSUPPORTED, "mx4_topk: k = %zu (1..%u)", k, MX4_KMAX);
    if (nq == 0) return VSGPU_OK;
    if (n == 0) return fail(VSGPU_ERR_ARG, "mx4_topk: an empty table");
    if (!ids || !scores || !workspace || ((uintptr_t)workspace & 255))
        return fail(VSGPU_ERR_ARG, "mx4_topk: no output, or a workspace that is not 256-byte aligned");
    if ((rc = check_device(device))) return rc;
    DeviceScope scope(device);
    if (!scope.ok) return fail(VSGPU_ERR_HIP, "hipSetDevice(%d) failed", device);
    const Mx4Rows R = mx4_rows_of(table, n, dim);
    for (size_t q = 0; q < nq; q += QUERY_BATCH) {
        rc = mx4_topk_batch(static_cast<hipStream_t>(stream), device, R, static_cast<const char *>(queries) + q * qstride, type,
                            std::min(QUERY_BATCH, nq - q), qstride, k, metric, bits, ids + q * k, scores + q * k, workspace, workspace_bytes);
        if (rc) return rc;
    }
    return VSGPU_OK;
}
