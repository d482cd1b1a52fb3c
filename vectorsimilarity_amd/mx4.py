"""Row stores in the OCP microscaling format MXFP4, on torch tensors: rows are rounded to 4 bits as they are written, read
back, scored against queries, and searched for the k best (include/vsgpu.h: vsgpu_mx4_*).

    store = mx4.empty(100_000, 768, "cuda")
    mx4.write(store, embeddings)                        # or write(store, embeddings, slots=...)
    ids, scores = mx4.topk(store, 100_000, queries, 10, VecSim.VecSimMetric_Cosine)
    rows = mx4.read(store, 768, ids[0], torch.bfloat16)

A store is a uint8 tensor [panels, panel_bytes(dim)], 32 rows a panel: 412 bytes a row of 768 elements.  Every 32 elements
share a power of two, elements are E2M1 codes; queries are rounded to 6 bits an element (MXFP6 E2M3) or to 4, and scores
are the metrics between the rounded vectors (nothing is normalised first).  VecSim.MX4Index is the same store behind the
index API: labels, deletes, batch iterators.

Calls enqueue on torch's current stream of the store's device, whatever the current device is, and can be captured into a
graph.  Tensors must live on the store's device; a tensor made on another stream needs the usual wait and record_stream.
"""
import functools

import torch   # before the native libraries: the process takes torch's HIP runtime

from . import _capi
from ._capi import VecSimMetric_Cosine, VecSimMetric_IP, VecSimMetric_L2

PANEL_ROWS = 32
_TYPES = {torch.float32: _capi.VecSimType_FLOAT32, torch.float16: _capi.VecSimType_FLOAT16,
          torch.bfloat16: _capi.VecSimType_BFLOAT16}
_METRICS = (VecSimMetric_L2, VecSimMetric_IP, VecSimMetric_Cosine)
_ERR_ARG, _ERR_UNSUPPORTED = 3, 4
_lib = None
# torch.cuda.current_stream(device).cuda_stream, a microsecond sooner
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _load():
    global _lib
    lib = _capi.load_gpu()
    with open("/proc/self/maps") as f:
        runtimes = {line.split()[-1] for line in f if "libamdhip64.so" in line}
    if len(runtimes) > 1:
        raise RuntimeError("two HIP runtimes in this process (%s): import torch (or vectorsimilarity_amd.mx4) before the "
                           "first index is made" % ", ".join(sorted(runtimes)))
    _lib = lib
    return lib


def _raise(rc):
    message = _lib.vsgpu_last_error().decode()
    raise (ValueError if rc in (_ERR_ARG, _ERR_UNSUPPORTED) else RuntimeError)(message)


@functools.lru_cache(maxsize=None)
def panel_bytes(dim):
    """bytes of a panel of 32 rows of `dim` elements (1 .. 65536)"""
    n = (_lib or _load()).vsgpu_mx4_panel_bytes(int(dim)) if dim > 0 else 0
    if n == 0:
        raise ValueError("mx4: rows of %s elements (1..65536)" % (dim,))
    return n


@functools.lru_cache(maxsize=4096)
def _scores_bytes(dim, nq, bits):
    return (_lib or _load()).vsgpu_mx4_scores_workspace(dim, nq, bits)


@functools.lru_cache(maxsize=4096)
def _topk_bytes(n, dim, nq, k, bits):
    return (_lib or _load()).vsgpu_mx4_topk_workspace(n, dim, nq, k, bits)


def empty(capacity, dim, device=None):
    """a store of `capacity` rows (rounded up to whole panels), every row zero"""
    if capacity < 0:
        raise ValueError("mx4: capacity %s" % (capacity,))
    device = torch.device("cuda" if device is None else device)
    return torch.zeros((int(capacity) + PANEL_ROWS - 1) // PANEL_ROWS, panel_bytes(dim), dtype=torch.uint8, device=device)


def _capacity(table, dim):
    """rows a store of rows of `dim` elements holds"""
    if not isinstance(table, torch.Tensor) or table.dtype != torch.uint8 or table.dim() != 2 or not table.is_cuda:
        raise ValueError("mx4: a store is a uint8 tensor [panels, panel_bytes(dim)] on a GPU")
    panels, size = table.shape
    if size != panel_bytes(dim) or not table.is_contiguous():
        raise ValueError("mx4: a contiguous store of rows of %d elements has %d bytes a panel, not %s" % (dim, panel_bytes(dim), tuple(table.shape)))
    return panels * PANEL_ROWS


def _vectors(x, table, what):
    """(tensor, type, rows, bytes between rows) of a 2-D tensor"""
    kind = _TYPES.get(x.dtype)
    if kind is None:
        raise ValueError("mx4: %s must be float32, float16 or bfloat16, not %s" % (what, x.dtype))
    if x.device != table.device:
        raise ValueError("mx4: %s on %s, the store on %s" % (what, x.device, table.device))
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("mx4: %s require a gradient; rounding to codes has none (detach them)" % what)
    m, dim = x.shape
    between, inner = x.stride()
    if (dim > 1 and inner != 1) or (m > 1 and between < dim):
        x = x.contiguous()
        between = dim
    return x, kind, m, (between if m > 1 else dim) * x.element_size()


def _slots(slots, table):
    """(contiguous tensor, bytes each)"""
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("mx4: slots must be a 1-D tensor of int32 or int64")
    if slots.device != table.device:
        raise ValueError("mx4: slots on %s, the store on %s" % (slots.device, table.device))
    return slots.contiguous(), slots.element_size()


def _two_d(x, what):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("mx4: %s must be a 2-D tensor" % what)
    return x.shape[1]


def write(table, vectors, slots=None, first=0):
    """Rounds `vectors` [m, dim] into the store, in place: into slots[i] (a negative slot is padding and skipped; of several
    vectors with one slot the last stays), or into rows first .. first + m - 1.  Slots are not checked on the host: one at
    or beyond the store's end is skipped too."""
    lib = _lib or _load()
    dim = _two_d(vectors, "vectors")
    capacity = _capacity(table, dim)
    x, kind, m, stride = _vectors(vectors, table, "vectors")
    where, size = None, 0
    if slots is not None:
        slots, size = _slots(slots, table)
        if slots.numel() != m:
            raise ValueError("mx4: %d slots for %d vectors" % (slots.numel(), m))
        if first != 0:
            raise ValueError("mx4: slots and first together")
        where = slots.data_ptr()
    if first < 0:
        raise ValueError("mx4: first row %d" % first)
    if m == 0:
        return
    device = table.device.index
    rc = lib.vsgpu_mx4_write(device, _stream(device), table.data_ptr(), capacity, dim, x.data_ptr(), kind, m, stride,
                             where, size, first)
    if rc:
        _raise(rc)


def read(table, dim, slots=None, dtype=torch.float32, n=None):
    """The values of the rows in `slots` (a negative one reads zeros, one beyond the store NaN), or of the first n rows, as
    a new tensor [m, dim] of float32, bfloat16 (both exact) or float16 (rounded)."""
    lib = _lib or _load()
    capacity = _capacity(table, dim)
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError("mx4: rows are read as float32, float16 or bfloat16, not %s" % dtype)
    if (slots is None) == (n is None):
        raise ValueError("mx4: read either slots or the first n rows")
    where, size = None, 0
    if slots is None:
        if not 0 <= n <= capacity:
            raise ValueError("mx4: %d rows of %d" % (n, capacity))
        m = int(n)
    else:
        slots, size = _slots(slots, table)
        where, m = slots.data_ptr(), slots.numel()
    out = torch.empty((m, dim), dtype=dtype, device=table.device)
    if m:
        device = table.device.index
        rc = lib.vsgpu_mx4_read(device, _stream(device), table.data_ptr(), capacity, dim, where, size, 0, m,
                                out.data_ptr(), kind, dim * out.element_size())
        if rc:
            _raise(rc)
    return out


def _query(table, n, queries, metric, query_bits):
    dim = _two_d(queries, "queries")
    capacity = _capacity(table, dim)
    if not 0 <= n <= capacity:
        raise ValueError("mx4: %s rows of %d" % (n, capacity))
    if metric not in _METRICS:
        raise ValueError("mx4: metric %s" % (metric,))
    if query_bits not in (4, 6):
        raise ValueError("mx4: queries of %s bits (4 or 6)" % (query_bits,))
    return (dim, *_vectors(queries, table, "queries"))


def scores(table, n, queries, metric, query_bits=6):
    """fp32 scores [nq, n] of every query [nq, dim] against rows 0 .. n - 1 of the store.  Dots are fp32 sums: Cosine scores have
    few digits where |q| |x| is below 2^-120, vectors longer than 2^62 may score infinite or NaN (topk has neither limit)."""
    lib = _lib or _load()
    dim, q, kind, nq, stride = _query(table, n, queries, metric, query_bits)
    out = torch.empty((nq, n), dtype=torch.float32, device=table.device)
    if nq and n:
        size = _scores_bytes(dim, nq, query_bits)
        ws = torch.empty(size, dtype=torch.uint8, device=table.device)
        device = table.device.index
        rc = lib.vsgpu_mx4_scores(device, _stream(device), table.data_ptr(), n, dim, q.data_ptr(), kind, nq, stride,
                                  metric, query_bits, out.data_ptr(), n, ws.data_ptr(), size)
        if rc:
            _raise(rc)
    return out


def topk(table, n, queries, k, metric, query_bits=6):
    """(ids int64 [nq, k], scores float32 [nq, k]): per query the k (1 .. 4096) rows of smallest score among rows 0 .. n - 1,
    ascending by (score, row), padded with -1.  Scores are computed in 64 bits and rounded once, so the order is the
    definition's; rows that score NaN are not returned."""
    lib = _lib or _load()
    dim, q, kind, nq, stride = _query(table, n, queries, metric, query_bits)
    if not 1 <= k <= 4096:
        raise ValueError("mx4: k = %s (1..4096)" % (k,))
    ids = torch.empty((nq, k), dtype=torch.int64, device=table.device)
    best = torch.empty((nq, k), dtype=torch.float32, device=table.device)
    if n == 0:
        return ids.fill_(-1), best.fill_(-1.0)
    if nq:
        size = _topk_bytes(n, dim, nq, k, query_bits)
        ws = torch.empty(size, dtype=torch.uint8, device=table.device)
        device = table.device.index
        rc = lib.vsgpu_mx4_topk(device, _stream(device), table.data_ptr(), n, dim, q.data_ptr(), kind, nq, stride, k,
                                metric, query_bits, ids.data_ptr(), best.data_ptr(), ws.data_ptr(), size)
        if rc:
            _raise(rc)
    return ids, best
