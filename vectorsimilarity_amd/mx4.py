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
import ctypes as C

import torch   # before the native libraries: the process takes torch's HIP runtime

from . import _capi
from ._capi import VecSimMetric_Cosine, VecSimMetric_IP, VecSimMetric_L2

PANEL_ROWS = 32
_TYPES = {torch.float32: _capi.VecSimType_FLOAT32, torch.float16: _capi.VecSimType_FLOAT16,
          torch.bfloat16: _capi.VecSimType_BFLOAT16}
_ERR_ARG, _ERR_UNSUPPORTED = 3, 4


def _lib():
    first = _capi._gpu is None
    lib = _capi.load_gpu()
    if first:
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64.so" in line}
        if len(runtimes) > 1:
            _capi._gpu = None
            raise RuntimeError("two HIP runtimes in this process (%s): import torch (or vectorsimilarity_amd.mx4) before the "
                               "first index is made" % ", ".join(sorted(runtimes)))
    return lib


def _check(lib, rc):
    if rc == 0:
        return
    message = lib.vsgpu_last_error().decode()
    raise (ValueError if rc in (_ERR_ARG, _ERR_UNSUPPORTED) else RuntimeError)(message)


def panel_bytes(dim):
    """bytes of a panel of 32 rows of `dim` elements (1 .. 65536)"""
    n = _lib().vsgpu_mx4_panel_bytes(int(dim)) if dim > 0 else 0
    if n == 0:
        raise ValueError("mx4: rows of %s elements (1..65536)" % (dim,))
    return n


def empty(capacity, dim, device=None):
    """a store of `capacity` rows (rounded up to whole panels), every row zero"""
    if capacity < 0:
        raise ValueError("mx4: capacity %s" % (capacity,))
    device = torch.device("cuda" if device is None else device)
    return torch.zeros((int(capacity) + PANEL_ROWS - 1) // PANEL_ROWS, panel_bytes(dim), dtype=torch.uint8, device=device)


def _table(table, dim):
    if not isinstance(table, torch.Tensor) or table.dtype != torch.uint8 or table.dim() != 2 or not table.is_cuda:
        raise ValueError("mx4: a store is a uint8 tensor [panels, panel_bytes(dim)] on a GPU")
    if table.shape[1] != panel_bytes(dim) or not table.is_contiguous():
        raise ValueError("mx4: a contiguous store of rows of %d elements has %d bytes a panel, not %s" % (dim, panel_bytes(dim), tuple(table.shape)))
    return table.shape[0] * PANEL_ROWS


def _vectors(x, table, what):
    """(tensor, type, rows, dim, bytes between rows)"""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.dtype not in _TYPES:
        raise ValueError("mx4: %s must be a 2-D tensor of float32, float16 or bfloat16" % what)
    if x.device != table.device:
        raise ValueError("mx4: %s on %s, the store on %s" % (what, x.device, table.device))
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("mx4: %s require a gradient; rounding to codes has none (detach them)" % what)
    m, dim = x.shape
    if dim < 1:
        raise ValueError("mx4: %s without elements" % what)
    if (dim > 1 and x.stride(1) != 1) or (m > 1 and x.stride(0) < dim):
        x = x.contiguous()
    return x, _TYPES[x.dtype], m, dim, (x.stride(0) if m > 1 else dim) * x.element_size()


def _slots(slots, table, m=None):
    """(contiguous tensor or None, bytes each, count)"""
    if slots is None:
        return None, 0, m
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("mx4: slots must be a 1-D tensor of int32 or int64")
    if slots.device != table.device:
        raise ValueError("mx4: slots on %s, the store on %s" % (slots.device, table.device))
    if m is not None and slots.numel() != m:
        raise ValueError("mx4: %d slots for %d vectors" % (slots.numel(), m))
    return slots.contiguous(), slots.element_size(), slots.numel()


def _where(table):
    return table.device.index, C.c_void_p(torch.cuda.current_stream(table.device).cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr() if t is not None and t.numel() else None)


def write(table, vectors, slots=None, first=0):
    """Rounds `vectors` [m, dim] into the store, in place: into slots[i] (a negative slot is padding and skipped; of several
    vectors with one slot the last stays), or into rows first .. first + m - 1.  Slots are not checked on the host: one at
    or beyond the store's end is skipped too."""
    lib = _lib()
    if not isinstance(table, torch.Tensor) or not isinstance(vectors, torch.Tensor) or vectors.dim() != 2:
        raise ValueError("mx4: write(store, vectors [m, dim])")
    capacity = _table(table, vectors.shape[1])
    x, kind, m, dim, stride = _vectors(vectors, table, "vectors")
    slots, size, _ = _slots(slots, table, m)
    if slots is not None and first != 0:
        raise ValueError("mx4: slots and first together")
    if first < 0:
        raise ValueError("mx4: first row %d" % first)
    device, stream = _where(table)
    _check(lib, lib.vsgpu_mx4_write(device, stream, _ptr(table), capacity, dim, _ptr(x), kind, m, stride, _ptr(slots) if m else None, size, int(first)))


def read(table, dim, slots=None, dtype=torch.float32, n=None):
    """The values of the rows in `slots` (a negative one reads zeros, one beyond the store NaN), or of the first n rows, as
    a new tensor [m, dim] of float32, bfloat16 (both exact) or float16 (rounded)."""
    lib = _lib()
    capacity = _table(table, dim)
    if dtype not in _TYPES:
        raise ValueError("mx4: rows are read as float32, float16 or bfloat16, not %s" % dtype)
    if (slots is None) == (n is None):
        raise ValueError("mx4: read either slots or the first n rows")
    if n is not None and not 0 <= n <= capacity:
        raise ValueError("mx4: %d rows of %d" % (n, capacity))
    slots, size, m = _slots(slots, table, n)
    out = torch.empty(m, dim, dtype=dtype, device=table.device)
    device, stream = _where(table)
    if m:
        _check(lib, lib.vsgpu_mx4_read(device, stream, _ptr(table), capacity, dim, _ptr(slots), size, 0, m, _ptr(out), _TYPES[dtype],
                                       dim * out.element_size()))
    return out


def _query(table, n, queries, metric, query_bits):
    if not isinstance(queries, torch.Tensor) or queries.dim() != 2:
        raise ValueError("mx4: queries must be a 2-D tensor")
    capacity = _table(table, queries.shape[1])
    if not 0 <= n <= capacity:
        raise ValueError("mx4: %s rows of %d" % (n, capacity))
    if metric not in (VecSimMetric_L2, VecSimMetric_IP, VecSimMetric_Cosine):
        raise ValueError("mx4: metric %s" % (metric,))
    if query_bits not in (4, 6):
        raise ValueError("mx4: queries of %s bits (4 or 6)" % (query_bits,))
    return _vectors(queries, table, "queries")


def scores(table, n, queries, metric, query_bits=6):
    """fp32 scores [nq, n] of every query [nq, dim] against rows 0 .. n - 1 of the store."""
    lib = _lib()
    q, kind, nq, dim, stride = _query(table, n, queries, metric, query_bits)
    out = torch.empty(nq, n, dtype=torch.float32, device=table.device)
    if nq and n:
        size = lib.vsgpu_mx4_scores_workspace(dim, nq, query_bits)
        ws = torch.empty(size, dtype=torch.uint8, device=table.device)
        device, stream = _where(table)
        _check(lib, lib.vsgpu_mx4_scores(device, stream, _ptr(table), n, dim, _ptr(q), kind, nq, stride, metric, query_bits, _ptr(out), n, _ptr(ws), size))
    return out


def topk(table, n, queries, k, metric, query_bits=6):
    """(ids int64 [nq, k], scores float32 [nq, k]): per query the k (1 .. 4096) rows of smallest score among rows 0 .. n - 1,
    ascending by (score, row), padded with -1.  Scores are computed in 64 bits and rounded once, so the order is the
    definition's; rows that score NaN are not returned."""
    lib = _lib()
    q, kind, nq, dim, stride = _query(table, n, queries, metric, query_bits)
    if not 1 <= k <= 4096:
        raise ValueError("mx4: k = %s (1..4096)" % (k,))
    ids = torch.empty(nq, k, dtype=torch.int64, device=table.device)
    best = torch.empty(nq, k, dtype=torch.float32, device=table.device)
    if n == 0:
        return ids.fill_(-1), best.fill_(-1.0)
    if nq:
        size = lib.vsgpu_mx4_topk_workspace(n, dim, nq, k, query_bits)
        ws = torch.empty(size, dtype=torch.uint8, device=table.device)
        device, stream = _where(table)
        _check(lib, lib.vsgpu_mx4_topk(device, stream, _ptr(table), n, dim, _ptr(q), kind, nq, stride, k, metric, query_bits, _ptr(ids), _ptr(best),
                                       _ptr(ws), size))
    return ids, best
