"""CPU: the refusals of the MXFP4 entries (include/vsgpu.h), and the float64 definition the GPU tests compare with."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch  # noqa: F401  (before the native libraries)

import mx4_ref as ref
from vectorsimilarity_amd import _capi, mx4

ARG, UNSUPPORTED = 3, 4
F32 = _capi.VecSimType_FLOAT32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_panel_bytes():
    """codes of whole steps of 64, scale dwords of whole groups of four steps, 32 norms"""
    for dim, want in ((1, 1024 + 256 + 128), (64, 1024 + 256 + 128), (65, 2048 + 256 + 128), (257, 5 * 1024 + 512 + 128), (768, 412 * 32)):
        assert mx4.panel_bytes(dim) == want
    for dim in (0, -1, 65537):
        with pytest.raises(ValueError):
            mx4.panel_bytes(dim)


def test_entries_refuse_bad_calls_before_they_touch_a_device():
    g = _capi.load_gpu()
    p, odd, none = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 2), C.c_void_p(None)
    write = lambda table=p, capacity=64, dim=64, x=p, kind=F32, m=4, stride=256, slots=none, size=0, first=0: \
        g.vsgpu_mx4_write(0, None, table, capacity, dim, x, kind, m, stride, slots, size, first)
    for rc, call in ((ARG, dict(dim=0)), (ARG, dict(dim=65537)), (ARG, dict(table=none)), (ARG, dict(table=odd)), (ARG, dict(x=none)), (ARG, dict(x=odd)),
                     (ARG, dict(stride=252)), (ARG, dict(stride=258)), (UNSUPPORTED, dict(kind=1)), (UNSUPPORTED, dict(kind=4)), (ARG, dict(m=65)),
                     (ARG, dict(first=61)), (ARG, dict(first=2 ** 63)), (ARG, dict(slots=p, size=2)), (ARG, dict(slots=odd, size=4)), (ARG, dict(m=2 ** 31)),
                     (ARG, dict(capacity=2 ** 32))):
        assert write(**call) == rc, call
    read = lambda table=p, capacity=64, dim=64, first=0, m=4, out=p, kind=F32, stride=256: \
        g.vsgpu_mx4_read(0, None, table, capacity, dim, none, 0, first, m, out, kind, stride)
    for rc, call in ((ARG, dict(out=none)), (ARG, dict(out=odd)), (UNSUPPORTED, dict(kind=5)), (ARG, dict(m=65)), (ARG, dict(first=64)), (ARG, dict(stride=0))):
        assert read(**call) == rc, call
    scores = lambda table=p, n=64, dim=64, q=p, kind=F32, nq=2, stride=256, metric=0, bits=6, out=p, out_stride=64, ws=p, size=1 << 20: \
        g.vsgpu_mx4_scores(0, None, table, n, dim, q, kind, nq, stride, metric, bits, out, out_stride, ws, size)
    for rc, call in ((ARG, dict(metric=3)), (ARG, dict(metric=-1)), (ARG, dict(bits=8)), (ARG, dict(out=none)), (ARG, dict(out_stride=63)), (ARG, dict(ws=none)),
                     (ARG, dict(ws=C.c_void_p((1 << 20) + 16))), (ARG, dict(nq=2 ** 25)), (UNSUPPORTED, dict(kind=1))):
        assert scores(**call) == rc, call
    topk = lambda n=64, k=3, ids=p, best=p, ws=p, size=1 << 30: \
        g.vsgpu_mx4_topk(0, None, p, n, 64, p, F32, 2, 256, k, 0, 6, ids, best, ws, size)
    for rc, call in ((UNSUPPORTED, dict(k=0)), (UNSUPPORTED, dict(k=4097)), (ARG, dict(n=0)), (ARG, dict(ids=none)), (ARG, dict(best=none)), (ARG, dict(ws=none))):
        assert topk(**call) == rc, call
    # nothing to do: fine without a device
    assert write(m=0) == 0 and read(m=0) == 0 and scores(nq=0) == 0 and scores(n=0) == 0


def test_workspace_sizes():
    g = _capi.load_gpu()
    assert g.vsgpu_mx4_scores_workspace(0, 1, 6) == 0 and g.vsgpu_mx4_scores_workspace(64, 1, 5) == 0
    assert g.vsgpu_mx4_topk_workspace(100, 64, 1, 0, 6) == 0 and g.vsgpu_mx4_topk_workspace(100, 64, 1, 4097, 6) == 0
    assert 0 < g.vsgpu_mx4_scores_workspace(768, 64, 6) < 1 << 20
    # batches of 256: as much as the largest of them, the last one may plan a wider probe
    for n, dim, k in ((10 ** 6, 768, 10), (50000, 64, 100), (4000, 300, 7), (300000, 128, 4096)):
        for rest in (1, 40, 65, 130, 255):
            both = max(g.vsgpu_mx4_topk_workspace(n, dim, 256, k, 6), g.vsgpu_mx4_topk_workspace(n, dim, rest, k, 6))
            assert g.vsgpu_mx4_topk_workspace(n, dim, 512 + rest, k, 6) == both
    assert g.vsgpu_mx4_topk_workspace(10 ** 6, 768, 256, 10, 6) == g.vsgpu_mx4_topk_workspace(10 ** 6, 768, 5000, 10, 6)


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(4, 64)
    table = torch.zeros(1, mx4.panel_bytes(64), dtype=torch.uint8)
    for call in (lambda: mx4.write(table, x), lambda: mx4.read(table, 64, n=1), lambda: mx4.scores(table, 4, x, 0), lambda: mx4.topk(table, 4, x, 1, 0),
                 lambda: mx4.empty(-1, 64, "cpu"), lambda: mx4.empty(3, 0, "cpu")):
        with pytest.raises(ValueError):
            call()


def test_the_definition():
    """E2M1 and E2M3 by their tables of values"""
    four = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    six = np.concatenate([np.arange(0, 16) / 8, np.arange(8, 16) / 4, np.arange(8, 16) / 2])
    rng = np.random.default_rng(0)
    for bits, table in ((4, four), (6, six)):
        values = np.concatenate([-table[::-1], table])
        for scale in (1.0, 2.0 ** -130, 2.0 ** 100):
            x = rng.uniform(-8, 8, (200, 32))
            x[:, 0] = 7.9    # the block's scale is one
            got = ref.micro(x * scale, bits) / scale
            best = np.abs(x[..., None] - values).min(-1)
            s = 1.0 if scale >= 2.0 ** -127 else 2.0 ** 3      # 2^-130 lies below the smallest scale, 2^-127
            if s == 1.0:
                assert np.isin(got, values).all()
                np.testing.assert_array_equal(np.abs(got - x), best)
            else:
                assert np.isin(got / s, values).all()
    np.testing.assert_array_equal(ref.micro(np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 4]]), 4), [[0, 1, 1, 2, 2, 4, 4, 4]])
    assert np.isnan(ref.micro(np.array([[1.0] * 31 + [np.inf] + [1.0]]), 6)).tolist() == [[True] * 32 + [False]]


# ---- reading rows: how the kernel divides its work (csrc/mx4_read_plan.h) ---------------------------------------------------------
@pytest.fixture(scope="module")
def read_plan():
    helpers = os.path.join(ROOT, "tests", "helpers")
    csrc = os.path.join(ROOT, "vectorsimilarity_amd", "csrc")
    so, src = os.path.join(helpers, "libmx4_read_plan.so"), os.path.join(helpers, "mx4_read_plan.cpp")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", csrc, "-o", so, src], check=True)
    L = C.CDLL(so)
    L.wrong_rows.restype = C.c_long
    L.wrong_rows.argtypes = [C.c_uint32, C.c_uint32]
    L.pieces.restype = L.rows.restype = C.c_uint32
    L.pieces.argtypes = [C.c_uint32]
    L.rows.argtypes = [C.c_uint64, C.c_uint32, C.c_uint32]
    return L


def test_read_takes_every_piece_of_every_row_once(read_plan):
    """a piece of eight elements goes to row t / pieces of a row: for every row length that a store may have"""
    assert [read_plan.pieces(d) for d in (1, 8, 9, 16, 17, 65536)] == [1, 1, 2, 2, 3, 8192]
    for per_row in range(1, 8193):
        most = max(read_plan.rows(m, per_row, cus) for cus in (1, 256, 304) for m in (1, 2, 255, 256, 257, 100000, 2 ** 31 - 1))
        assert 1 <= most and most * per_row < 1 << 16
        assert read_plan.wrong_rows(per_row, 1 << 16) == 0, per_row
