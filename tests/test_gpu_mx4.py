"""GPU: the MXFP4 row store (vectorsimilarity_amd/mx4.py) against the format's definition in float64 (mx4_ref.py)."""
import numpy as np
import pytest
import torch

import mx4_ref as ref
from vectorsimilarity_amd import mx4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
METRICS = [ref.L2, ref.IP, ref.COSINE]


def vectors(m, dim, seed, dtype=torch.float32):
    """values over a few powers of two, exact in dtype"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, dim, generator=g) * torch.exp(0.7 * torch.randn(dim, generator=g)) / dim ** 0.5
    return x.to(dtype)


def store_of(x, capacity=None):
    t = mx4.empty(x.shape[0] if capacity is None else capacity, x.shape[1], DEV)
    mx4.write(t, x.to(DEV))
    return t


def same(a, b):
    """equal values, NaN at the same places"""
    a, b = a.double().cpu().numpy(), np.asarray(b, dtype=np.float64)
    assert a.shape == b.shape
    np.testing.assert_array_equal(a, b)


# ---- write and read -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,dim", [(1, 1), (1, 768), (3, 31), (32, 32), (33, 33), (64, 64), (65, 65), (7, 127), (100, 300), (257, 1000),
                                   (40, 1024), (5, 4097), (2, 20001)])
def test_rows_come_back_rounded(m, dim, dtype):
    x = vectors(m, dim, m * 7 + dim, dtype)
    got = mx4.read(store_of(x), dim, n=m)
    same(got, ref.micro(x.double().numpy(), 4))
    # bf16 holds every value; fp16 is the rounding of the exact value
    same(mx4.read(store_of(x), dim, n=m, dtype=torch.bfloat16), got.double().cpu().numpy())
    same(mx4.read(store_of(x), dim, n=m, dtype=torch.float16), got.half().double().cpu().numpy())


def test_every_tie_and_border():
    """all multiples of 1/64 up to 8 beside a largest element that fixes the scale, at several scales"""
    v = torch.arange(-512, 513) / 64.0
    rows = []
    for e in (-120, -20, -1, 0, 1, 30, 120):
        for a in range(0, len(v), 31):
            piece = torch.zeros(32)
            piece[:len(v[a:a + 31])] = v[a:a + 31]
            piece[31] = 7.5
            rows.append(piece.double() * 2.0 ** e)
    x = torch.stack(rows)
    assert torch.equal(x.float().double(), x)
    same(mx4.read(store_of(x.float()), 32, n=len(x)), ref.micro(x.numpy(), 4))


def test_extreme_and_special_values():
    big, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    rows = torch.zeros(12, 40)
    rows[1, :4] = torch.tensor([big, -big, big / 2, big / 16])
    rows[2, :4] = torch.tensor([tiny, -tiny, 2.0 ** -126, 2.0 ** -127])
    rows[3, 0] = tiny
    rows[4, 3] = float("inf")
    rows[5, 35] = float("-inf")
    rows[6, 7] = float("nan")
    rows[7, :32] = -0.0
    rows[8, :8] = torch.tensor([2.0 ** -128, 2.0 ** -129, 1.5 * 2.0 ** -128, 2.0 ** -127, 2.0 ** -126, 2.0 ** -125, 0, -2.0 ** -128])
    rows[9] = 1e-30
    rows[10, 39] = 5
    rows[11, :3] = torch.tensor([float("nan"), float("inf"), 1.0])
    got = mx4.read(store_of(rows), 40, n=12)
    same(got, ref.micro(rows.double().numpy(), 4))
    assert torch.isnan(got[4, :32]).all() and not torch.isnan(got[4, 32:]).any()
    same(mx4.read(store_of(rows), 40, n=12, dtype=torch.bfloat16), got.double().cpu().numpy())


@pytest.mark.parametrize("slot_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("m", [1, 50, 4096, 5000])
def test_slots_padding_and_the_last_of_equal_slots(m, slot_type):
    dim, capacity = 70, 6000
    g = torch.Generator().manual_seed(m)
    x = vectors(m, dim, m + 1)
    slots = torch.randint(0, max(2, m // 2), (m,), generator=g, dtype=slot_type) * 3
    slots[torch.rand(m, generator=g) < 0.1] = -1
    if m > 3:
        slots[2] = capacity + 500    # beyond the store: skipped
        slots[3] = torch.iinfo(slot_type).max
    before = vectors(capacity, dim, 5)
    table = store_of(before)
    mx4.write(table, x.to(DEV), slots.to(DEV))
    want = ref.micro(before.double().numpy(), 4)
    rounded = ref.micro(x.double().numpy(), 4)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < capacity:
            want[s] = rounded[i]
    same(mx4.read(table, dim, n=capacity), want)
    # norms belong to the rows that stayed
    s = mx4.scores(table, capacity, torch.zeros(1, dim, device=DEV), ref.L2)[0].cpu().numpy()
    np.testing.assert_allclose(s, (want ** 2).sum(1), rtol=2.0 ** -22, atol=0)


def test_read_by_slots():
    x = vectors(500, 96, 3)
    table = store_of(x)
    slots = torch.tensor([499, 0, -1, 33, 33, 5000, -7, 250], device=DEV)
    want = ref.micro(x.double().numpy(), 4)
    got = mx4.read(table, 96, slots).double().cpu().numpy()
    for i, s in enumerate(slots.tolist()):
        want_row = np.zeros(96) if s < 0 else (np.full(96, np.nan) if s >= 512 else want[s])
        np.testing.assert_array_equal(got[i], want_row)
    assert mx4.read(table, 96, slots[:0]).shape == (0, 96)


def test_first_and_rows_beside():
    table = store_of(vectors(100, 50, 1))
    old = mx4.read(table, 50, n=128).clone()
    x = vectors(10, 50, 2)
    mx4.write(table, x.to(DEV), first=45)
    new = mx4.read(table, 50, n=128)
    same(new[45:55], ref.micro(x.double().numpy(), 4))
    assert torch.equal(new[:45], old[:45]) and torch.equal(new[55:], old[55:])
    mx4.write(table, x[:0].to(DEV), first=3)
    mx4.write(table, x.to(DEV), slots=torch.full((10,), -1, device=DEV))
    assert torch.equal(mx4.read(table, 50, n=128), new)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """rows of a wider matrix, from odd offsets, every second row, transposed"""
    wide = vectors(41, 333, 9, dtype).to(DEV)
    for x in (wide[:, 1:300], wide[:, 8:296], wide[::2, 3:131], wide.T[:, :40], wide[:1, 5:], wide[5:6].expand(3, -1)):
        table = mx4.empty(x.shape[0], x.shape[1], DEV)
        mx4.write(table, x)
        same(mx4.read(table, x.shape[1], n=x.shape[0]), ref.micro(x.double().cpu().numpy(), 4))
        q = x[:3]
        got = mx4.scores(table, x.shape[0], q, ref.IP, 4)
        assert torch.equal(got, mx4.scores(table, x.shape[0], q.contiguous().clone(), ref.IP, 4))


# ---- scores ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("nq,n,dim", [(1, 1, 1), (1, 33, 64), (2, 31, 65), (5, 1000, 128), (33, 257, 300), (64, 100, 768), (65, 999, 1000),
                                      (130, 64, 1024), (300, 40, 200), (3, 70, 4096), (40, 50, 6500), (2, 35, 9001)])
def test_scores(nq, n, dim, bits, metric):
    dtype = DTYPES[(nq + n + dim) % 3]
    x, q = vectors(n, dim, 1, dtype), vectors(nq, dim, 2, dtype)
    values = ref.micro(x.double().numpy(), 4)
    got = mx4.scores(store_of(x), n, q.to(DEV), metric, bits).double().cpu().numpy()
    want = ref.scores(q.double().numpy(), values, metric, bits)
    assert got.shape == (nq, n)
    assert (np.abs(got - want) <= ref.bound(q.double().numpy(), values, metric, bits)).all()


def test_scores_of_part_of_a_store_and_of_rows_that_are_not_numbers():
    x = vectors(200, 100, 4)
    x[17, 50] = float("nan")
    x[18] = 0
    q = vectors(3, 100, 5)
    q[1, 3] = float("inf")
    values = ref.micro(x.double().numpy(), 4)
    for metric in METRICS:
        for n in (19, 97, 200):
            got = mx4.scores(store_of(x), n, q.to(DEV), metric).double().cpu().numpy()
            want = ref.scores(q.double().numpy(), values[:n], metric, 6)
            np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
            ok = ~np.isnan(want)
            assert (np.abs(got - want)[ok] <= ref.bound(q.double().numpy(), values[:n], metric, 6)[ok]).all()


# ---- the k best -----------------------------------------------------------------------------------------------------------------
def check_topk(x, q, k, metric, bits, table=None, n=None):
    n = x.shape[0] if n is None else n
    table = store_of(x) if table is None else table
    values = ref.micro(x.double().numpy(), 4)[:n]
    ids, best = mx4.topk(table, n, q.to(DEV), k, metric, bits)
    want_ids, want = ref.topk(q.double().numpy(), values, k, metric, bits)
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    np.testing.assert_array_equal(best.cpu().numpy(), want)


@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("nq,n,dim,k", [(1, 1, 1, 1), (1, 5, 3, 10), (2, 33, 64, 33), (3, 2000, 100, 1), (1, 3000, 128, 10), (33, 5000, 300, 10),
                                        (70, 4000, 768, 5), (130, 3000, 64, 100), (5, 20000, 96, 1000), (2, 9000, 40, 4096), (9, 700, 6500, 7),
                                        (300, 2500, 32, 3)])
def test_topk(nq, n, dim, k, bits, metric):
    dtype = DTYPES[(nq + n + dim) % 3]
    check_topk(vectors(n, dim, 1, dtype), vectors(nq, dim, 2, dtype), k, metric, bits)


@pytest.mark.parametrize("metric", METRICS)
def test_topk_probed_table(metric):
    """a table large enough for the sampled probe (n >= 64 k)"""
    x, q = vectors(60000, 64, 1), vectors(40, 64, 2)
    table = store_of(x)
    for k in (1, 10, 100):
        check_topk(x, q, k, metric, 6, table)
    check_topk(x, q[:1], 10, metric, 4, table)
    check_topk(x, q[:7], 10, metric, 6, table, n=50001)


@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("kind", ["equal", "two", "cluster", "copies"])
def test_topk_ties_and_crowded_thresholds(kind, metric):
    """more rows at the threshold than the candidate list holds: every row is looked at, and the lowest rows win ties"""
    n, dim = 60000, 64
    x = vectors(n, dim, 3)
    if kind == "equal":
        x[:] = x[0]
    elif kind == "two":
        x[0::2], x[1::2] = x[0].clone(), x[1].clone()
    elif kind == "cluster":      # one run of near rows that the probe's panels hardly meet
        x[20000:26000] = x[0] + 1e-3 * x[20000:26000]
    else:
        x[1000:] = x[torch.randint(0, 1000, (n - 1000,), generator=torch.Generator().manual_seed(1))]
    q = torch.cat([x[:2] * 1.01, vectors(3, dim, 8)])
    check_topk(x, q, 10, metric, 6)
    check_topk(x, q, 300, metric, 4)


def test_topk_rows_that_are_not_numbers():
    x = vectors(40000, 64, 6)
    x[::3] = 0
    x[1::6, 5] = float("nan")
    q = vectors(4, 64, 7)
    q[1] = 0
    q[2, 1] = float("inf")
    for metric in METRICS:
        check_topk(x, q, 10, metric, 6)
    few = x[:60]
    few[3:] = float("nan")
    for metric in METRICS:
        check_topk(few, q, 10, metric, 6)


def test_topk_far_apart_magnitudes():
    """thresholds of rows and queries between 2^-60 and 2^60"""
    g = torch.Generator().manual_seed(2)
    x = vectors(20000, 64, 1) * torch.exp2(torch.randint(-60, 60, (20000, 1), generator=g).float())
    q = vectors(6, 64, 2) * torch.exp2(torch.tensor([[-60.0], [-10], [0], [10], [50], [60]]))
    for metric in METRICS:
        check_topk(x, q, 10, metric, 6)
        check_topk(x, q, 10, metric, 4)


# ---- in use -----------------------------------------------------------------------------------------------------------------------
def test_a_store_in_use():
    """filled in pieces, overwritten, searched, read back: as one program would"""
    dim = 384
    x = vectors(9000, dim, 1, torch.bfloat16)
    table = mx4.empty(9000, dim, DEV)
    for a in range(0, 9000, 1234):
        mx4.write(table, x[a:a + 1234].to(DEV), first=a)
    x[100] = x[8999]
    mx4.write(table, x[8999:].to(DEV), torch.tensor([100], device=DEV))
    q = x[[100, 4000]].to(DEV)
    ids, best = mx4.topk(table, 9000, q, 3, ref.COSINE)
    assert ids[0, :2].tolist() == [100, 8999] and best[0, 0] == best[0, 1] and ids[1, 0] == 4000
    dense = mx4.scores(table, 9000, q, ref.COSINE)
    picked = torch.gather(dense, 1, ids)
    assert (picked - best).abs().max() <= 2 * (7 * 2.0 ** -22)
    same(mx4.read(table, dim, ids[0]), ref.micro(x.double().numpy(), 4)[ids[0].cpu().numpy()])


def test_other_streams():
    x, q = vectors(3000, 128, 1).to(DEV), vectors(5, 128, 2).to(DEV)
    want = mx4.topk(store_of(x), 3000, q, 10, ref.L2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = mx4.topk(store_of(x), 3000, q, 10, ref.L2)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed():
    """one graph of a write, a read, scores and two searches (their workspaces apart), replayed over new inputs"""
    n, dim = 30000, 96
    table = store_of(vectors(n, dim, 1))
    x, q = torch.empty(64, dim, device=DEV), torch.empty(5, dim, device=DEV)
    slots = torch.empty(64, dtype=torch.int64, device=DEV)

    def body():
        mx4.write(table, x, slots)
        return (mx4.read(table, dim, slots), mx4.scores(table, n, q, ref.L2), *mx4.topk(table, n, q, 10, ref.L2), *mx4.topk(table, n, q, 100, ref.IP, 4))

    def fill(seed):
        x.copy_(vectors(64, dim, seed))
        q.copy_(vectors(5, dim, seed + 1))
        slots.copy_(torch.randperm(n, generator=torch.Generator().manual_seed(seed))[:64])
        slots[60:] = -1

    fill(1)
    body()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    with torch.cuda.graph(other):
        out2 = mx4.topk(table, n, q, 10, ref.COSINE)
    for seed in (10, 20, 30):
        fill(seed)
        graph.replay()
        got = [t.clone() for t in out]
        other.replay()
        got += [t.clone() for t in out2]
        torch.cuda.synchronize()
        for a, b in zip(got, (*body(), *mx4.topk(table, n, q, 10, ref.COSINE))):
            assert torch.equal(a, b)


def test_results_repeat():
    x, q = vectors(50000, 96, 1).to(DEV), vectors(70, 96, 2).to(DEV)
    table = store_of(x)
    first = (mx4.scores(table, 50000, q, ref.L2), *mx4.topk(table, 50000, q, 50, ref.L2))
    for _ in range(3):
        again = (mx4.scores(table, 50000, q, ref.L2), *mx4.topk(table, 50000, q, 50, ref.L2))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals():
    table = store_of(vectors(40, 96, 1))
    x = vectors(4, 96, 2).to(DEV)
    slots = torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: mx4.write(table, x[:, :64]), lambda: mx4.write(table, x.double()), lambda: mx4.write(table, x.cpu()),
                 lambda: mx4.write(table, x, slots.cpu()), lambda: mx4.write(table, x, slots[:3]), lambda: mx4.write(table, x, slots.float()),
                 lambda: mx4.write(table, x, slots, first=1), lambda: mx4.write(table, x, first=61), lambda: mx4.write(table, x, first=-1),
                 lambda: mx4.write(table, x[0]), lambda: mx4.write(table.float(), x), lambda: mx4.write(table[:, :-128], x),
                 lambda: mx4.write(table, x.clone().requires_grad_()), lambda: mx4.read(table, 96), lambda: mx4.read(table, 96, slots, n=3),
                 lambda: mx4.read(table, 96, n=65), lambda: mx4.read(table, 0, n=1), lambda: mx4.read(table, 96, n=1, dtype=torch.float64),
                 lambda: mx4.scores(table, 65, x, ref.L2), lambda: mx4.scores(table, -1, x, ref.L2), lambda: mx4.scores(table, 40, x, 3),
                 lambda: mx4.scores(table, 40, x, ref.L2, 8), lambda: mx4.topk(table, 40, x, 0, ref.L2), lambda: mx4.topk(table, 40, x, 4097, ref.L2)):
        with pytest.raises(ValueError):
            call()
    # empty ones are not errors
    assert mx4.scores(table, 0, x, ref.L2).shape == (4, 0) and mx4.scores(table, 40, x[:0], ref.L2).shape == (0, 40)
    ids, best = mx4.topk(table, 0, x, 3, ref.L2)
    assert (ids == -1).all() and (best == -1).all() and mx4.topk(table, 40, x[:0], 3, ref.L2)[0].shape == (0, 3)


# ---- 65 to 256 queries: panels in an LDS ring -----------------------------------------------------------------------------------
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("nq,n,dim,k,bits", [(65, 7001, 64, 1, 6), (128, 20000, 300, 10, 4), (129, 12345, 257, 100, 6), (256, 9000, 700, 10, 6),
                                             (257, 6400, 1024, 20, 4), (65, 7100, 600, 3, 6), (100, 6999, 1000, 40, 4), (128, 9001, 1024, 10, 6), (200, 8200, 1, 5, 6), (66, 70000, 96, 1000, 6), (256, 33000, 128, 500, 4)])
def test_topk_of_many_queries(nq, n, dim, k, bits, metric):
    dtype = DTYPES[(nq + n + dim) % 3]
    check_topk(vectors(n, dim, 1, dtype), vectors(nq, dim, 2, dtype), k, metric, bits)


@pytest.mark.parametrize("nq", [5, 100, 200])
@pytest.mark.parametrize("metric", METRICS)
def test_topk_rows_without_a_score_and_short_ones(metric, nq):
    """zero rows, rows of NaN, rows whose norm is far below the others', a table with fewer scores than k, queries without any"""
    n, dim = 30000, 96 if nq == 5 else 640
    x, q = vectors(n, dim, 3), vectors(nq, dim, 4)
    x[::5] = 0
    x[1::7, 90] = float("nan")
    x[2::11] *= 1e-25
    q[1] = 0
    q[3, 7] = float("inf")
    q[4] *= 1e-22
    check_topk(x, q, 10, metric, 6)
    few = x[:7000].clone()
    few[:] = float("nan")
    few[[3, 40, 41, 6999]] = x[[3, 42, 41, 6999]]
    check_topk(few, q, 10, metric, 6)


@pytest.mark.parametrize("nq", [3, 70, 150])
@pytest.mark.parametrize("metric", METRICS)
def test_topk_dots_that_leave_fp32(metric, nq):
    """partial sums beyond fp32 whose total is not: the rows' true scores decide"""
    dim = 64 if nq == 3 else 576
    for n in (500, 9000):
        x, q = vectors(n, dim, 5), vectors(nq, dim, 6)
        x[7::50] *= 2.0 ** 90
        x[11] = 0
        x[11, 0], x[11, 40] = 2.0 ** 126, 2.0 ** 60
        q[0, 40] = 0.5
        q[1] *= 2.0 ** 100
        q[2] = 0
        q[2, 0], q[2, 32], q[2, 5] = 2.0 ** 70, 2.0 ** 70, 2.0 ** 69
        x[13], x[14] = 0, 0
        x[13, 0], x[13, 32], x[13, 40] = 2.0 ** 70, -(2.0 ** 70), 1.0
        x[14, 0], x[14, 32], x[14, 5] = -(2.0 ** 70), 2.0 ** 70, 2.0 ** 63
        check_topk(x, q, 10, metric, 6)
        check_topk(x, q, 300, metric, 4)


@pytest.mark.parametrize("nq", [2, 90])
def test_topk_many_best_rows_that_crowd(nq):
    """k best of which one is far from the others, and scores equal in groups"""
    n, dim = 50000, 64 if nq == 2 else 520
    x, q = vectors(n, dim, 7), vectors(nq, dim, 8)
    x[100] *= 1e4
    x[200:700] = x[200]
    for metric in METRICS:
        check_topk(x, q, 1000, metric, 6)
    check_topk(x[:20000], q[:2], 4096, ref.IP, 4)


def test_a_store_beyond_4_gib():
    n, dim = 8_400_000, 1024
    table = mx4.empty(n, dim, DEV)
    assert table.numel() > 1 << 32
    x, q = vectors(1000, dim, 9), vectors(100, dim, 10)
    slots = torch.cat([torch.arange(500), torch.arange(n - 500, n)])
    mx4.write(table, x.to(DEV), slots.to(DEV))
    values = ref.micro(x.double().numpy(), 4)
    same(mx4.read(table, dim, slots.to(DEV)), values)
    for nq in (1, 40, 100):
        ids, best = mx4.topk(table, n, q[:nq].to(DEV), 5, ref.COSINE)
        want_ids, want = ref.topk(q[:nq].double().numpy(), values, 5, ref.COSINE, 6)
        np.testing.assert_array_equal(ids.cpu().numpy(), slots.numpy()[want_ids])
        np.testing.assert_array_equal(best.cpu().numpy(), want)
    got = mx4.scores(table, n, q[:70].to(DEV), ref.IP)
    want = ref.scores(q[:70].double().numpy(), values, ref.IP, 6)
    assert (np.abs(got[:, slots.to(DEV)].double().cpu().numpy() - want) <= ref.bound(q[:70].double().numpy(), values, ref.IP, 6)).all()
    assert (got[:, 500:n - 500] == 1).all()


# ---- the C entries -----------------------------------------------------------------------------------------------------------------
def entry_topk(table, n, q, k, metric, bits, ws, size):
    ids = torch.empty(len(q), k, dtype=torch.int64, device=DEV)
    best = torch.empty(len(q), k, device=DEV)
    rc = mx4._load().vsgpu_mx4_topk(0, torch.cuda.current_stream().cuda_stream, table.data_ptr(), n, q.shape[1], q.data_ptr(), mx4._TYPES[q.dtype],
                                    len(q), q.stride(0) * q.element_size(), k, metric, bits, ids.data_ptr(), best.data_ptr(), ws.data_ptr(), size)
    return rc, ids, best


@pytest.mark.parametrize("nq,n,dim,k", [(1, 5000, 64, 10), (7, 20000, 300, 1000), (60, 20000, 64, 10), (100, 9000, 1024, 50), (256, 9000, 64, 1),
                                        (300, 30000, 64, 10), (2, 7000, 9001, 5)])
def test_workspaces_are_as_large_as_said(nq, n, dim, k):
    """nothing is written behind one, and a smaller one is refused"""
    table, q = store_of(vectors(n, dim, 1)), vectors(nq, dim, 2).to(DEV)
    lib = mx4._load()
    size = lib.vsgpu_mx4_topk_workspace(n, dim, nq, k, 6)
    ws = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
    rc, ids, best = entry_topk(table, n, q, k, ref.L2, 6, ws, size)
    assert rc == 0 and (ws[size:] == 0x5A).all()
    want = mx4.topk(table, n, q, k, ref.L2)
    assert torch.equal(ids, want[0]) and torch.equal(best, want[1])
    assert entry_topk(table, n, q, k, ref.L2, 6, ws, size - 256)[0] != 0
    size = lib.vsgpu_mx4_scores_workspace(dim, nq, 6)
    ws.fill_(0x5A)
    out = torch.full((nq, n + 5), -7.0, device=DEV)
    rc = lib.vsgpu_mx4_scores(0, torch.cuda.current_stream().cuda_stream, table.data_ptr(), n, dim, q.data_ptr(), mx4._TYPES[q.dtype], nq, dim * 4,
                              ref.L2, 6, out.data_ptr(), n + 5, ws.data_ptr(), size)
    assert rc == 0 and (ws[size:] == 0x5A).all() and (out[:, n:] == -7).all()
    assert torch.equal(out[:, :n], mx4.scores(table, n, q, ref.L2))


def test_two_threads_at_once():
    import threading
    table, q = store_of(vectors(40000, 96, 1)), [vectors(5, 96, 2).to(DEV), vectors(120, 96, 3).to(DEV)]
    want = [mx4.topk(table, 40000, v, 20, ref.L2) for v in q]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = mx4.topk(table, 40000, q[i], 20, ref.L2)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_many_queries_captured_and_replayed():
    n, dim = 20000, 640
    table, q = store_of(vectors(n, dim, 1)), torch.empty(130, dim, device=DEV)
    q.copy_(vectors(130, dim, 2))
    mx4.topk(table, n, q, 1000, ref.IP)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (*mx4.topk(table, n, q, 10, ref.L2), *mx4.topk(table, n, q[:20], 1000, ref.IP))
    for seed in (5, 6, 7):
        q.copy_(vectors(130, dim, seed))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, (*mx4.topk(table, n, q, 10, ref.L2), *mx4.topk(table, n, q[:20], 1000, ref.IP))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("nq,n,dim,k", [(1, 64, 1024, 5), (40, 65, 1024, 64), (3, 512, 128, 100), (300, 513, 100, 7), (2, 1024, 64, 1024), (2, 1025, 64, 9), (5, 16, 9000, 4)])
def test_topk_of_very_small_tables(nq, n, dim, k, metric):
    """on both sides of the size up to which every row is scored without a probe; zero, short, long and NaN rows among them"""
    x, q = vectors(n, dim, 1), vectors(nq, dim, 2)
    x[1], x[2, 0], x[3], x[5] = 0, float("nan"), x[3] * 1e-30, x[5] * 2.0 ** 80
    q[-1] *= 2.0 ** 90
    check_topk(x, q, k, metric, 6)
    check_topk(x, q, k, metric, 4)


# ---- many short rows read at once -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 9, 16, 17])
@pytest.mark.parametrize("m", [2, 33, 700, 5000])
def test_many_short_rows_come_back(m, dim):
    x = vectors(m, dim, m + dim)
    want = ref.micro(x.double().numpy(), 4)
    table = store_of(x)
    slots = torch.randint(-1, m, (m,), generator=torch.Generator().manual_seed(dim))
    by_slots = np.where(slots.numpy()[:, None] < 0, 0.0, want[slots.numpy().clip(min=0)])
    for dtype in DTYPES:
        def rounded(v):
            return torch.from_numpy(np.ascontiguousarray(v)).to(dtype).double().numpy()
        same(mx4.read(table, dim, n=m, dtype=dtype), rounded(want))
        same(mx4.read(table, dim, slots.to(DEV), dtype=dtype), rounded(by_slots))
        same(mx4.read(table, dim, slots.int().to(DEV), dtype=dtype), rounded(by_slots))


def test_reading_short_rows_writes_nothing_beside_them():
    """rows a stride apart, the elements between them and behind the last one as they were"""
    m, dim, stride = 1000, 5, 11
    x = vectors(m, dim, 1)
    table, out = store_of(x), torch.full((m + 3, stride), -7.0, device=DEV)
    rc = mx4._load().vsgpu_mx4_read(0, torch.cuda.current_stream().cuda_stream, table.data_ptr(), m, dim, None, 0, 3, m - 3, out.data_ptr(),
                                    mx4._TYPES[torch.float32], stride * 4)
    assert rc == 0
    same(out[:m - 3, :dim], ref.micro(x.double().numpy(), 4)[3:])
    assert (out[:m - 3, dim:] == -7).all() and (out[m - 3:] == -7).all()


# ---- matrix-core dots at their worst ----------------------------------------------------------------------------------------------
# An instruction leaves a block of 32 products out when its scales' power of two is 2^32 below the sum so far: up to 32 x 7.5 x 6 x 2^-32 of
# it (4 bits: 32 x 6 x 6), for each of its two blocks.
def left_out_blocks(dim, bits, sign, first, q_first):
    """a query and a row: a product of 2^40 in front, then blocks of the largest codes that are all left out beside it"""
    q, x = np.zeros(dim), np.zeros(dim)
    q[0] = x[0] = 2.0 ** 20
    q[32:64], x[32:32 + len(first)] = q_first, first
    q[64:], x[64:] = (7.5 if bits == 6 else 6) * 16, sign * 6 * 16
    return q, x


@pytest.mark.parametrize("dim,bits,lead", [(1024, 6, (1, .5)), (4096, 6, (4, 1)), (16384, 6, (4, 1)), (65536, 6, (4, 1)), (65536, 4, (6, 2, .5))])
def test_topk_when_dots_are_off_by_their_most(dim, bits, lead):
    """the nearest row's dot comes back too small, another's too large, by more than lies between them"""
    n = 6200   # (more rows than are scored exactly or bounded one by one)
    # the other row's lead: more than twice the errors' difference allows for, less than the errors
    first = np.array(lead) * {1024: 2.0 ** 11, 4096: 2.0 ** 12, 16384: 2.0 ** 14, 65536: 2.0 ** 16 if bits == 6 else 2.0 ** 15}[dim]
    q, near = left_out_blocks(dim, bits, 1, (), 4096.0)
    _, other = left_out_blocks(dim, bits, -1, first, 4096.0)
    assert near @ q > other @ q
    rows = torch.from_numpy(np.stack([other, near])).float()
    same(rows, ref.micro(rows.double().numpy(), 4))
    assert np.array_equal(ref.micro(q[None], bits)[0], q)
    table = mx4.empty(n, dim, DEV)
    mx4.write(table, rows.to(DEV), torch.tensor([3, 5000], device=DEV))
    query = torch.from_numpy(q[None]).float().to(DEV)
    want = np.array([1 - near @ q, 1 - other @ q]).astype(np.float32)
    for nq in (1, 70, 130):
        for k in (1, 2):
            ids, best = mx4.topk(table, n, query.expand(nq, -1), k, ref.IP, bits)
            assert (ids.cpu().numpy() == np.array([5000, 3])[:k]).all()
            assert (best.cpu().numpy() == want[:k]).all()


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("dim", [64, 1000, 4096])
def test_scores_of_blocks_far_apart(dim, bits):
    """steps of which a dot keeps nothing, and others: within 2^-20 of |q| |x| each"""
    g = torch.Generator().manual_seed(dim + bits)
    spread = torch.exp2(torch.randint(-20, 1, (300, (dim + 31) // 32), generator=g).float()).repeat_interleave(32, 1)[:, :dim]
    x, q = vectors(300, dim, 1).abs() * spread, vectors(40, dim, 2).abs() * spread[:40]
    far = left_out_blocks(dim, bits, 1, (), 0.0)
    q[0], x[0] = torch.from_numpy(far[0]).float() * 2.0 ** -20, torch.from_numpy(far[1]).float() * 2.0 ** -20
    values, q64 = ref.micro(x.double().numpy(), 4), ref.micro(q.double().numpy(), bits)
    size = np.sqrt((q64 ** 2).sum(1))[:, None] * np.sqrt((values ** 2).sum(1))[None]
    got = mx4.scores(store_of(x), 300, q.to(DEV), ref.IP, bits).double().cpu().numpy()
    # 1 - dot is rounded once more
    assert (np.abs(got - (1 - q64 @ values.T)) <= (dim + 63) // 64 * 2.0 ** -20 * size + 2.0 ** -24 * (1 + size)).all()


@pytest.mark.parametrize("dim", [64, 1000])
@pytest.mark.parametrize("power", [-25, -40, -50, -58])
def test_cosine_scores_of_short_vectors(power, dim):
    """on both sides, down to a product of norms of about 2^-116"""
    x, q = vectors(200, dim, 3) * 2.0 ** power, vectors(20, dim, 4) * 2.0 ** power
    values = ref.micro(x.double().numpy(), 4)
    for bits in (4, 6):
        got = mx4.scores(store_of(x), 200, q.to(DEV), ref.COSINE, bits).double().cpu().numpy()
        want = ref.scores(q.double().numpy(), values, ref.COSINE, bits)
        assert (np.abs(got - want) <= ref.bound(q.double().numpy(), values, ref.COSINE, bits)).all()


@pytest.mark.parametrize("nq", [3, 70, 150])
def test_topk_cosine_of_norms_beside_the_shortest_bounded_one(nq):
    """rows and queries between 2e-19 and 5e-18: on both sides of 1e-18, below which no bound is made"""
    n, dim = 9000, 64 if nq == 3 else 576
    g = torch.Generator().manual_seed(nq)
    x, q = vectors(n, dim, 5), vectors(nq, dim, 6)
    x *= 1e-18 * torch.exp(3.2 * torch.rand(n, 1, generator=g) - 1.6) / x.norm(dim=1, keepdim=True)
    q *= 1e-18 * torch.exp(3.2 * torch.rand(nq, 1, generator=g) - 1.6) / q.norm(dim=1, keepdim=True)
    for bits in (4, 6):
        check_topk(x, q, 10, ref.COSINE, bits)
        check_topk(x, q, 200, ref.COSINE, bits)


@pytest.mark.parametrize("nq,dim", [(3, 64), (70, 300), (200, 1024), (40, 5000)])
def test_l2_scores_of_zero_rows_are_the_squares_of_the_queries(nq, dim):
    """|q|^2 comes from 64 bits, rounded once"""
    q = vectors(nq, dim, 7)
    for bits in (4, 6):
        got = mx4.scores(mx4.empty(40, dim, DEV), 40, q.to(DEV), ref.L2, bits).cpu().numpy()
        want = (ref.micro(q.double().numpy(), bits) ** 2).sum(1).astype(np.float32)
        assert (got == want[:, None]).all()
