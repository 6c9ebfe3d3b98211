"""Rows ordered by group, and products with one weight matrix per group, against plain loops in
64 bits.

Tolerance of a sum of L products in float32: every product and every addition is off by at most
2^-23 of what it gives (an adder that truncates; 2^-24 for one that rounds to nearest), so the sum
is off by at most (L + 8) 2^-23 times the sum of the magnitudes of its terms, whatever the order;
then half a step of the result's type (eps / 2), and its smallest value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -24}


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


@pytest.fixture(scope="module")
def ops():
    from torch_geometric_autoscale import ops
    return ops


@pytest.fixture(scope="module")
def nn():
    from torch_geometric_autoscale import nn
    return nn


@pytest.fixture(autouse=True)
def clean_error_latch():
    from torch_geometric_autoscale import _lib
    yield
    _lib.check_device_errors()


def _expected_groups(ids, n_groups):
    ids = ids.cpu()
    key = torch.where((ids < 0) | (ids >= n_groups), torch.full_like(ids, n_groups), ids)
    order = torch.sort(key, stable=True).indices
    ptr = torch.tensor([int((key < g).sum()) for g in range(n_groups + 1)])
    return order.int(), ptr.int()


# ------------------------------------------------------------------ ordering rows
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("rows,n_groups", [
    (0, 3), (1, 1), (1, 7), (63, 2), (64, 64), (65, 5), (4095, 16), (4096, 2048), (4097, 2048),
    (8192, 1), (8193, 3), (40_000, 100), (70_001, 16), (1_200_003, 4)])
def test_group_rows_is_the_stable_order(ops, dev, rows, n_groups, dtype):
    gen = torch.Generator(device=dev).manual_seed(rows + n_groups)
    ids = torch.randint(-1, n_groups, (rows,), device=dev, generator=gen).to(dtype)
    got = ops.group_rows(ids, n_groups)
    order, ptr = _expected_groups(ids, n_groups)
    assert got.n_groups == n_groups and got.n_rows == rows
    assert torch.equal(got.order.cpu(), order) and torch.equal(got.ptr.cpu(), ptr)


@pytest.mark.parametrize("fill", ["one", "none", "sorted", "reversed", "first", "last"])
def test_group_rows_of_special_inputs(ops, dev, fill):
    rows, n_groups = 30_011, 9
    at = torch.arange(rows, device=dev)
    ids = {"one": torch.full_like(at, 4), "none": torch.full_like(at, -1),
           "sorted": at * n_groups // rows, "reversed": (rows - 1 - at) * n_groups // rows,
           "first": torch.where(at == 0, 0, 8), "last": torch.where(at == rows - 1, 0, 8)}[fill]
    got = ops.group_rows(ids, n_groups)
    order, ptr = _expected_groups(ids, n_groups)
    assert torch.equal(got.order.cpu(), order) and torch.equal(got.ptr.cpu(), ptr)


def test_group_rows_reports_bad_ids(ops, dev):
    from torch_geometric_autoscale import _lib
    for rows in (100, 9000):
        for dtype, bad in ((torch.int64, (7, -2, 2 ** 40, -2 ** 62)), (torch.int32, (7, -2))):
            for b in bad:
                ids = torch.arange(rows, device=dev, dtype=dtype) % 7
                ids[rows // 2] = b
                got = ops.group_rows(ids, 7)
                order, ptr = _expected_groups(ids, 7)
                assert torch.equal(got.order.cpu(), order) and torch.equal(got.ptr.cpu(), ptr)
                with pytest.raises(RuntimeError):
                    _lib.check_device_errors()


def test_groups_from_ptr(ops, dev):
    from torch_geometric_autoscale import _lib
    for dtype in (torch.int64, torch.int32):
        ptr = torch.tensor([0, 0, 5, 5, 9, 12], device=dev, dtype=dtype)
        got = ops.groups_from_ptr(ptr, 12)
        assert got.order is None and got.ptr.tolist() == ptr.tolist() and got.n_groups == 5
    long = torch.arange(0, 2049, device=dev) * 3
    assert torch.equal(ops.groups_from_ptr(long, 7000).ptr, long.int())
    _lib.check_device_errors()
    for bad, fixed in (([1, 5, 9], [0, 5, 9]), ([0, 6, 4], [0, 6, 6]), ([0, 5, 2 ** 40], [0, 5, 9]),
                       ([0, -3, 9], [0, 0, 9])):
        got = ops.groups_from_ptr(torch.tensor(bad, device=dev), 9)
        assert got.ptr.tolist() == fixed
        with pytest.raises(RuntimeError):
            _lib.check_device_errors()


# ------------------------------------------------------------------ products
def _ids(kind, rows, n_groups, dev, gen):
    if kind == "random":
        return torch.randint(0, n_groups, (rows,), device=dev, generator=gen)
    if kind == "ragged":            # one group has most rows, some have none, some rows no group
        ids = torch.randint(-1, max(1, n_groups // 2), (rows,), device=dev, generator=gen)
        ids[torch.rand(rows, device=dev, generator=gen) < 0.6] = n_groups - 1
        return ids
    if kind == "none":
        return torch.full((rows,), -1, device=dev)
    return torch.full((rows,), n_groups // 2, device=dev)              # "one"


def _rows64(x, w, b, ids, trans_w):
    n = w.size(1 if trans_w else 2)
    y, mag = (torch.zeros(x.size(0), n, dtype=torch.float64, device=x.device) for _ in range(2))
    for g in range(w.size(0)):
        mine = torch.nonzero(ids == g).view(-1)
        if mine.numel() == 0:
            continue
        xg, wg = x[mine].double(), w[g].double()
        wg = wg.t().contiguous() if trans_w else wg
        y[mine] = xg @ wg
        mag[mine] = xg.abs() @ wg.abs()
        if b is not None:
            y[mine] += b[g].double()
            mag[mine] += b[g].double().abs()
    return y, mag


def _tn64(a, b, ids, n_groups):
    shape = (n_groups, a.size(1), b.size(1))
    d, mag = (torch.zeros(shape, dtype=torch.float64, device=a.device) for _ in range(2))
    s, smag = (torch.zeros(shape[:2], dtype=torch.float64, device=a.device) for _ in range(2))
    count = torch.zeros(n_groups, device=a.device)
    for g in range(n_groups):
        mine = torch.nonzero(ids == g).view(-1)
        if mine.numel():
            ag, bg = a[mine].double(), b[mine].double()
            at = ag.t().contiguous()
            d[g], mag[g] = at @ bg, at.abs() @ bg.abs()
            s[g], smag[g] = ag.sum(0), ag.abs().sum(0)
            count[g] = mine.numel()
    return d, mag, s, smag, count


def _close(got, want, mag, length, dtype):
    tol = (length + 8) * 2.0 ** -23 * mag + HALF_STEP[dtype] * want.abs() + TINY[dtype]
    off = (got.double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert bool((off <= tol).all()), \
        f"off by {float((off / tol.clamp(min=1e-300)).max()):.2f} of the tolerance"


def _case(dev, rows, n_groups, k, n, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, k, device=dev, generator=gen).to(dtype)
    w = (torch.randn(n_groups, n, k, device=dev, generator=gen) / math.sqrt(k)).to(dtype)
    b = torch.randn(n_groups, n, device=dev, generator=gen).to(dtype)
    dy = torch.randn(rows, n, device=dev, generator=gen).to(dtype)
    return gen, x, w, b, dy


SHAPES = [
    # rows, groups, k, n
    (1, 1, 1, 1), (1, 64, 256, 256), (2, 3, 5, 7), (12, 64, 1024, 1024), (17, 1, 33, 65),
    (64, 4, 64, 64), (127, 5, 100, 47), (129, 5, 130, 129), (300, 2, 31, 257), (513, 37, 602, 41),
    (1000, 7, 256, 256), (2500, 3, 47, 256), (4097, 11, 128, 40), (700, 300, 24, 48),
    (5000, 2, 520, 264), (20_011, 4, 100, 256),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n_groups,k,n", SHAPES)
def test_products_and_gradients_match_the_loops(ops, dev, rows, n_groups, k, n, dtype):
    kinds = ["random", "ragged"] if rows > 2 else ["random", "one", "none"]
    for j, kind in enumerate(kinds):
        gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, dtype, 7 * rows + k + j)
        ids = _ids(kind, rows, n_groups, dev, gen)
        groups = ops.group_rows(ids, n_groups)
        y = ops.grouped_gemm(x, w, groups, trans_w=True, bias=b)
        _close(y, *_rows64(x, w, b, ids, True), k + 1, dtype)
        dx = ops.grouped_gemm(dy, w, groups)
        _close(dx, *_rows64(dy, w, None, ids, False), n, dtype)
        dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
        d, mag, s, smag, count = _tn64(dy, x, ids, n_groups)
        _close(dw, d, mag, count.view(-1, 1, 1), dtype)
        _close(db, s, smag, count.view(-1, 1), dtype)
        # the same bits every time, with and without the sums
        assert torch.equal(ops.grouped_tn(dy, x, groups), dw)
        assert torch.equal(ops.grouped_gemm(x, w, groups, trans_w=True, bias=b), y)
        # rows that lie sorted already: the same rows, the same results
        order = groups.order.long()
        here = ops.groups_from_ptr(groups.ptr, rows)
        ys = ops.grouped_gemm(x[order], w, here, trans_w=True, bias=b)
        assert torch.equal(ys, y[order])
        dws, dbs = ops.grouped_tn(dy[order], x[order], here, column_sums=True)
        assert torch.equal(dws, dw) and torch.equal(dbs, db)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,k,n", [(700, 96, 64), (9, 96, 64), (700, 33, 21)])
def test_strides_offsets_and_padding(ops, dev, dtype, rows, k, n):
    """Operands that are windows of wider matrices filled with NaN, starting at odd elements; the
    result goes into a window too, and nothing around it changes."""
    n_groups = 3
    gen, x0, w0, b0, dy0 = _case(dev, rows, n_groups, k, n, dtype, 3)
    ids = _ids("ragged", rows, n_groups, dev, gen)
    groups = ops.group_rows(ids, n_groups)
    for pad, off in ((8, 8), (3, 1), (7, 5), (16, 4)):
        def window(t, fill=math.nan):
            wide = torch.full((*t.shape[:-1], t.size(-1) + off + pad), fill, device=dev, dtype=dtype)
            view = wide[..., off:off + t.size(-1)]
            view.copy_(t)
            return wide, view
        (_, x), (_, w), (_, b), (_, dy) = (window(t) for t in (x0, w0, b0, dy0))
        wide, out = window(torch.zeros(rows, n, device=dev), 3.0)
        y = ops.grouped_gemm(x, w, groups, trans_w=True, bias=b, out=out)
        assert y is out
        _close(y, *_rows64(x0, w0, b0, ids, True), k + 1, dtype)
        assert bool((wide[:, :off] == 3.0).all()) and bool((wide[:, off + n:] == 3.0).all())
        _close(ops.grouped_gemm(dy, w, groups), *_rows64(dy0, w0, None, ids, False), n, dtype)
        dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
        d, mag, s, smag, count = _tn64(dy0, x0, ids, n_groups)
        _close(dw, d, mag, count.view(-1, 1, 1), dtype)
        _close(db, s, smag, count.view(-1, 1), dtype)
    # transposed and expanded operands
    y = ops.grouped_gemm(x0.t().contiguous().t(), w0.transpose(1, 2).contiguous().transpose(1, 2),
                         groups, trans_w=True, bias=b0[:1].expand(n_groups, n))
    _close(y, *_rows64(x0, w0, b0[:1].expand(n_groups, n), ids, True), k + 1, dtype)
    row = dy0[:1].expand(rows, n)
    _close(ops.grouped_gemm(row, w0[:1].expand(n_groups, n, k), groups),
           *_rows64(row, w0[:1].expand(n_groups, n, k), None, ids, False), n, dtype)
    d, mag, s, smag, count = _tn64(row, x0, ids, n_groups)
    dw, db = ops.grouped_tn(row, x0, groups, column_sums=True)
    _close(dw, d, mag, count.view(-1, 1, 1), dtype)
    _close(db, s, smag, count.view(-1, 1), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [20, 700])
def test_values_that_are_not_finite_stay_where_they_are(ops, dev, dtype, rows):
    """An infinity or NaN in one row of x reaches that row of y alone -- with the infinity's own
    sign --, one in the weights of a group only that group's rows, and one in a row of no group
    nothing at all."""
    n_groups, k, n = 4, 64, 96
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, dtype, 5)
    ids = torch.arange(rows, device=dev) % n_groups
    ids[5] = -1
    x[5], dy[5] = math.nan, math.inf
    x[7, 11], x[8, 3], x[9, 60] = math.inf, math.nan, -math.inf
    w[2, 13, 9] = math.inf                       # rows 2 mod 4
    groups = ops.group_rows(ids, n_groups)
    y = ops.grouped_gemm(x, w, groups, trans_w=True, bias=b).double()
    clean = x.clone()
    clean[torch.tensor([5, 7, 8, 9], device=dev)] = 0
    wc = w.clone()
    wc[2, 13, 9] = 0
    want, mag = _rows64(clean, wc, b, ids, True)
    special = torch.zeros(rows, n, dtype=torch.bool, device=dev)
    special[7] = special[8] = special[9] = True
    special[ids == 2, 13] = True
    tol = (k + 9) * 2.0 ** -23 * mag + HALF_STEP[dtype] * want.abs() + TINY[dtype]
    assert bool(((y - want).abs() <= tol)[~special].all())
    assert bool((y[5] == 0).all())
    for r, c, sign in ((7, 11, 1), (9, 60, -1)):
        assert torch.equal(y[r], sign * w[int(ids[r]), :, c].double().sign() * math.inf)
    assert bool(y[8].isnan().all())
    two = (ids == 2).nonzero().view(-1)
    assert torch.equal(y[two, 13], x[two, 9].double().sign() * math.inf)
    # dW: the infinity reaches its group's column alone
    x[5], x[8], x[9] = 0, 0, 0                   # (dy[5] is still infinite: a row of no group)
    dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
    g7 = int(ids[7])
    assert torch.equal(dw[g7, :, 11].double(), dy[7].double().sign() * math.inf)
    bad = torch.zeros_like(dw, dtype=torch.bool)
    bad[g7, :, 11] = True
    xc, dyc = x.clone(), dy.clone()
    xc[7, 11] = 0
    dyc[5] = 0
    d, mag, s, smag, count = _tn64(dyc, xc, ids, n_groups)
    tol = (count.view(-1, 1, 1) + 8) * 2.0 ** -23 * mag + HALF_STEP[dtype] * d.abs() + TINY[dtype]
    assert bool(((dw.double() - d).abs() <= tol)[~bad].all())
    _close(db, s, smag, count.view(-1, 1), dtype)


def test_float32_keeps_its_precision_and_range(ops, dev):
    """Values far from 1, and sums that cancel: float32 operands are not cut to fewer bits."""
    rows, n_groups, k, n = 300, 2, 64, 64
    for scale_x, scale_w in ((1e20, 1e-20), (1e-18, 1e15), (3e37, 1e-3), (1e-25, 1e-6)):
        gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, F32, 21)
        x, w = x * scale_x, w * scale_w
        ids = _ids("random", rows, n_groups, dev, gen)
        groups = ops.group_rows(ids, n_groups)
        _close(ops.grouped_gemm(x, w, groups, trans_w=True), *_rows64(x, w, None, ids, True), k, F32)
    x = torch.randn(rows, k, device=dev, generator=gen)
    x[:, 1::2] = -x[:, ::2] * (1 + 2.0 ** -20)
    w = torch.ones(n_groups, n, k, device=dev)
    _close(ops.grouped_gemm(x, w, groups, trans_w=True), *_rows64(x, w, None, ids, True), k, F32)


def test_a_long_reduction_and_many_rows(ops, dev):
    """A group whose rows are cut into many pieces of the weight gradient, next to tiny ones."""
    rows, n_groups, k, n = 150_001, 6, 40, 72
    for dtype in (F32, BF16):
        gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, dtype, 31)
        ids = _ids("ragged", rows, n_groups, dev, gen)
        ids[:3] = 4
        groups = ops.group_rows(ids, n_groups)
        dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
        d, mag, s, smag, count = _tn64(dy, x, ids, n_groups)
        _close(dw, d, mag, count.view(-1, 1, 1), dtype)
        _close(db, s, smag, count.view(-1, 1), dtype)
        assert torch.equal(ops.grouped_tn(dy, x, groups), dw)
        _close(ops.grouped_gemm(x, w, groups, trans_w=True), *_rows64(x, w, None, ids, True), k,
               dtype)


@pytest.mark.parametrize("dtype,rows,n_groups,k,n", [
    (BF16, 20_003, 5, 200, 1024),      # large tiles, a ragged last chunk of the reduction
    (F16, 40_000, 3, 128, 520),        # large tiles, columns that end inside one
    (BF16, 70_001, 2, 8, 272),         # one chunk, most of it zeros
    (F16, 33_000, 130, 64, 640),       # more groups than large tiles hold rows for
    (F32, 100_003, 4, 40, 512),        # the large tiles of float32
    (BF16, 9_000, 4, 72, 100)])        # 16-byte rows on the one side, not on the other
def test_large_problems(ops, dev, dtype, rows, n_groups, k, n):
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, dtype, rows + n)
    for kind in ("ragged", "random"):
        ids = _ids(kind, rows, n_groups, dev, gen)
        groups = ops.group_rows(ids, n_groups)
        _close(ops.grouped_gemm(x, w, groups, trans_w=True, bias=b), *_rows64(x, w, b, ids, True),
               k + 1, dtype)
        _close(ops.grouped_gemm(dy, w, groups), *_rows64(dy, w, None, ids, False), n, dtype)
        wt = w.transpose(1, 2).contiguous()             # the forward product with W given as [k, n]
        _close(ops.grouped_gemm(x, wt, groups, bias=b), *_rows64(x, wt, b, ids, False), k + 1, dtype)
        dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
        d, mag, s, smag, count = _tn64(dy, x, ids, n_groups)
        _close(dw, d, mag, count.view(-1, 1, 1), dtype)
        _close(db, s, smag, count.view(-1, 1), dtype)
        assert torch.equal(ops.grouped_tn(dy, x, groups), dw)


def test_no_rows(ops, dev):
    groups = ops.group_rows(torch.empty(0, dtype=torch.int64, device=dev), 3)
    w = torch.randn(3, 5, 4, device=dev)
    assert ops.grouped_gemm(torch.empty(0, 4, device=dev), w, groups, trans_w=True).shape == (0, 5)
    dw, db = ops.grouped_tn(torch.empty(0, 5, device=dev), torch.empty(0, 4, device=dev), groups,
                            column_sums=True)
    assert float(dw.abs().sum()) == 0.0 and float(db.abs().sum()) == 0.0 and dw.shape == (3, 5, 4)


def test_offsets_past_32_bits(ops, dev):
    """A matrix of more than 2^32 elements: rows at its end are read and written where they are."""
    rows, k = 2_200_000, 2048
    x = torch.zeros(rows, k, device=dev, dtype=BF16)
    gen = torch.Generator(device=dev).manual_seed(1)
    last = torch.randn(300, k, device=dev, generator=gen).to(BF16)
    x[-300:] = last
    ids = torch.zeros(rows, dtype=torch.int32, device=dev)
    ids[-300:] = 1
    w = torch.randn(2, 8, k, device=dev, generator=gen).to(BF16)
    groups = ops.group_rows(ids, 2)
    y = ops.grouped_gemm(x, w, groups, trans_w=True)
    want, mag = _rows64(last, w[1:], None, torch.zeros(300, device=dev), True)
    _close(y[-300:], want, mag, k, BF16)
    assert float(y[:-300].abs().sum()) == 0.0
    dw = ops.grouped_tn(y, x, groups)
    d, mag, _, _, count = _tn64(y[-300:], last, torch.zeros(300, device=dev), 1)
    _close(dw[1:], d, mag, 300, BF16)
    assert float(dw[0].abs().sum()) == 0.0
    dx = ops.grouped_gemm(y, w, groups)
    want, mag = _rows64(y[-300:], w[1:], None, torch.zeros(300, device=dev), False)
    _close(dx[-300:], want, mag, 8, BF16)
    assert float(dx[:100].abs().sum()) == 0.0
    del x, dx


# ------------------------------------------------------------------ the layer
def test_a_last_row_near_the_limit(ops, dev):
    """The segments of a sum over nearly 2^31 rows end at the last row (not at a sum that passed
    2^31)."""
    rows = 2 ** 31 - 5000
    a, b = (torch.zeros(rows, 1, device=dev, dtype=BF16) for _ in range(2))
    a[-5:] = 1.0
    b[-5:] = 3.0
    ptr = torch.tensor([0, rows - 300, rows], device=dev)
    d, sums = ops.grouped_tn(a, b, ops.groups_from_ptr(ptr, rows), column_sums=True)
    assert d.flatten().tolist() == [0.0, 15.0] and sums.flatten().tolist() == [0.0, 5.0]


def test_out_may_lie_beside_an_operand_but_not_over_it(ops, dev):
    gen, x, w, bias, dy = _case(dev, 300, 3, 24, 24, F32, 7)
    groups = ops.group_rows(_ids("random", 300, 3, dev, gen), 3)
    want = ops.grouped_gemm(x, w, groups, trans_w=True)
    wide = torch.zeros(300, 60, device=dev)
    wide[:, 10:34] = x
    got = ops.grouped_gemm(wide[:, 10:34], w, groups, trans_w=True, out=wide[:, 34:58])
    assert torch.equal(got, want) and torch.equal(wide[:, 10:34], x)
    assert float(wide[:, :10].abs().sum()) == 0.0 and float(wide[:, 58:].abs().sum()) == 0.0
    flat = torch.randn(40_000, device=dev, generator=gen)
    rows = flat[:7200].view(300, 24)
    for over in (wide[:, 11:35], wide[:, 33:57], wide[:, 9:33]):
        with pytest.raises(RuntimeError, match="alias"):
            ops.grouped_gemm(wide[:, 10:34], w, groups, trans_w=True, out=over)
    with pytest.raises(RuntimeError, match="alias"):
        ops.grouped_gemm(x, flat[7000:7000 + 1728].view(3, 24, 24), groups, out=rows)
    with pytest.raises(RuntimeError, match="alias"):
        ops.grouped_gemm(x, w, groups, bias=flat[7199:7199 + 72].view(3, 24), out=rows)


def test_recorded_backward_beside_an_eager_graph(nn, ops, dev):
    """A backward pass is recorded after the eager graph of the same layer is gone; while one lives
    the recording is refused."""
    layer = nn.GroupedLinear(24, 16, 3).to(dev)
    x = torch.randn(100, 24, device=dev)
    groups = ops.group_rows(torch.arange(100, device=dev) % 3, 3)
    for p in layer.parameters():
        p.grad = torch.zeros_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        for p in layer.parameters():
            p.grad.zero_()
        layer(x, groups).square().sum().backward()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    alive = layer(x, groups).square().sum()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph, stream=side):
            step()
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for it in range(4):
        x.copy_(torch.randn(100, 24, device=dev) * (it + 1))
        graph.replay()
        got = [p.grad.clone() for p in layer.parameters()]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, p.grad) for a, p in zip(got, layer.parameters()))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_gradients_match_the_formulas(nn, ops, dev, dtype):
    rows, n_groups, k, n = 777, 5, 40, 24
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, dtype, 13)
    ids = _ids("ragged", rows, n_groups, dev, gen)
    layer = nn.GroupedLinear(k, n, n_groups).to(dev, dtype)
    with torch.no_grad():
        layer.weight.copy_(w)
        layer.bias.copy_(b)
    x.requires_grad_()
    groups = ops.group_rows(ids, n_groups)
    y = layer(x, groups)
    y.backward(dy)
    with torch.no_grad():
        _close(y, *_rows64(x, w, b, ids, True), k + 1, dtype)
        _close(x.grad, *_rows64(dy, w, None, ids, False), n, dtype)
        d, mag, s, smag, count = _tn64(dy, x, ids, n_groups)
        _close(layer.weight.grad, d, mag, count.view(-1, 1, 1), dtype)
        _close(layer.bias.grad, s, smag, count.view(-1, 1), dtype)
    # only what is asked for; a broadcast incoming gradient; no bias
    x.grad = None
    free = nn.GroupedLinear(k, n, n_groups, bias=False, gathered=False).to(dev, dtype)
    free.weight.requires_grad_(False)
    free(x, groups).sum().backward()
    with torch.no_grad():
        _close(x.grad, *_rows64(torch.ones_like(dy), free.weight, None, ids, False), n, dtype)
    assert free.weight.grad is None


def test_layer_gradients_match_differences(nn, ops, dev):
    rows, n_groups, k, n = 40, 3, 9, 6
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, F32, 17)
    ids = _ids("ragged", rows, n_groups, dev, gen)
    groups = ops.group_rows(ids, n_groups)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(nn.grouped_linear(x, w, b, groups), leaves, dy)
    # the layer is linear in each of them: a difference over a step h is exact up to rounding,
    # (k + 1) 2^-23 of the sums of magnitudes on either side, divided by h = 0.5
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        step = torch.zeros_like(leaf)
        flat = torch.randn(leaf.shape, device=dev, generator=gen)
        with torch.no_grad():
            step.copy_(flat)
            def value(sign):
                args = [t.detach() for t in leaves]
                args[i] = args[i] + sign * 0.25 * step
                return (nn.grouped_linear(*args, groups).double() * dy.double()).sum()
            slope = (value(1) - value(-1)) / 0.5
            want = (grad.double() * step.double()).sum()
            mags = sum(float((_rows64(x, w, b, ids, True)[1] * dy.double().abs()).sum())
                       for _ in range(2))
        assert abs(float(slope - want)) <= (k + 9) * 2.0 ** -23 * 4 * mags


def test_padded_output_pitch(nn, ops, dev):
    """``gathered``: a float32 output of width 256 has the row pitch an aggregation wants."""
    layer = nn.GroupedLinear(32, 256, 2).to(dev)
    groups = ops.group_rows(torch.arange(100, device=dev) % 2, 2)
    x = torch.randn(100, 32, device=dev, requires_grad=True)
    y = layer(x, groups)
    assert y.stride(0) == ops.row_pitch(256) and y.shape == (100, 256)
    y.backward(torch.ones_like(y))
    assert x.grad.shape == (100, 32)


def test_second_derivatives_are_refused(nn, ops, dev):
    x = torch.randn(6, 4, device=dev, requires_grad=True)
    w = torch.randn(2, 3, 4, device=dev, requires_grad=True)
    groups = ops.group_rows(torch.arange(6, device=dev) % 2, 2)
    y = nn.grouped_linear(x, w, None, groups)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_forward_mode_derivatives_are_refused(nn, ops, dev):
    from torch.autograd import forward_ad
    layer = nn.GroupedLinear(8, 4, 2).to(dev).requires_grad_(False)
    groups = ops.group_rows(torch.arange(10, device=dev) % 2, 2)
    x = torch.randn(10, 8, device=dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError)):
                layer(dual, groups)
    assert layer(x, groups).shape == (10, 4)


def test_recorded_products_replay(nn, ops, dev):
    """Ordering, forward and gradients recorded into a HIP graph: replays see new rows AND new
    groups, with eager calls of the same operators in between."""
    rows, n_groups, k, n = 5000, 6, 48, 40
    ids = torch.zeros(rows, dtype=torch.int64, device=dev)
    x, dy = (torch.zeros(rows, c, device=dev) for c in (k, n))
    w, b = torch.zeros(n_groups, n, k, device=dev), torch.zeros(n_groups, n, device=dev)

    def step():
        groups = ops.group_rows(ids, n_groups)
        y = ops.grouped_gemm(x, w, groups, trans_w=True, bias=b)
        dx = ops.grouped_gemm(dy, w, groups)
        return (groups.order, groups.ptr, y, dx, *ops.grouped_tn(dy, x, groups, column_sums=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):                        # two graphs that share nothing but their inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            results.append(step())
        graphs.append(graph)
    for it in range(4):
        gen, xn, wn, bn, dyn = _case(dev, rows, n_groups, k, n, F32, 50 + it)
        for old, new in ((x, xn), (w, wn), (b, bn), (dy, dyn)):
            old.copy_(new)
        ids.copy_(_ids("ragged" if it % 2 else "random", rows, n_groups, dev, gen))
        for graph in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_calls_on_two_streams_at_once(ops, dev):
    """Two products that overlap in time share nothing."""
    rows, n_groups, k, n = 30_000, 4, 128, 96
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs, wants = [], []
    for i in range(2):
        gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, F32, 70 + i)
        ids = _ids("random", rows, n_groups, dev, gen)
        inputs.append((ids, x, w, b, dy))
        groups = ops.group_rows(ids, n_groups)
        wants.append((ops.grouped_gemm(x, w, groups, trans_w=True, bias=b),
                      *ops.grouped_tn(dy, x, groups, column_sums=True)))
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, (ids, x, w, b, dy) in zip(streams, inputs):
            with torch.cuda.stream(s):
                groups = ops.group_rows(ids, n_groups)
                got.append((groups, ops.grouped_gemm(x, w, groups, trans_w=True, bias=b),
                            *ops.grouped_tn(dy, x, groups, column_sums=True)))
        torch.cuda.synchronize()
        for g, want in zip(got, wants):
            assert all(torch.equal(a, c) for a, c in zip(g[1:], want))


def test_row_numbers_outside_the_matrix_are_skipped(ops, dev):
    from torch_geometric_autoscale import _lib
    groups = ops.group_rows(torch.arange(200, device=dev) % 3, 3)
    order = groups.order.clone()
    lost = int(order[10])
    order[10] = 10 ** 6
    bad = ops.RowGroups(order, groups.ptr, 200)
    x, w = torch.randn(200, 16, device=dev), torch.randn(3, 8, 16, device=dev)
    out = torch.full((200, 8), 5.0, device=dev)
    ops.grouped_gemm(x, w, bad, trans_w=True, out=out)
    with pytest.raises(RuntimeError):
        _lib.check_device_errors()
    good = ops.grouped_gemm(x, w, groups, trans_w=True)
    keep = torch.arange(200, device=dev) != lost
    assert torch.equal(out[keep], good[keep]) and bool((out[lost] == 5.0).all())
    dw = ops.grouped_tn(good, x, bad)
    with pytest.raises(RuntimeError):
        _lib.check_device_errors()
    gz = good.clone()
    gz[lost] = 0
    assert torch.equal(dw, ops.grouped_tn(gz, x, groups))
    # row pointers that are no row pointers lead nowhere outside either
    wild = ops.RowGroups(None, torch.tensor([0, 150, 40, 10 ** 9], dtype=torch.int32, device=dev), 200)
    ops.grouped_gemm(x, w, wild, trans_w=True, out=out)
    ops.grouped_tn(good, x, wild)


def test_refusals(ops, nn, dev):
    ids = torch.arange(10, device=dev) % 3
    groups = ops.group_rows(ids, 3)
    x, w = torch.randn(10, 4, device=dev), torch.randn(3, 5, 4, device=dev)
    b = torch.randn(3, 5, device=dev)
    for args, kw, err in [
            ((x.double(), w, groups), dict(trans_w=True), TypeError),
            ((x, w.half(), groups), dict(trans_w=True), TypeError),
            ((x, w, groups), dict(trans_w=True, bias=b.half()), TypeError),
            ((x[:9], w, groups), dict(trans_w=True), ValueError),
            ((x, w[:2], groups), dict(trans_w=True), ValueError),
            ((x, w, groups), dict(), ValueError),
            ((x[0], w, groups), dict(trans_w=True), ValueError),
            ((x, w, groups), dict(trans_w=True, bias=b[:, :4]), ValueError),
            ((x, w, groups), dict(trans_w=True, out=torch.empty(10, 4, device=dev)), ValueError),
            ((x, w, groups), dict(trans_w=True, out=torch.empty(5, 10, device=dev).t()), ValueError),
            ((x[:, :0], w[:, :, :0], groups), dict(trans_w=True), ValueError),
            ((x.cpu(), w, groups), dict(trans_w=True), RuntimeError)]:
        with pytest.raises(err):
            ops.grouped_gemm(*args, **kw)
    square = torch.randn(3, 4, 4, device=dev)
    with pytest.raises(RuntimeError, match="alias"):
        ops.grouped_gemm(x, square, groups, out=x)
    with pytest.raises(TypeError):
        ops.grouped_tn(x, x.half(), groups)
    with pytest.raises(ValueError):
        ops.grouped_tn(x, x[:9], groups)
    for bad in (ids.float(), ids.view(2, 5), torch.arange(20, device=dev)[::2]):
        with pytest.raises(TypeError):
            ops.group_rows(bad, 3)
    for bad in (0, -1, 2049):
        with pytest.raises(ValueError):
            ops.group_rows(ids, bad)


# ------------------------------------------------------------------ all of them, as they are used
def test_training_a_typed_network_end_to_end(nn, ops, dev):
    """Order the rows, two typed layers, mean cross entropy, gradients, and the Adam step that
    clips -- against the same steps in float64.  Every float32 step of this small network errs by
    about 1e-6 of what it computes (256-term sums and rounding); lr-sized Adam moves amplify the
    relative error of a gradient that is small against its neighbours, so weights are compared to
    0.02 of the distance they moved, in the 2-norm."""
    from torch_geometric_autoscale.optim import Adam
    gen = torch.Generator(device=dev).manual_seed(77)
    rows, n_groups, k, hidden, classes = 3000, 4, 64, 96, 11
    x = torch.randn(rows, k, device=dev, generator=gen)
    ids = torch.randint(0, n_groups, (rows,), device=dev, generator=gen)
    y = torch.randint(0, classes, (rows,), device=dev, generator=gen)
    torch.manual_seed(3)
    l1, l2 = nn.GroupedLinear(k, hidden, n_groups).to(dev), \
        nn.GroupedLinear(hidden, classes, n_groups, gathered=False).to(dev)
    params = [*l1.parameters(), *l2.parameters()]
    start = [p.detach().double().clone() for p in params]
    ref = [p.clone().requires_grad_() for p in start]
    moments = [[torch.zeros_like(p), torch.zeros_like(p)] for p in ref]
    opt = Adam(params, lr=1e-2)
    criterion = nn.CrossEntropyLoss()
    groups = ops.group_rows(ids, n_groups)
    masks = [(ids == g).nonzero().view(-1) for g in range(n_groups)]
    for it in range(1, 5):
        loss = criterion(l2(nn.relu_into(l1(x, groups)), groups), y)
        opt.zero_grad()
        loss.backward()
        norm = opt.step(max_norm=0.3)
        h = torch.zeros(rows, classes, dtype=torch.float64, device=dev)
        for g, m in enumerate(masks):
            hid = torch.relu(x[m].double() @ ref[0][g].t() + ref[1][g])
            h = h.index_copy(0, m, hid @ ref[2][g].t() + ref[3][g])
        want = torch.nn.functional.cross_entropy(h, y)
        grads = torch.autograd.grad(want, ref)
        total = math.sqrt(sum(float((g * g).sum()) for g in grads))
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-4
        assert abs(float(norm) - total) <= 1e-3 * total
        coef = min(1.0, 0.3 / (total + 1e-6))
        with torch.no_grad():
            for p, g, mv in zip(ref, grads, moments):
                mv[0].mul_(0.9).add_(g * coef, alpha=0.1)
                mv[1].mul_(0.999).add_((g * coef) ** 2, alpha=0.001)
                p -= 1e-2 * (mv[0] / (1 - 0.9 ** it)) / ((mv[1] / (1 - 0.999 ** it)).sqrt() + 1e-8)
    for p, r, s in zip(params, ref, start):
        moved = float((r.detach() - s).norm())
        assert moved > 0 and float((p.detach().double() - r.detach()).norm()) <= 0.02 * moved


@pytest.mark.parametrize("trained", ["x", "weight", "bias"])
def test_recorded_backward_of_one_leaf_beside_an_eager_graph(nn, ops, dev, trained):
    """Whichever of the layer's inputs is the only one with a gradient: the recording is refused while
    an eager graph of it lives, and runs once that graph is gone."""
    gen, x, w, b, dy = _case(dev, 90, 3, 20, 12, F32, 41)
    leaves = {"x": x, "weight": w, "bias": b}
    leaf = leaves[trained].requires_grad_()
    leaf.grad = torch.zeros_like(leaf)
    groups = ops.group_rows(torch.arange(90, device=dev) % 3, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        leaf.grad.zero_()
        nn.grouped_linear(x, w, b, groups).square().sum().backward()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    alive = nn.grouped_linear(x, w, b, groups).sum()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph, stream=side):
            step()
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for it in range(3):
        with torch.no_grad():
            leaf.copy_(torch.randn(leaf.shape, device=dev, generator=gen))
        graph.replay()
        got = leaf.grad.clone()
        step()
        torch.cuda.synchronize()
        assert float(got.abs().sum()) > 0 and torch.equal(got, leaf.grad)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n_groups", [1, 3])
@pytest.mark.parametrize("rows", [40, 700])
def test_weights_with_a_dimension_of_one(nn, ops, dev, dtype, n_groups, rows):
    """Transposed views whose dimension of one has a stride that means nothing, and that count as
    contiguous: one output per kind, one input."""
    gen, x, _, _, dy = _case(dev, rows, n_groups, 40, 24, dtype, 43)
    ids = _ids("ragged", rows, n_groups, dev, gen)
    groups = ops.group_rows(ids, n_groups)
    for k, n in ((40, 1), (1, 24), (1, 1)):
        xk, dyn = x[:, :k], dy[:, :n]
        plain = torch.randn(n_groups, n, k, device=dev, generator=gen).to(dtype)
        flip = plain.transpose(1, 2).contiguous().transpose(1, 2)         # [G, n, k] out of [G, k, n]
        odd = torch.as_strided(flip, flip.shape, [flip.stride(0)] + [
            3 if size == 1 else stride for size, stride in zip(flip.shape[1:], flip.stride()[1:])])
        for w in (flip, odd):
            assert torch.equal(w, plain)
            _close(ops.grouped_gemm(xk, w, groups, trans_w=True), *_rows64(xk, plain, None, ids, True),
                   k, dtype)
            _close(ops.grouped_gemm(dyn, w, groups), *_rows64(dyn, plain, None, ids, False), n, dtype)
            wt = w.transpose(1, 2)                                        # [G, k, n]
            _close(ops.grouped_gemm(xk, wt, groups), *_rows64(xk, plain, None, ids, True), k, dtype)
            xl, wl = xk.detach().clone().requires_grad_(), w.detach().requires_grad_()
            y = nn.grouped_linear(xl, wl, None, groups)
            _close(y.detach(), *_rows64(xk, plain, None, ids, True), k, dtype)
            dx, dw = torch.autograd.grad(y, [xl, wl], dyn)
            _close(dx, *_rows64(dyn, plain, None, ids, False), n, dtype)
            d, mag, _, _, count = _tn64(dyn, xk, ids, n_groups)
            _close(dw, d, mag, count.view(-1, 1, 1), dtype)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -3.4e38])
@pytest.mark.parametrize("rows,n_groups", [(60, 5), (700, 5), (200_000, 3)])
def test_rows_and_columns_of_others_leave_no_trace(ops, dev, rows, n_groups, bad):
    """float32 tiles are filled up with rows and columns that belong to others.  One that is not
    finite (or rounds to an infinity in 16 bits) changes no bit of anything it does not belong to."""
    k, n = 129, 129
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, F32, 47)
    ids = _ids("random", rows, n_groups, dev, gen)
    ids[0] = -1                                  # the first row belongs to no group
    x[0], dy[0] = 0, 0
    groups = ops.group_rows(ids, n_groups)
    wt = w.transpose(1, 2).contiguous()                                   # [G, k, n]

    def results():
        dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
        return (ops.grouped_gemm(x, w, groups, trans_w=True, bias=b), ops.grouped_gemm(x, wt, groups),
                ops.grouped_gemm(dy, w, groups), dw, db, ops.grouped_tn(x, dy, groups))
    clean = results()
    x[0], dy[0] = bad, bad
    assert all(torch.equal(a, c) for a, c in zip(results(), clean))
    # a column of the operands: the tile of the last column is filled up with the ones in front of it,
    # which belong to another tile
    x[0], dy[0] = 0, 0
    last = slice(128, None)
    for at in (126, 127):
        keep = [(t, t.clone()) for t in (x, dy, w, wt)]
        x[:, at], dy[:, at] = bad, bad
        dw, db = ops.grouped_tn(dy, x, groups, column_sums=True)
        assert torch.equal(dw[:, last, last], clean[3][:, last, last])
        assert torch.equal(db[:, last], clean[4][:, last])
        assert torch.equal(ops.grouped_tn(x, dy, groups)[:, last, last], clean[5][:, last, last])
        for t, old in keep:
            t.copy_(old)
        wt[:, :, at], w[:, :, at] = bad, bad
        assert torch.equal(ops.grouped_gemm(x, wt, groups)[:, last], clean[1][:, last])
        assert torch.equal(ops.grouped_gemm(dy, w, groups)[:, last], clean[2][:, last])
        for t, old in keep:
            t.copy_(old)


@pytest.mark.parametrize("rows", [20, 700])
@pytest.mark.parametrize("power", [-140, -126, -118, -110, -100, 60, 100, 111, 113, 120])
def test_float32_over_its_whole_range(ops, dev, rows, power):
    """Factors around 2^power and 2^-power (at most 2^122): products near 1, so the tolerance is that of
    any float32 sum, whatever parts the factors are taken into."""
    n_groups, k, n = 3, 64, 48
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, F32, 53)
    ids = _ids("random", rows, n_groups, dev, gen)
    groups = ops.group_rows(ids, n_groups)
    other = min(-power, 122)

    def at(t, p):           # (in two steps: 2^-140 is no normal float32)
        return t * 2.0 ** (p // 2) * 2.0 ** (p - p // 2)
    xs, ws, dys, xo = at(x, power), at(w, other), at(dy, power), at(x, other)
    _close(ops.grouped_gemm(xs, ws, groups, trans_w=True, bias=b), *_rows64(xs, ws, b, ids, True), k + 1,
           F32)
    _close(ops.grouped_gemm(dys, ws, groups), *_rows64(dys, ws, None, ids, False), n, F32)
    dw, db = ops.grouped_tn(dys, xo, groups, column_sums=True)
    d, mag, s, smag, count = _tn64(dys, xo, ids, n_groups)
    _close(dw, d, mag, count.view(-1, 1, 1), F32)
    _close(db, s, smag, count.view(-1, 1), F32)


@pytest.mark.parametrize("power", [-40, -60, -66, -72, 40, 46, 50, 60])
def test_float32_results_over_their_whole_range(ops, dev, power):
    """Both factors around 2^power: results down to where float32 loses them (2^-149 in the tolerance:
    half a step of the smallest values, and one more for a partial sum), and up to 2^124."""
    rows, n_groups, k, n = 300, 3, 64, 48
    gen, x, w, b, dy = _case(dev, rows, n_groups, k, n, F32, 59)
    ids = _ids("random", rows, n_groups, dev, gen)
    groups = ops.group_rows(ids, n_groups)
    x, w, dy = x * 2.0 ** power, w * 2.0 ** power, dy * 2.0 ** power

    def close(got, want, mag, length):
        tol = (length + 8) * 2.0 ** -23 * mag + HALF_STEP[F32] * want.abs() + 2 * 2.0 ** -149
        assert bool(((got.double() - want).abs() <= tol).all())
    close(ops.grouped_gemm(x, w, groups, trans_w=True), *_rows64(x, w, None, ids, True), k)
    close(ops.grouped_gemm(dy, w, groups), *_rows64(dy, w, None, ids, False), n)
    dw = ops.grouped_tn(dy, x, groups)
    d, mag, _, _, count = _tn64(dy, x, ids, n_groups)
    close(dw, d, mag, count.view(-1, 1, 1))
