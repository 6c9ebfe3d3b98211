"""What the grouped products, the gradient norm and the clipped Adam step refuse, without a GPU."""
import array
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from torch_geometric_autoscale import _lib
    return _lib.lib()


def _refused(rc, text):
    from torch_geometric_autoscale import _lib
    assert rc < 0 and text in _lib.last_error(), _lib.last_error()


def test_host_tensors_are_refused():
    from torch_geometric_autoscale import nn, ops, optim
    with pytest.raises(RuntimeError, match="GPU"):
        ops.group_rows(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.groups_from_ptr(torch.zeros(4, dtype=torch.int64), 2)
    groups = ops.RowGroups(None, torch.zeros(3, dtype=torch.int32), 4)
    assert groups.n_groups == 2 and groups.n_rows == 4
    with pytest.raises(RuntimeError, match="GPU"):
        ops.grouped_gemm(torch.zeros(4, 3), torch.zeros(2, 5, 3), groups, trans_w=True)
    with pytest.raises(RuntimeError, match="GPU"):
        nn.GroupedLinear(3, 5, 2)(torch.zeros(4, 3), groups)
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    for fn in (lambda: optim.grad_norm(p), lambda: optim.clip_grad_norm_([p], 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            fn()
    with pytest.raises(ValueError, match="norm_type"):
        optim.grad_norm(p, 4)
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_(p, float("nan"))
    p.grad = None
    assert float(optim.clip_grad_norm_(p, 1.0)) == 0.0


def test_row_groups_are_checked():
    from torch_geometric_autoscale import ops
    ptr, order = torch.zeros(3, dtype=torch.int32), torch.arange(4, dtype=torch.int32)
    assert ops.RowGroups(order, ptr, 4).n_groups == 2
    for bad in ((order[:3], ptr, 4), (order.long(), ptr, 4), (order, ptr.long(), 4),
                (order.repeat(2)[::2], ptr, 4), (order, ptr.view(1, 3), 4), (order, ptr[:1], 4),
                (None, torch.zeros(2050, dtype=torch.int32), 4)):
        with pytest.raises(ValueError):
            ops.RowGroups(*bad)


def test_layer_parameters():
    from torch_geometric_autoscale import nn
    torch.manual_seed(0)
    layer = nn.GroupedLinear(16, 7, 3)
    assert layer.weight.shape == (3, 7, 16) and layer.bias.shape == (3, 7)
    assert float(layer.weight.detach().abs().max()) <= 0.25      # 1 / sqrt(16), as Linear
    assert nn.GroupedLinear(16, 7, 3, bias=False).bias is None
    assert set(layer.state_dict()) == {"weight", "bias"}


FAKE = 1 << 20       # never dereferenced: every call below is refused before a launch


def test_c_entries_refuse_bad_sizes(L):
    _refused(L.incagg_group_rows(FAKE, 1, -1, 3, None, 0, FAKE, FAKE, None), "rows")
    _refused(L.incagg_group_rows(FAKE, 1, 2 ** 31 - 1, 3, None, 0, FAKE, FAKE, None), "rows")
    _refused(L.incagg_group_rows(FAKE, 1, 8, 0, None, 0, FAKE, FAKE, None), "n_groups")
    _refused(L.incagg_group_rows(FAKE, 1, 8, 2 ** 20, None, 0, FAKE, FAKE, None), "n_groups")
    _refused(L.incagg_group_rows(None, 1, 8, 3, None, 0, FAKE, FAKE, None), "null")
    _refused(L.incagg_group_rows(FAKE, 1, 100000, 3, FAKE, 5, FAKE, FAKE, None), "workspace")
    _refused(L.incagg_group_rows_ws_ints(10, 10 ** 6), "out of range")
    _refused(L.incagg_group_ptr(FAKE, 1, 0, 8, FAKE, None), "n_groups")
    _refused(L.incagg_group_ptr(None, 1, 2, 8, FAKE, None), "null")

    def gemm(x=FAKE, ldx=8, w=FAKE * 2, ldw=8, wg=64, trans=1, bias=None, ldb=0, ptr=FAKE, groups=2,
             rows=8, k=8, n=8, dtype=0, y=FAKE * 3, ldy=8):
        return L.incagg_grouped_gemm(x, ldx, w, ldw, wg, trans, bias, ldb, ptr, None, groups, rows, k,
                                     n, dtype, y, ldy, None)
    for bad, text in ((dict(rows=-1), "rows"), (dict(groups=0), "n_groups"), (dict(ptr=None), "null"),
                      (dict(k=0), "widths"), (dict(n=1 << 21), "widths"), (dict(x=None), "null"),
                      (dict(ldx=7), "leading"), (dict(ldy=7), "leading"), (dict(ldw=7), "leading"),
                      (dict(bias=FAKE, ldb=7), "leading"), (dict(y=FAKE), "alias"),
                      (dict(dtype=7), "type")):
        _refused(gemm(**bad), text)
    assert gemm(rows=0) == 0

    def tn(a=FAKE, lda=8, b=FAKE * 2, ldb=8, ptr=FAKE, groups=2, rows=8, m=8, n=8, dtype=0,
           d=FAKE * 3, dg=64, ws=FAKE * 4, wsb=1 << 40):
        return L.incagg_grouped_tn(a, lda, b, ldb, ptr, None, groups, rows, m, n, dtype, d, dg, None,
                                   ws, wsb, None)
    for bad, text in ((dict(rows=-1), "rows"), (dict(groups=0), "n_groups"), (dict(ptr=None), "null"),
                      (dict(m=0), "widths"), (dict(a=None), "null"), (dict(lda=7), "leading"),
                      (dict(dg=63), "d_group"), (dict(d=FAKE), "alias"), (dict(dtype=-1), "type")):
        _refused(tn(**bad), text)


def test_c_norm_entries_refuse_bad_lists(L):
    def segs(*rows):
        flat = array.array("q", [v for r in rows for v in r])
        return flat, flat.buffer_info()[0]
    keep, one = segs((FAKE, 10, 0))
    _refused(L.incagg_grad_norm(one, 1, 5, FAKE, 1, FAKE, None), "norm type")
    _refused(L.incagg_grad_norm(one, 1, 2, FAKE, 0, FAKE, None), "workspace")
    _refused(L.incagg_grad_norm(one, 1, 2, FAKE, 1, None, None), "null")
    _refused(L.incagg_grad_norm(None, 1, 2, FAKE, 1, FAKE, None), "list")
    _refused(L.incagg_grad_clip(one, 1, 2, -1.0, FAKE, 1, FAKE, None), "max_norm")
    _refused(L.incagg_grad_clip(one, 1, 2, float("nan"), FAKE, 1, FAKE, None), "max_norm")
    for row, text in (((FAKE, -1, 0), "length"), ((FAKE, 10, 3), "type"), ((0, 10, 0), "null"),
                      ((FAKE + 2, 10, 0), "aligned"), ((FAKE + 1, 10, 1), "aligned"),
                      ((FAKE, 1 << 50, 0), "length")):
        keep, bad = segs(row)
        _refused(L.incagg_grad_norm(bad, 1, 2, FAKE, 1 << 20, FAKE, None), text)
    keep, both = segs((FAKE, 10, 0), (FAKE + 36, 10, 0))
    _refused(L.incagg_grad_clip(both, 2, 2, 1.0, FAKE, 8, FAKE, None), "overlap")
    _refused(L.incagg_grad_norm_ws_doubles(-1, 5), "negative")
    from torch_geometric_autoscale import _lib
    hyper = (_lib.AdamHyper * 1)(_lib.AdamHyper(1e-3, 0.9, 0.999, 1e-8, 0.0))
    h = ctypes.addressof(hyper)
    good = (FAKE, FAKE * 2, FAKE * 3, FAKE * 4, FAKE * 5, 16, 0)
    for row, text in (((FAKE, FAKE * 2, FAKE * 3, FAKE * 4, FAKE * 5, 16, 1), "hyper"),
                      ((FAKE, FAKE * 2, FAKE * 3, FAKE * 3 + 32, FAKE * 5, 16, 0), "overlap"),
                      ((FAKE, 0, FAKE * 3, FAKE * 4, FAKE * 5, 16, 0), "null"),
                      ((FAKE, FAKE * 2, FAKE * 3, FAKE * 4, FAKE * 5, -4, 0), "length")):
        keep, bad = segs(row)
        _refused(L.incagg_adam_step_clipped_f32(bad, 1, h, 1, 1.0, FAKE, 8, FAKE, None), text)
    keep, twice = segs(good, good)
    _refused(L.incagg_adam_step_clipped_f32(twice, 2, h, 1, 1.0, FAKE, 8, FAKE, None), "twice")
    keep, one = segs(good)
    _refused(L.incagg_adam_step_clipped_f32(one, 1, h, 1, -1.0, FAKE, 8, FAKE, None), "max_norm")
    _refused(L.incagg_adam_step_clipped_f32(one, 1, h, 1, 1.0, FAKE, 0, FAKE, None), "workspace")
    _refused(L.incagg_adam_step_clipped_f32(one, 1, h, 0, 1.0, FAKE, 8, FAKE, None), "hyper")


def test_workspace_bounds_cover_the_launches(L):
    """Never fewer partials than the launches leave: units of 8192 elements, 128 tensors and at most
    1024 partials a launch."""
    import random
    rng = random.Random(1)
    for _ in range(200):
        sizes = [rng.choice([0, 1, 8192, 8193, rng.randrange(1, 10 ** 7)])
                 for _ in range(rng.randrange(0, 400))]
        live = [n for n in sizes if n]
        need = sum(min(1024, sum(-(-n // 8192) for n in live[i:i + 128]))
                   for i in range(0, len(live), 128))
        assert L.incagg_grad_norm_ws_doubles(len(sizes), sum(sizes)) >= need


def test_a_missing_training_module_fails_loudly(monkeypatch):
    from torch_geometric_autoscale import _lib, ops, optim
    assert ops.train_ops_built()
    monkeypatch.setattr(ops, "_train_ops", None)
    monkeypatch.setattr(ops, "TRAIN_OPS_PATH", "/nonexistent/_train_ops.so")
    assert not ops.train_ops_built()
    p = torch.nn.Parameter(torch.zeros(3))
    for call in (ops.train_ops, lambda: optim.clip_grad_norm_(p, 1.0), lambda: optim.grad_norm(p),
                 lambda: ops.group_rows(torch.zeros(3, dtype=torch.int64), 2)):
        with pytest.raises(_lib.IncAggLibraryError):
            call()
    assert not optim.clips([p])
