"""Global gradient norm, clipping and the Adam step that clips as it reads, against the formulas in
64 bits.

Tolerances.  The norm is added up in float64 and rounded to float32 once: 2^-24 of itself (plus
the float64 sums, below 2^-40).  A clipped value is x * coef with coef a float32 (2^-24) and one
product (2^-24), then rounded to its type (half a step, eps / 2): 2^-23 + eps / 2 for 16-bit types,
2^-23 for float32 (whose product rounding is the rounding to its type) -- written as 1.5 * 2^-23.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


@pytest.fixture(scope="module")
def optim():
    from torch_geometric_autoscale import optim
    return optim


def _params(dev, sizes, dtypes, seed, scale=0.1):
    gen = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for i, s in enumerate(sizes):
        t = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.empty(s, device=dev, dtype=t))
        p.grad = (torch.randn(s, device=dev, generator=gen) * scale).to(t)
        out.append(p)
    return out


def _norm64(grads, p):
    flat = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(0)
    if p == math.inf:
        return float(flat.abs().max()) if flat.numel() else 0.0
    return float(flat.abs().sum()) if p == 1 else math.sqrt(float((flat * flat).sum()))


def _check_clipped(before, after, coef):
    for b, a in zip(before, after):
        want = b.double() * coef
        tol = (1.5 * 2.0 ** -23 + HALF_STEP[b.dtype]) * want.abs() + TINY[b.dtype]
        assert bool(((a.double() - want).abs() <= tol).all())


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CASES = [
    ([(1,)], [F32]),
    ([(3, 5), (7,), (0,), (256, 100)], [F32]),
    ([(8192,), (8193,), (8191,), (16384, 3)], [F32, BF16]),
    ([(17, 9)] * 129, [BF16]),                         # one tensor more than a launch takes
    ([(1000 + 7 * i,) for i in range(300)], [F32, F16, BF16]),
    ([(3_000_001,), (5,), (2_000_003,)], [BF16, F32]),  # more units than partials? (611 units)
    ([(20_000_000,)], [F16]),                          # 2442 units on 1024 workgroups
]


@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_norm_and_clip_match_the_formulas(optim, dev, case, norm_type):
    sizes, dtypes = CASES[case]
    params = _params(dev, sizes, dtypes, case)
    grads = [p.grad for p in params]
    before = [g.clone() for g in grads]
    want = _norm64(before, norm_type)
    norm = optim.grad_norm(params, norm_type)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    assert all(torch.equal(a, b) for a, b in zip(grads, before))       # only read
    max_norm = 0.37 * want
    got = optim.clip_grad_norm_(params, max_norm, norm_type)
    assert torch.equal(got, norm)                                      # the same bits
    _check_clipped(before, grads, min(1.0, max_norm / (want + 1e-6)))
    # a second time, now within the bound: nothing changes
    after = [g.clone() for g in grads]
    optim.clip_grad_norm_(params, 10.0 * want + 1.0, norm_type)
    assert all(torch.equal(a, b) for a, b in zip(grads, after))


def test_norm_of_values_whose_squares_leave_float32(optim, dev):
    p = torch.nn.Parameter(torch.zeros(1000, device=dev))
    for value in (1e30, 1e-30):
        p.grad = torch.full((1000,), value, device=dev)
        want = math.sqrt(1000.0) * float(p.grad[0])
        assert abs(float(optim.grad_norm(p)) - want) <= 2.0 ** -23 * want


def test_views_at_odd_offsets_and_strides(optim, dev):
    """Gradients cut from one flat buffer start at any element; others are transposed views."""
    for dtype in (F32, BF16, F16):
        gen = torch.Generator(device=dev).manual_seed(5)
        flat = (torch.randn(40_000, device=dev, generator=gen) * 0.1).to(dtype)
        guard = flat.clone()
        params, spans, off = [], [], 1
        for n in (1, 2, 3, 5, 1021, 8191, 8195, 16387):
            p = torch.nn.Parameter(torch.empty(n, device=dev, dtype=dtype))
            p.grad = flat[off:off + n]
            params.append(p)
            spans.append((off, n))
            off += n + 1                                              # one element between them
        wide = (torch.randn(33, 70, device=dev, generator=gen) * 0.1).to(dtype)
        q = torch.nn.Parameter(torch.empty(70, 33, device=dev, dtype=dtype))
        q.grad = wide.t()
        params.append(q)
        before = [p.grad.clone() for p in params]
        want = _norm64(before, 2.0)
        got = optim.clip_grad_norm_(params, 0.5 * want)
        assert abs(float(got) - want) <= 2.0 ** -23 * want
        _check_clipped(before, [p.grad for p in params], 0.5 * want / (want + 1e-6))
        untouched = torch.ones(40_000, dtype=torch.bool, device=dev)
        for at, n in spans:
            untouched[at:at + n] = False
        assert torch.equal(flat[untouched], guard[untouched])


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
def test_values_that_are_not_finite(optim, dev, bad, norm_type):
    params = _params(dev, [(100,), (9000,)], [F32], 3)
    params[1].grad[8999] = bad
    twins = [torch.nn.Parameter(torch.empty_like(p)) for p in params]
    for p, t in zip(params, twins):
        t.grad = p.grad.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        optim.clip_grad_norm_(params, 1.0, norm_type, error_if_nonfinite=True)
    assert all(torch.equal(p.grad[:90], t.grad[:90]) for p, t in zip(params, twins))
    norm = optim.clip_grad_norm_(params, 1.0, norm_type)
    ref = torch.nn.utils.clip_grad_norm_(twins, 1.0, norm_type)
    assert float(norm) == float(ref) or (math.isnan(float(norm)) and math.isnan(float(ref)))
    for p, t in zip(params, twins):
        assert torch.equal(p.grad.isnan(), t.grad.isnan())
        assert torch.equal(p.grad.nan_to_num(7.0), t.grad.nan_to_num(7.0))


def test_bounds_at_the_ends(optim, dev):
    params = _params(dev, [(100,), (0,)], [F32], 4)
    before = params[0].grad.clone()
    assert float(optim.clip_grad_norm_(params, math.inf)) > 0        # the norm alone
    assert torch.equal(params[0].grad, before)
    optim.clip_grad_norm_(params, 0.0)
    assert float(params[0].grad.abs().sum()) == 0.0
    params[0].grad.zero_()
    assert float(optim.clip_grad_norm_(params, 1.0)) == 0.0           # a norm of zero
    params[0].grad = None
    assert float(optim.clip_grad_norm_(params, 1.0)) == 0.0           # only an empty gradient
    params[1].grad = None
    assert float(optim.grad_norm(params)) == 0.0


def test_refusals(optim, dev):
    p = torch.nn.Parameter(torch.zeros(64, device=dev))
    q = torch.nn.Parameter(torch.zeros(64, device=dev))
    flat = torch.ones(100, device=dev)
    p.grad, q.grad = flat[:64], flat[36:]
    with pytest.raises(RuntimeError, match="overlap"):
        optim.clip_grad_norm_([p, q], 0.1)
    q.grad = p.grad
    with pytest.raises(RuntimeError, match="overlap"):
        optim.clip_grad_norm_([p, q], 0.1)
    q.grad = torch.ones(1, device=dev).expand(64)
    with pytest.raises(RuntimeError, match="overlap"):
        optim.clip_grad_norm_([p, q], 0.1)
    assert float(flat.sum()) == 100.0                                 # nothing was scaled
    assert abs(float(optim.grad_norm([p, q])) - math.sqrt(128.0)) <= 2.0 ** -20
    q.grad = None
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            optim.clip_grad_norm_([p], bad)
    with pytest.raises(ValueError, match="norm_type"):
        optim.grad_norm([p], 3.0)
    d = torch.nn.Parameter(torch.zeros(4, device=dev, dtype=torch.float64))
    d.grad = torch.ones(4, device=dev, dtype=torch.float64)
    with pytest.raises(TypeError):
        optim.grad_norm([d])


def test_gradients_with_gaps_and_transposed_ones(optim, dev):
    """A transposed gradient is scaled where it lies; columns of a wider matrix keep their
    neighbours; the same columns listed twice are refused."""
    gen = torch.Generator(device=dev).manual_seed(9)
    wide = torch.randn(50, 40, device=dev, generator=gen)
    flip = torch.randn(30, 20, device=dev, generator=gen)
    params = [torch.nn.Parameter(torch.empty(50, 15, device=dev)) for _ in range(2)]
    params.append(torch.nn.Parameter(torch.empty(20, 30, device=dev)))
    params[0].grad, params[1].grad, params[2].grad = wide[:, 3:18], wide[:, 18:33], flip.t()
    before, guard = [p.grad.clone() for p in params], wide.clone()
    want = _norm64(before, 2.0)
    got = optim.clip_grad_norm_(params, 0.25 * want)
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    _check_clipped(before, [p.grad for p in params], 0.25 * want / (want + 1e-6))
    assert torch.equal(wide[:, :3], guard[:, :3]) and torch.equal(wide[:, 33:], guard[:, 33:])
    params[1].grad = params[0].grad
    kept = wide.clone()
    with pytest.raises(RuntimeError, match="overlap"):
        optim.clip_grad_norm_(params, 0.1)
    assert torch.equal(wide, kept)


# ------------------------------------------------------------------ Adam
def _adam64(p, g, m, v, t, coef, lr, b1, b2, eps, wd):
    d = g * coef + wd * p
    m = b1 * m + (1 - b1) * d
    v = b2 * v + (1 - b2) * d * d
    return p - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps), m, v


@pytest.mark.parametrize("sizes", [
    [(256, 256), (47,), (256, 100), (1,), (3, 5), (12032,), (0,)],
    [(17, 9)] * 150,                                   # three update launches, two norm launches
    [(5_000_000,), (4_000_001,), (7,)],                # the large workgroups, ragged ends
])
def test_clipped_adam_matches_the_formulas(optim, dev, sizes):
    """Six steps against float64.  A step moves an element by at most lr * (1 - b1) /
    sqrt(1 - b2) < 3.2 lr and usually by lr; float32 arithmetic on it (under ten operations) and
    the rounding of p (2^-24 |p|) err by less than 16 * 2^-24 * lr * 3.2 + 2^-24 |p| a step, and m
    and v carry theirs along for ten and a thousand steps: six steps stay below 2e-5 lr-sized
    moves plus 6 * 2^-24 |p|."""
    gen = torch.Generator(device=dev).manual_seed(11)
    lr, betas, eps = 1e-2, (0.9, 0.999), 1e-8
    ours = [(torch.randn(s, device=dev, generator=gen)).requires_grad_() for s in sizes]
    k = len(sizes) // 2
    opt = optim.Adam([dict(params=ours[:k], weight_decay=5e-4),
                      dict(params=ours[k:], weight_decay=0.0, lr=2 * lr)], lr=lr, betas=betas,
                     eps=eps)
    ref = [[p.detach().double(), torch.zeros_like(p, dtype=torch.float64),
            torch.zeros_like(p, dtype=torch.float64), 0] for p in ours]
    for it in range(6):
        for i, p in enumerate(ours):
            p.grad = None if (i == 4 and it % 2) else \
                torch.randn(p.shape, device=dev, generator=gen) * (1 + 0.1 * i)
        grads = [p.grad for p in ours if p.grad is not None]
        kept = [g.clone() for g in grads]
        want = _norm64(grads, 2.0)
        max_norm = want * (0.25 if it != 3 else 4.0)           # one step without clipping
        norm = opt.step(max_norm=max_norm)
        assert abs(float(norm) - want) <= 2.0 ** -23 * want
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
        for i, (p, r) in enumerate(zip(ours, ref)):
            if p.grad is None:
                continue
            r[3] += 1
            r[0], r[1], r[2] = _adam64(r[0], p.grad.double(), r[1], r[2], r[3],
                                       min(1.0, max_norm / (want + 1e-6)),
                                       lr if i < k else 2 * lr, *betas, eps,
                                       5e-4 if i < k else 0.0)
    for p, r in zip(ours, ref):
        tol = 2e-5 * 2 * lr * 6 + 6 * 2.0 ** -24 * r[0].abs()
        assert bool(((p.detach().double() - r[0]).abs() <= tol).all())
        # (a tensor without elements does not age, as in step() without clipping)
        assert float(opt.state[p]["step"]) == (r[3] if p.numel() else 0)


def test_clipped_adam_equals_clip_then_step(optim, dev):
    """Against clip_grad_norm_ followed by step() on twins: the same update up to the bias
    corrections, which step() evaluates in float32 (1 - 0.999^t off by up to 6e-5 of itself after
    one step, half of that under the root)."""
    gen = torch.Generator(device=dev).manual_seed(2)
    a = [torch.randn(300, 40, device=dev, generator=gen).requires_grad_() for _ in range(3)]
    b = [p.detach().clone().requires_grad_() for p in a]
    one, two = optim.Adam(a, lr=1e-2), optim.Adam(b, lr=1e-2)
    for _ in range(4):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, device=dev, generator=gen)
            q.grad = p.grad.clone()
        n1 = one.step(max_norm=1.0)
        n2 = optim.clip_grad_norm_(b, 1.0)
        two.step()
        assert torch.equal(n1, n2)
    for p, q in zip(a, b):
        assert float((p.detach() - q.detach()).abs().max()) <= 4 * 1e-2 * 1e-4 + 1e-6


def test_clipped_adam_refusals(optim, dev):
    p = torch.zeros(8, device=dev, requires_grad=True)
    opt = optim.Adam([p], lr=1e-2)
    assert float(opt.step(max_norm=1.0)) == 0.0               # no gradient: nothing to do
    assert float(opt.state[p]["step"]) == 0.0
    p.grad = torch.ones(8, device=dev)
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-1.0)
    twice = optim.Adam([p, p], lr=1e-2)
    with pytest.raises(RuntimeError, match="twice"):
        twice.step(max_norm=1.0)
    assert float(p.detach().abs().sum()) == 0.0
    # an infinite gradient: the others see 0, as with torch's clipping
    q = torch.zeros(8, device=dev, requires_grad=True)
    opt = optim.Adam([p, q], lr=1e-2)
    q.grad = torch.full((8,), math.inf, device=dev)
    assert math.isinf(float(opt.step(max_norm=1.0)))
    assert float(p.detach().abs().sum()) == 0.0 and bool(q.isnan().all())


def test_recorded_clip_and_step_replay(optim, dev):
    """Clip and step recorded into two HIP graphs that replay alternately, with eager work between
    them; checked after every replay against an eager twin."""
    gen = torch.Generator(device=dev).manual_seed(9)
    make = lambda: [torch.randn(s, device=dev, generator=torch.Generator(device=dev).manual_seed(1))  # noqa: E731
                    .requires_grad_() for s in ((300, 7), (64,), (9001,))]
    ours, twin = make(), make()
    opt, ref = optim.Adam(ours, lr=3e-3), optim.Adam(twin, lr=3e-3)
    for p, q in zip(ours, twin):
        p.grad, q.grad = torch.empty_like(p), torch.empty_like(q)
    side = torch.cuda.Stream()
    graphs, norms = [], []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.clip_grad_norm_(ours, 1.0)
    torch.cuda.synchronize()
    for fn in (lambda: optim.clip_grad_norm_(ours, 0.5), lambda: opt.step(max_norm=0.25)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            norms.append(fn())
        graphs.append(g)
    for it in range(4):
        for p, q in zip(ours, twin):
            new = torch.randn(p.shape, device=dev, generator=gen)
            p.grad.copy_(new)
            q.grad.copy_(new)
        graphs[0].replay()
        want = optim.clip_grad_norm_(twin, 0.5)
        torch.cuda.synchronize()
        assert torch.equal(norms[0], want)
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(ours, twin))
        graphs[1].replay()
        want = ref.step(max_norm=0.25)
        torch.cuda.synchronize()
        assert torch.equal(norms[1], want)
        assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(ours, twin))
        assert all(float(opt.state[p]["step"]) == it + 1 for p in ours)


def test_clip_on_another_stream(optim, dev):
    params = _params(dev, [(5000,), (300, 31)], [F32], 8)
    before = [p.grad.clone() for p in params]
    want = _norm64(before, 2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = optim.clip_grad_norm_(params, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    _check_clipped(before, [p.grad for p in params], 0.1 / (want + 1e-6))


def _stepped(optim, shapes, change, clipped):
    """Two steps with `change(optimizer, parameters)` between them; the parameters by name."""
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(31)
    params = [torch.randn(s, device=dev, generator=gen).requires_grad_() for s in shapes]
    opt = optim.Adam([dict(params=params[:2]), dict(params=params[2:], lr=3e-3)], lr=1e-2)
    for it in range(2):
        for p in params:
            p.grad = torch.randn(p.shape, device=dev, generator=gen)
        if it == 1:
            change(opt, params)
        opt.step(max_norm=math.inf) if clipped else opt.step()
    return params, opt


def _replace_state(opt, params):
    p = params[1]
    opt.state[p] = {"step": torch.full((), 5.0, device=p.device),
                    "exp_avg": torch.full_like(p, 0.5).detach(),
                    "exp_avg_sq": torch.full_like(p, 0.25).detach()}


def _reorder_parameters(opt, params):
    for group in opt.param_groups:
        group["params"].reverse()


def _move_between_groups(opt, params):
    opt.param_groups[1]["params"].insert(0, opt.param_groups[0]["params"].pop(0))


def _reorder_states(opt, params):
    opt.state[params[0]] = opt.state.pop(params[0])


def _no_gradient(opt, params):
    params[0].grad = params[3].grad = None


@pytest.mark.parametrize("change", [
    _replace_state, _reorder_parameters, _move_between_groups, _reorder_states, _no_gradient])
def test_clipped_adam_finds_the_states_that_step_finds(optim, dev, change):
    """Whatever was done to the state and the groups between two steps: with a bound that clips
    nothing (a factor of exactly 1) the clipped step updates the same moments as step().  Both compute
    the same formula in float32; step() evaluates 1 - 0.999^t in float32, off by up to 6e-5 of itself
    at t = 1 and less later, half of that under the root: two moves of at most 3.2 lr = 0.032 differ by
    less than 2 * 0.032 * 4e-5, the moments by a few roundings."""
    shapes = [(40, 3), (40, 3), (40, 3), (7,), (40, 3)]
    ours, opt = _stepped(optim, shapes, change, True)
    ref, twin = _stepped(optim, shapes, change, False)
    for p, r in zip(ours, ref):
        assert float((p.detach() - r.detach()).abs().max()) <= 2 * 0.032 * 4e-5 + 2.0 ** -20
        # (1 - beta from float32 betas: off by 2^-25 / 0.1 and by 2^-25 / 0.001, below 2^-15)
        for key, part in (("exp_avg", 2.0 ** -20), ("exp_avg_sq", 2.0 ** -15), ("step", 0.0)):
            a, b = opt.state[p][key], twin.state[r][key]
            assert float((a - b).abs().max()) <= part * float(b.abs().max())


def test_clipped_adam_refuses_a_parameter_without_state(optim, dev):
    ours, opt = _stepped(optim, [(8,), (8,), (8,)], lambda *_: None, True)
    kept = [p.detach().clone() for p in ours]
    stranger = torch.zeros(8, device=dev, requires_grad=True)
    stranger.grad = torch.ones(8, device=dev)
    opt.param_groups[0]["params"][1] = stranger
    for step in (lambda: opt.step(max_norm=1.0), opt.step):
        with pytest.raises(KeyError):
            step()
    assert all(torch.equal(p.detach(), k) for p, k in zip(ours, kept))
    assert float(stranger.detach().abs().sum()) == 0.0


def test_clipped_adam_with_more_groups_than_a_launch_takes(optim, dev):
    """Twenty groups, each with hyperparameters of its own (a launch holds eight), first step: a move of
    at most lr (a factor of sqrt(1 - b2) / (1 - b1) more for the moments' weights) in under ten float32
    operations, and the rounding of p."""
    gen = torch.Generator(device=dev).manual_seed(61)
    ours = [torch.randn(33 + i, device=dev, generator=gen).requires_grad_() for i in range(40)]
    hyper = [dict(lr=1e-3 * (i + 1), betas=(0.9 - 0.01 * i, 0.999 - 0.01 * i), eps=1e-8,
                  weight_decay=1e-3 * (i % 3)) for i in range(20)]
    opt = optim.Adam([dict(params=ours[2 * i:2 * i + 2], **h) for i, h in enumerate(hyper)])
    for p in ours:
        p.grad = torch.randn(p.shape, device=dev, generator=gen)
    start = [p.detach().double() for p in ours]
    want = _norm64([p.grad for p in ours], 2.0)
    norm = opt.step(max_norm=0.5 * want)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    coef = 0.5 * want / (want + 1e-6)
    for j, (p, s) in enumerate(zip(ours, start)):
        h = hyper[j // 2]
        zero = torch.zeros_like(s)
        new, m, v = _adam64(s, p.grad.double(), zero, zero, 1, coef, h["lr"], *h["betas"], h["eps"],
                            h["weight_decay"])
        tol = 16 * 2.0 ** -24 * h["lr"] * 3.2 + 2.0 ** -24 * new.abs()
        assert bool(((p.detach().double() - new).abs() <= tol).all())
        assert bool(((opt.state[p]["exp_avg"].double() - m).abs() <= 2.0 ** -21 * m.abs()).all())
        assert bool(((opt.state[p]["exp_avg_sq"].double() - v).abs() <= 2.0 ** -21 * v.abs()).all())
