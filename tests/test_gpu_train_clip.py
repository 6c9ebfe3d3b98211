"""train.mini_train with gradient clipping and whatever model and optimizer it is given: the same
weights as a plain loop of backward pass, torch.nn.utils.clip_grad_norm_ and step."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


class Model(torch.nn.Module):
    """Two layers with mini_train's calling convention."""

    def __init__(self, dtype, sparse=False):
        super().__init__()
        torch.manual_seed(5)
        self.a = torch.nn.Embedding(50, 12, sparse=sparse)
        self.b = torch.nn.Linear(12, 4)
        self.to("cuda", dtype)
        self.device = torch.device("cuda", 0)

    def forward(self, x, adj_t, batch_size, n_id, offset, count, **kw):
        return {"out": self.b(self.a(x))}


def _loader():
    gen = torch.Generator().manual_seed(8)
    out = []
    for _ in range(4):
        x, y = torch.randint(0, 50, (20,), generator=gen), torch.randint(0, 4, (20,), generator=gen)
        adj = types.SimpleNamespace(to=lambda device: None)
        batch = types.SimpleNamespace(x=x, y=y, adj_t=adj, train_mask=torch.ones(20, dtype=torch.bool))
        out.append((batch, 20, torch.arange(20), None, None))
    return out


def _plain(model, optimizer, criterion, bound, each=lambda model: None, steps=4):
    for batch, *_ in _loader()[:steps]:
        optimizer.zero_grad()
        loss = criterion(model(batch.x.cuda(), None, 20, None, None, None)["out"], batch.y.cuda())
        loss.backward()
        each(model)
        torch.nn.utils.clip_grad_norm_(model.parameters(), bound)
        optimizer.step()


def _mini(model, optimizer, criterion, bound, steps=4):
    from torch_geometric_autoscale import train
    train.mini_train(model, _loader()[:steps], criterion, optimizer, 100, grad_norm=bound)


def _same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def test_float64_gradients_are_clipped():
    criterion = torch.nn.CrossEntropyLoss()
    ours, ref = Model(torch.float64), Model(torch.float64)
    start = [p.detach().clone() for p in ref.parameters()]
    _mini(ours, torch.optim.SGD(ours.parameters(), lr=0.5), criterion, 0.05)
    _plain(ref, torch.optim.SGD(ref.parameters(), lr=0.5), criterion, 0.05)
    assert _same(ours, ref)
    assert not any(torch.equal(p.detach(), s) for p, s in zip(ours.parameters(), start))


def test_a_tree_without_the_training_module_clips(monkeypatch):
    """The package runs without its compiled operator objects; so does the training loop."""
    from torch_geometric_autoscale import ops
    from torch_geometric_autoscale.optim import Adam
    monkeypatch.setattr(ops, "_train_ops", None)
    monkeypatch.setattr(ops, "TRAIN_OPS_PATH", "/nonexistent/_train_ops.so")
    criterion = torch.nn.CrossEntropyLoss()
    for make in (lambda m: Adam(m.parameters(), lr=1e-2),
                 lambda m: torch.optim.SGD(m.parameters(), lr=0.5)):
        ours, ref = Model(torch.float32), Model(torch.float32)
        _mini(ours, make(ours), criterion, 0.05)
        _plain(ref, make(ref), criterion, 0.05)
        assert _same(ours, ref)


def test_a_gradient_that_two_parameters_share():
    """It counts twice in the norm, and training goes on.  (What torch's clipping makes of the shared
    gradient itself is not determined: one launch scales it twice at once.)"""
    from torch_geometric_autoscale.optim import Adam
    criterion = torch.nn.CrossEntropyLoss()
    for make in (lambda m: Adam(m.parameters(), lr=1e-2),
                 lambda m: torch.optim.SGD(m.parameters(), lr=0.5)):
        ours, ref = Model(torch.float32), Model(torch.float32)
        for m in (ours, ref):
            m.c = torch.nn.Parameter(torch.ones_like(m.b.weight))
        hook = ours.b.weight.register_post_accumulate_grad_hook(
            lambda p: setattr(ours.c, "grad", p.grad))

        def share(m):
            m.c.grad = m.b.weight.grad
        _mini(ours, make(ours), criterion, 0.05, 1)
        _plain(ref, make(ref), criterion, 0.05, share, 1)
        hook.remove()
        assert torch.equal(ours.a.weight, ref.a.weight) and torch.equal(ours.b.bias, ref.b.bias)
        assert bool(ours.c.isfinite().all()) and not torch.equal(ours.c, torch.ones_like(ours.c))


def test_an_optimizer_with_a_step_of_its_own():
    """A step() that is not the package's is called as it is, behind the clipping."""
    from torch_geometric_autoscale.optim import Adam
    calls = []

    class Counting(Adam):
        def step(self):
            calls.append(float(sum(p.grad.square().sum() for g in self.param_groups
                                   for p in g["params"]).sqrt()))
            return super().step()
    criterion = torch.nn.CrossEntropyLoss()
    ours = Model(torch.float32)
    _mini(ours, Counting(ours.parameters(), lr=1e-2), criterion, 0.05)
    assert len(calls) == 4 and all(c <= 0.05 * (1 + 2.0 ** -20) for c in calls)
    # one wrapped on the object
    ours = Model(torch.float32)
    opt = Adam(ours.parameters(), lr=1e-2)
    inner = opt.step
    opt.step = lambda: calls.append(0.0) or inner()
    _mini(ours, opt, criterion, 0.05)
    assert len(calls) == 8


def test_clips_names_the_gradients_that_the_kernels_take():
    from torch_geometric_autoscale.optim import clips
    p, q = (torch.nn.Parameter(torch.zeros(6, device="cuda")) for _ in range(2))
    assert clips([]) and clips([p, q])
    p.grad, q.grad = torch.ones(6, device="cuda"), torch.ones(6, device="cuda")
    assert clips([p, q]) and clips(p)
    q.grad = p.grad
    assert not clips([p, q])
    d = torch.nn.Parameter(torch.zeros(6, device="cuda", dtype=torch.float64))
    d.grad = torch.ones_like(d)
    assert not clips([p, d])
    s = Model(torch.float32, sparse=True)
    s.a(torch.tensor([1, 2], device="cuda")).sum().backward()
    assert s.a.weight.grad.is_sparse and not clips(s.parameters())
    h = torch.nn.Parameter(torch.zeros(3))
    h.grad = torch.ones(3)
    assert not clips([h]) and not clips([p, h])
    e = [torch.nn.Parameter(torch.zeros(0, device="cuda")) for _ in range(2)]
    for t in e:
        t.grad = torch.zeros_like(t)
    assert clips(e)
