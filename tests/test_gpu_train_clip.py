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


def _mini(model, optimizer, criterion, bound, steps=4):
    from torch_geometric_autoscale import train
    train.mini_train(model, _loader()[:steps], criterion, optimizer, 100, grad_norm=bound)


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
