"""train_step on what it took before the decoder knew fused operators: any module that returns logits,
with or without a `cfg`, wrapped or not, and any optimizer with step() and zero_grad()."""

from types import SimpleNamespace

import pytest
import torch
from torch import nn


class Bigram(nn.Module):
    def __init__(self, cfg=None):
        super().__init__()
        self.table = nn.Embedding(32, 32)
        if cfg is not None:
            self.cfg = cfg

    def forward(self, tokens):
        return self.table(tokens)


class Wrapped(nn.Module):
    def __init__(self, module):
        super().__init__()
        self.module = module

    def forward(self, tokens):
        return self.module(tokens)


class PlainSgd:
    def __init__(self, params):
        self.params = list(params)

    @torch.no_grad()
    def step(self):
        for p in self.params:
            p -= 0.1 * p.grad

    def zero_grad(self):
        for p in self.params:
            p.grad = None


@pytest.mark.parametrize("cfg", [None, SimpleNamespace(vocab=32),
                                 SimpleNamespace(fused=True)], ids=["no cfg", "another cfg", "fused"])
@pytest.mark.parametrize("wrap", [False, True])
@pytest.mark.parametrize("own_optimizer", [False, True])
def test_any_module_and_optimizer(cfg, wrap, own_optimizer):
    import luciole_train as LT
    torch.manual_seed(0)
    model = Bigram(cfg)
    before = model.table.weight.detach().clone()
    opt = PlainSgd(model.parameters()) if own_optimizer else \
        LT.MasterWeightAdamW(list(model.parameters()), lr=1e-2)
    tok = torch.randint(0, 32, (2, 9))
    loss = LT.train_step(Wrapped(model) if wrap else model, opt, tok[:, :-1], tok[:, 1:])
    want = nn.functional.cross_entropy(before[tok[:, :-1]].view(-1, 32), tok[:, 1:].reshape(-1))
    assert torch.allclose(loss, want) and not torch.equal(model.table.weight, before)
