"""AMD.FUSED_BLOCKS as a user turns it on: what the blocks' modules carry keeps running, and the models and trainers built from a config use it."""
import copy

import pytest
import torch
from torch import nn

from coin_amd import kernels as K
from coin_amd.modeling.swin import SwinBlock
from coin_amd.modeling.text_encoder import ResidualAttentionBlock

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def launches(monkeypatch):
    """How often the fused operators' forward kernels were called, by name."""
    seen = {}
    for name in ("attention_fwd", "residual_norm_fwd", "linear_fwd"):
        def wrap(*a, _f=getattr(K, name), _n=name, **k):
            seen[_n] = seen.get(_n, 0) + 1
            return _f(*a, **k)
        monkeypatch.setattr(K, name, wrap)
    return seen


def blocks():
    torch.manual_seed(0)
    for blk, x, names in ((ResidualAttentionBlock(64, 2, fused=True), torch.randn(3, 20, 64), ("ln_1", "attn", "ln_2")),
                          (SwinBlock(96, 3, 7, 3, fused=True), torch.randn(2, 17, 24, 96), ("norm1", "norm2"))):
        for p in blk.parameters():
            nn.init.normal_(p, std=0.1) if p.dim() > 1 else nn.init.normal_(p, mean=float(p.detach().mean()), std=0.1)
        yield blk.to(DEV), x.to(DEV), names


def test_hooks_on_a_fused_blocks_modules_run(launches):
    for blk, x, names in blocks():
        plain = copy.deepcopy(blk)
        plain.fused = False
        want = plain(x)
        for name in names:
            got = []
            handles = [blk.get_submodule(name).register_forward_hook(lambda m, i, o: got.append(o)),
                       blk.get_submodule(name).register_forward_pre_hook(lambda m, i: got.append(i[0]))]
            launches.clear()
            assert torch.equal(blk(x), want) and len(got) == 2 and not launches, name
            for h in handles:
                h.remove()
        double = blk.get_submodule(names[0]).register_forward_hook(lambda m, i, o: 2 * o)    # one that changes the result
        plain.get_submodule(names[0]).register_forward_hook(lambda m, i, o: 2 * o)
        assert torch.equal(blk(x), plain(x)) and not torch.equal(blk(x), want)
        double.remove()
        xg, grads = x.clone().requires_grad_(), []
        h = blk.get_submodule(names[-1]).register_full_backward_hook(lambda m, gi, go: grads.append(go[0]))
        blk(xg).sum().backward()
        assert len(grads) == 1 and grads[0].abs().sum() > 0
        h.remove()
        h = nn.modules.module.register_module_forward_hook(lambda m, i, o: got.append(m))
        got.clear()
        blk(x)
        h.remove()
        assert all(any(m is blk.get_submodule(n) for m in got) for n in names)
        launches.clear()
        blk(x)
        assert launches, "without hooks the block is fused again"


def test_a_replaced_norm_is_called(launches):
    class Twice(nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    for blk, x, names in blocks():
        for other in (nn.Identity(), Twice(x.shape[-1]).to(DEV)):
            b = copy.deepcopy(blk)
            setattr(b, names[0], other)
            plain = copy.deepcopy(b)
            plain.fused = False
            launches.clear()
            assert torch.equal(b(x), plain(x)) and not launches
