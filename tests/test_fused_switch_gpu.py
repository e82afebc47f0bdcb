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


def config(path, extra):
    import os

    from coin_amd.config import get_cfg

    cfg = get_cfg()
    cfg.merge_from_file(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs", "coin", path))
    cfg.merge_from_list(["MODEL.DEVICE", DEV, "AMD.TEXT_TEMPLATES", 2, "AMD.SYNTHETIC.NUM_IMAGES", 2, "SOLVER.IMG_PER_BATCH_UNLABEL", 2,
                         "AMD.SYNTHETIC.HEIGHT", 256, "AMD.SYNTHETIC.WIDTH", 384] + extra)
    return cfg


def seeded(cls, cfg):
    import random

    import numpy as np

    torch.manual_seed(7)
    np.random.seed(7)
    random.seed(7)
    tr = cls(cfg)
    torch.manual_seed(8)
    return tr


@pytest.mark.parametrize("graph", [False, True])
def test_pretrain_steps_with_the_switch_on(launches, graph):
    """The prompt-learning text encoder inside PRETrainer, float32: the first step's losses are those of the plain blocks."""
    from coin_amd.engine import PRETrainer

    recs = {}
    for fused in (False, True):
        tr = seeded(PRETrainer, config("PRETRAINS/CLIPDET_synthetic.yaml", ["AMD.COMPUTE_DTYPE", "fp32", "AMD.TEXT_GRAPH", graph, "AMD.FUSED_BLOCKS", fused]))
        prompts = {n: p for n, p in tr.model.named_parameters() if n.endswith("embedding_tmp") or n.endswith("add_in_embedding")}
        before = {n: p.detach().clone() for n, p in prompts.items() if p.requires_grad}
        launches.clear()
        recs[fused] = [{k: float(v) for k, v in tr.run_step().items()} for _ in range(2)]
        assert bool(launches) == fused and (not fused or len(launches) == 3), launches
        assert before and any(not torch.equal(prompts[n].detach(), b) for n, b in before.items())
        assert all(v == v and abs(v) < float("inf") for r in recs[fused] for v in r.values()), recs
    for k, v in recs[False][0].items():
        # text features of two float32 evaluations agree to 1e-5 or so, their cosines are scaled by 100 before the losses
        assert abs(recs[True][0][k] - v) <= 5e-3 * max(1.0, abs(v)), (k, recs)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_coin_steps_of_the_swin_student_with_the_switch_on(launches, dtype):
    """A step of the Swin student with its teacher and the text encoder on the fused blocks: finite losses, and the blocks' parameters move
    and all have gradients."""
    from coin_amd.engine import CoinTrainer

    tr = seeded(CoinTrainer, config("FPN/targetdet_swint_fpn_synthetic.yaml", ["AMD.COMPUTE_DTYPE", dtype, "AMD.FUSED_BLOCKS", True, "CLOUD.BURN_UP_STEP", 10 ** 6,
                                                                                "CLOUD.PROTOTYPE_UPDATE_START", 0]))
    blocks_ = {n: m for n, m in tr.model.backbone.bottom_up.named_modules() if isinstance(m, SwinBlock)}
    assert blocks_ and all(m.fused for m in blocks_.values())
    before = {n: p.detach().clone() for n, p in tr.model.backbone.bottom_up.named_parameters() if "stages.2.1" in n}
    launches.clear()
    recs = [{k: float(v) for k, v in tr.run_step().items()} for _ in range(2)]
    assert len(launches) == 3 and all(v == v and abs(v) < float("inf") for r in recs for v in r.values()), (launches, recs)
    moved = [n for n, p in tr.model.backbone.bottom_up.named_parameters() if n in before and not torch.equal(p.detach(), before[n])]
    for part in ("norm1.bias", "norm2.bias", "qkv.weight", "proj.bias", "fc1.weight", "fc2.weight", "relative_position_bias_table"):
        assert any(part in n for n in moved), (part, moved)     # (a warm-up step is less than half a step of a norm's weight of 1)
    grads = {n: p.grad for n, p in tr.model.backbone.bottom_up.named_parameters() if n in before}
    assert all(g is not None and bool(g.isfinite().all()) and bool(g.any()) for g in grads.values()), grads.keys()


def test_swin_features_with_the_switch_on_are_the_plain_ones():
    from coin_amd.modeling import build_model

    feats = []
    img = torch.randint(0, 256, (3, 250, 331), dtype=torch.uint8, generator=torch.Generator().manual_seed(5)).to(DEV)
    state = None
    for fused in (False, True):
        torch.manual_seed(11)
        m = build_model(config("FPN/targetdet_swint_fpn_synthetic.yaml", ["AMD.COMPUTE_DTYPE", "fp32", "AMD.FUSED_BLOCKS", fused]))
        m = (m[0] if isinstance(m, (tuple, list)) else m).to(DEV).eval()
        state = state or m.state_dict()
        m.load_state_dict(state)
        with torch.no_grad():
            feats.append(m.backbone(m.preprocess_image([{"image": img}]).tensor))
    for k in feats[0]:
        a, b = (f[k].double() for f in feats)
        # twelve blocks, each four products of up to 4 * 768 terms and two norms in float32 on either side
        assert float((a - b).norm() / b.norm()) < 1e-4, k
