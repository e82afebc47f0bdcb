"""AMD.FUSED_BLOCKS from a config to the blocks, and its having no effect without a device."""
import pytest
import torch

from cpu_shim import cpu_kernels
from test_fpn_cpu import _tiny_cfg

from coin_amd.modeling import build_model
from coin_amd.modeling.swin import SwinBlock
from coin_amd.modeling.text_encoder import ResidualAttentionBlock

SWIN = ["MODEL.SWIN.EMBED_DIM", 16, "MODEL.SWIN.DEPTHS", (2, 2, 2, 2), "MODEL.SWIN.NUM_HEADS", (1, 2, 4, 8)]


def models(fused):
    cfg = _tiny_cfg("targetdet_swint_fpn_synthetic.yaml", SWIN + ([] if fused is None else ["AMD.FUSED_BLOCKS", fused]))
    torch.manual_seed(0)
    m = build_model(cfg)
    return m if isinstance(m, (tuple, list)) else (m,)


@pytest.mark.parametrize("fused", [None, False, True])
def test_the_switch_reaches_every_block(fused):
    with cpu_kernels():
        kinds = {SwinBlock: 0, ResidualAttentionBlock: 0}
        for model in models(fused):
            for m in model.modules() if isinstance(model, torch.nn.Module) else ():
                if type(m) in kinds:
                    kinds[type(m)] += 1
                    assert m.fused is bool(fused)      # off where the config says nothing
        assert all(kinds.values()), kinds


def test_the_switch_changes_nothing_on_the_cpu():
    with cpu_kernels():
        a, b = (next(m for m in models(fused) if isinstance(m, torch.nn.Module)).eval() for fused in (False, True))
        assert list(a.state_dict()) == list(b.state_dict())
        b.load_state_dict(a.state_dict())
        img = torch.randint(0, 256, (3, 90, 120), dtype=torch.uint8, generator=torch.Generator().manual_seed(5))
        with torch.no_grad():
            fa, fb = (m.backbone(m.preprocess_image([{"image": img}]).tensor) for m in (a, b))
        assert set(fa) == set(fb) and all(torch.equal(fa[k], fb[k]) for k in fa)
