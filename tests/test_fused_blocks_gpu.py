"""The text encoder and the Swin block on the fused operators (AMD.FUSED_BLOCKS) against the same weights in float64."""
import copy

import pytest
import torch
import torch.nn.functional as F

from coin_amd.modeling.swin import SwinBlock
from coin_amd.modeling.text_encoder import CLIP_TEXT, ResidualAttentionBlock

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rel(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())


def block64(x, blk):
    """ResidualAttentionBlock in float64, written out."""
    ln = lambda t, m: F.layer_norm(t, (t.shape[-1],), m.weight.double(), m.bias.double(), m.eps)  # noqa: E731
    n, l, d = x.shape
    a = blk.attn
    q, k, v = F.linear(ln(x, blk.ln_1), a.in_proj_weight.double(), a.in_proj_bias.double()).view(n, l, 3, a.heads, d // a.heads).permute(2, 0, 3, 1, 4)
    s = q @ k.transpose(-1, -2) * (d // a.heads) ** -0.5
    s = s.masked_fill(torch.ones(l, l, device=x.device, dtype=torch.bool).triu(1), float("-inf"))
    o = (s.softmax(-1) @ v).transpose(1, 2).reshape(n, l, d)
    x = x + F.linear(o, a.out_proj.weight.double(), a.out_proj.bias.double())
    h = F.linear(ln(x, blk.ln_2), blk.mlp.c_fc.weight.double(), blk.mlp.c_fc.bias.double())
    return x + F.linear(h * torch.sigmoid(1.702 * h), blk.mlp.c_proj.weight.double(), blk.mlp.c_proj.bias.double())


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2.0 ** -5)])
def test_text_block_forward_and_gradients(dtype, tol):
    """tol, of the 2-norm: float32 sums of up to 512 terms a step (2^-24 each way); in bfloat16 about ten roundings of 2^-8 at most between an
    input and a result, independent of one another: half of their sum."""
    torch.manual_seed(0)
    blk = ResidualAttentionBlock(128, 2, fused=True).to(DEV)
    for p in blk.parameters():
        torch.nn.init.normal_(p, std=0.08) if p.dim() > 1 else torch.nn.init.normal_(p, mean=float(p.mean()), std=0.1)
    x = torch.randn(9, 77, 128, device=DEV).to(dtype).requires_grad_()
    dy = torch.randn(9, 77, 128, device=DEV).to(dtype)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        y = blk(x)
    assert y.dtype == dtype
    names, leaves = zip(*blk.named_parameters())
    got = torch.autograd.grad(y, (x,) + leaves, dy)
    x64 = x.detach().double().requires_grad_()
    y64 = block64(x64, blk)
    want = torch.autograd.grad(y64, (x64,) + leaves, dy.double())
    for n, a, b in zip(("y", "x") + names, (y,) + got, (y64,) + want):
        assert rel(a, b) < tol, (n, rel(a, b))


def text(fused, graph=False):
    torch.manual_seed(3)
    return CLIP_TEXT("RN50", ["car", "person", "bus", "backgroud"], embed_dim=32, context_length=24, vocab_size=64, width=64, heads=4, layers=3, n_templates=2,
                     graph=graph, fused=fused).to(DEV)


def test_text_encoder_fused_and_not_agree_and_share_their_state():
    a, b = text(False), text(True)
    assert list(a.state_dict()) == list(b.state_dict())
    b.load_state_dict(a.state_dict())
    outs = []
    for m in (a, b):
        o = m(True)
        outs.append((o,) + torch.autograd.grad(o, [m.encoder.embedding_tmp, m.encoder.add_in_embedding], torch.linspace(-1, 1, o.numel(), device=DEV).view_as(o)))
    for p, q in zip(*outs):
        # two float32 evaluations of three blocks: a few hundred roundings of 2^-24 each side
        assert rel(q, p) < 1e-4


def test_fused_text_encoder_replayed_from_its_graphs_is_the_eager_pass():
    """The captured forward and backward, replayed as the prompt vectors move, with eager passes of the same leaves between the replays."""
    m, e = text(True, graph=True), text(True)
    e.load_state_dict(m.state_dict())
    g = torch.linspace(-1, 1, 4 * 32, device=DEV).view(4, 32)
    leaves = lambda t: [t.encoder.embedding_tmp, t.encoder.add_in_embedding]  # noqa: E731
    for turn in range(4):
        with torch.no_grad():
            for p, q in zip(leaves(m), leaves(e)):
                p.add_(0.01 * turn)
                q.copy_(p)
        o = m(True)
        got = torch.autograd.grad(o, leaves(m), g)
        w = e(True)
        want = torch.autograd.grad(w, leaves(e), g)
        torch.cuda.synchronize()
        assert torch.equal(o, w) and all(torch.equal(a, b) for a, b in zip(got, want)), turn
    assert m.encoder._graphs and not m.encoder._graph_failed


@pytest.mark.parametrize("dim,heads,shift", [(96, 3, 0), (192, 6, 3)])
def test_fused_swin_block_agrees_with_the_plain_one(dim, heads, shift):
    """float32: against the unfused block's float64 run.  The map needs window padding and is not a multiple of anything."""
    torch.manual_seed(1)
    blk = SwinBlock(dim, heads, 7, shift, fused=True).to(DEV)
    for p in blk.parameters():
        torch.nn.init.normal_(p, std=0.06) if p.dim() > 1 else torch.nn.init.normal_(p, mean=float(p.mean()), std=0.1)
    ref = copy.deepcopy(blk).double()
    ref.fused = False
    x = torch.randn(2, 17, 24, dim, device=DEV, requires_grad=True)
    dy = torch.randn(2, 17, 24, dim, device=DEV)
    x64 = x.detach().double().requires_grad_()
    names, leaves = zip(*blk.named_parameters())
    y, y64 = blk(x), ref(x64)
    got = torch.autograd.grad(y, (x,) + leaves, dy)
    want = torch.autograd.grad(y64, (x64,) + tuple(ref.parameters()), dy.double())
    for n, a, b in zip(("y", "x") + names, (y,) + got, (y64,) + want):
        # the reference's window attention runs in float32: sums of 49 terms and of the map's 816 rows
        assert rel(a, b) < 2e-5, (n, rel(a, b))


def test_fused_swin_block_under_autocast():
    torch.manual_seed(1)
    blk = SwinBlock(96, 3, 7, 3, fused=True).to(DEV)
    ref = copy.deepcopy(blk)
    ref.fused = False
    x = torch.randn(2, 17, 24, 96, device=DEV, requires_grad=True)
    dy = torch.randn(2, 17, 24, 96, device=DEV)
    leaves, rleaves = tuple(blk.parameters()), tuple(ref.parameters())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, z = blk(x), ref(x)
    assert y.dtype == z.dtype == torch.float32
    for a, b in zip((y,) + torch.autograd.grad(y, (x,) + leaves, dy), (z,) + torch.autograd.grad(z, (x,) + rleaves, dy)):
        assert rel(a, b) < 2.0 ** -4    # ten roundings of 2^-8 at most on either side, independent
