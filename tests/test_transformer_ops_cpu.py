"""The transformer-block entry points' refusals, which need no device: bad arguments come back before anything is launched."""
import ctypes
import os

import pytest
import torch

from coin_amd import _lib
from coin_amd import layers as L
from coin_amd._lib import CoinHipError

X = ctypes.c_void_p(0x10000)      # a non-NULL, 16-byte-aligned address that is never dereferenced
ODD = ctypes.c_void_p(0x10008)
S = (ctypes.c_int64 * 3)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


def attn(lib, q=X, qs=(64 * 4 * 7, 64 * 4, 64), ks=(64 * 4 * 9, 64 * 4, 64), k=X, b=2, lq=7, lk=9, hq=4, hkv=4, d=64, scale=0.125, dt=1, ws=None, n=0):
    return lib.coin_attention_fwd(q, S(*qs), k, S(*ks), X, S(*ks), X, S(64 * 4 * 7, 64 * 4, 64), None, None, None, b, lq, lk, hq, hkv, d, 0, scale, dt, ws, n, None)


def test_attention_refusals(lib):
    assert attn(lib, hq=3, hkv=2) == -2 and attn(lib, d=136) == -2 and attn(lib, d=12) == -2 and attn(lib, d=0) == -2
    assert attn(lib, dt=2) == -1 and attn(lib, b=-1) == -1 and attn(lib, hkv=0) == -1
    assert attn(lib, scale=0.0) == -1 and attn(lib, scale=-1.0) == -1 and attn(lib, scale=float("nan")) == -1 and attn(lib, scale=float("inf")) == -1
    assert attn(lib, q=None) == -1 and attn(lib, k=None) == -1
    assert attn(lib, q=ODD) == -3 and attn(lib, qs=(64 * 4 * 7, 64 * 4 + 1, 64)) == -3 and attn(lib, ks=(64 * 4 * 9, -64 * 4, 64)) == -3
    assert attn(lib, ks=(1 << 40, 1 << 24, 64)) == -2              # a staged tile would pass 32-bit offsets
    assert attn(lib, b=0) == 0 and attn(lib, lq=0) == 0             # nothing to do
    # few rows over a long cache are split: a workspace of that size, aligned, or nothing
    need = lib.coin_attention_workspace_bytes(1, 1, 4096, 4, 4, 64, 1, 0)
    assert need > 0 and lib.coin_attention_workspace_bytes(64, 4096, 4096, 8, 8, 64, 1, 0) == 0
    assert attn(lib, b=1, lq=1, lk=4096) == -1 and attn(lib, b=1, lq=1, lk=4096, ws=X, n=need - 1) == -1 and attn(lib, b=1, lq=1, lk=4096, ws=ODD, n=need) == -3
    assert lib.coin_attention_workspace_bytes(1, 1, 4096, 3, 2, 64, 1, 0) == 0
    z = S(0, 0, 0)
    assert lib.coin_attention_bwd(X, z, X, z, X, z, X, z, X, X, z, None, None, X, z, X, z, X, z, 1, 4, 4, 1, 1, 64, 0, 1.0, 1, X, 1 << 20, None) == -1   # no lse
    assert lib.coin_attention_bwd(X, z, X, z, X, z, X, z, None, X, z, X, None, X, z, X, z, X, z, 1, 4, 4, 1, 1, 64, 0, 1.0, 1, X, 1 << 20, None) == -1   # no residue
    assert lib.coin_attention_bwd(X, z, X, z, X, z, X, z, X, X, z, X, None, X, z, X, z, X, z, 1, 4, 4, 1, 1, 64, 0, 1.0, 1, None, 0, None) == -1        # no workspace


def test_workspace_queries_take_empty_shapes(lib):
    for b in (0, 1, 3):
        for lq in (0, 1, 5000):
            for lk in (0, 1, 5000):
                for back in (0, 1):
                    n = lib.coin_attention_workspace_bytes(b, lq, lk, 4, 2, 64, 1, back)
                    assert (n == 0) if b == 0 else n >= 0
    assert lib.coin_linear_workspace_bytes(0, 8, 8, 1, 0) == 0 and lib.coin_linear_workspace_bytes(0, 8, 8, 0, 1) == 0
    assert lib.coin_linear_workspace_bytes(1, 1, 1, 1, 1) > 0 and lib.coin_residual_norm_bwd_workspace_bytes(1, 1) > 0


def norm(lib, x=X, y=X, gate=None, group=8, post=0, pre=1, r=X, h=X, stats=None, m=8, d=16, ts=0, tb=0, tg=0):
    return lib.coin_residual_norm_fwd(x, y, gate, group, None, None, post, 1e-5, None, None, pre, 1e-5, 0, 1.0, r, h, stats, m, d, ts, tb, tg, None)


def test_residual_norm_refusals(lib):
    assert norm(lib, x=None) == -1 and norm(lib, h=None) == -1 and norm(lib, r=None) == -1 and norm(lib, y=None, pre=0) == -1
    assert norm(lib, y=None, gate=X) == -1 and norm(lib, y=None, post=1) == -1
    assert norm(lib, d=8193) == -2 and norm(lib, ts=1, tb=0) == -2 and norm(lib, gate=X, group=3) == -2
    assert norm(lib, group=0) == -1 and norm(lib, ts=5) == -1 and norm(lib, gate=X, tg=7) == -1 and norm(lib, d=0) == -1
    assert norm(lib, stats=ODD) == -3 and norm(lib, m=0) == 0
    n = lib.coin_residual_norm_bwd_workspace_bytes(8, 16)
    bwd = lambda dr=X, dh=X, dgate=None, dpw=None, dnw=None, ws=X, nb=n, m=8, post=0: lib.coin_residual_norm_bwd(  # noqa: E731
        X, X, None, 8, None, None, post, None, 1, 0, 1.0, X, dr, dh, X, X, dgate, dpw, None, dnw, None, m, 16, 0, 0, 0, ws, nb, None)
    assert n > 0 and bwd(dr=None, dh=None) == -1 and bwd(dgate=X) == -1 and bwd(dpw=X) == -1 and bwd(dh=None, dnw=X) == -1 and bwd(m=0) == -1
    assert bwd(dnw=X, ws=None) == -1 and bwd(dnw=X, nb=n - 1) == -1 and bwd(dnw=X, ws=ODD) == -3
    assert lib.coin_residual_norm_bwd_workspace_bytes(0, 16) == 0 and lib.coin_residual_norm_bwd_workspace_bytes(8, 9000) == 0


def test_linear_refusals(lib):
    fwd = lambda x=X, ldx=64, w=X, ldw=64, act=0, y=X, ldy=32, ty=1, m=8, n=32, k=64, dt=1, ws=None, nb=0, bias=None, tbias=0: lib.coin_linear_fwd(  # noqa: E731
        x, ldx, w, ldw, bias, tbias, act, None, 0, y, ldy, ty, None, 0, m, n, k, dt, ws, nb, None)
    assert fwd(act=1) == -1 and fwd(act=9) == -1 and fwd(y=None) == -1 and fwd(ldy=31) == -1 and fwd(dt=0, ty=1) == -1 and fwd(bias=X, tbias=4) == -1
    assert fwd(x=None) == -1 and fwd(x=ODD) == -3 and fwd(ldx=60) == -3 and fwd(ldw=56) == -3 and fwd(k=65) == -3
    assert fwd(ldx=1 << 24) == -2 and fwd(n=(1 << 24) + 8) == -2 and fwd(m=0) == 0 and fwd(k=0) == -1
    need = lib.coin_linear_workspace_bytes(4, 64, 8192, 1, 0)
    assert need > 0 and fwd(m=4, n=64, ldy=64, k=8192, ldx=8192, ldw=8192) == -1
    assert fwd(m=4, n=64, ldy=64, k=8192, ldx=8192, ldw=8192, ws=X, nb=need - 1) == -1 and fwd(m=4, n=64, ldy=64, k=8192, ldx=8192, ldw=8192, ws=ODD, nb=need) == -3
    full = lib.coin_linear_workspace_bytes(8, 32, 64, 1, 2)
    bwd = lambda dy=X, ldy=32, ty=1, slope=None, lds=0, x=X, ldx=64, w=X, ldw=64, dx=None, lddx=64, dw=None, lddw=64, tw=0, db=None, tb=0, m=8, n=32, dt=1, ws=X, nb=full: (  # noqa: E731
        lib.coin_linear_bwd(dy, ldy, ty, slope, lds, x, ldx, w, ldw, dx, lddx, dw, lddw, tw, db, tb, m, n, 64, dt, ws, nb, None))
    assert full > lib.coin_linear_workspace_bytes(8, 32, 64, 1, 1) > 0
    assert bwd() == -1 and bwd(dy=None, dx=X) == -1 and bwd(dx=X, m=0) == -1 and bwd(dx=X, ldy=31) == -1 and bwd(dx=X, slope=X, lds=31) == -1
    assert bwd(dx=X, lddx=63) == -1 and bwd(dw=X, lddw=63) == -1 and bwd(db=X, tb=3) == -1 and bwd(dx=X, ty=0, dt=0, ws=None) == -1
    assert bwd(dw=X, tw=1, dt=0, ty=0) == -1 and bwd(dx=X, dt=0, ty=1) == -1             # a float32 layer has float32 gradients
    assert bwd(dx=X, w=None) == -1 and bwd(dx=X, w=ODD) == -3 and bwd(dw=X, ldx=60) == -3 and bwd(dw=X, x=None) == -1
    assert bwd(dx=X, slope=X, lds=32, nb=full - 1) == -1 and bwd(dx=X, ws=ODD) == -3 and bwd(db=X, ws=None) == -1
    assert lib.coin_pad_rows(X, 5, X, 12, 4, 5, 1, None) == -2 and lib.coin_pad_rows(X, 5, X, 4, 4, 5, 1, None) == -1 and lib.coin_pad_rows(X, 5, X, 8, 0, 5, 1, None) == 0


def test_there_is_no_cpu_path():
    t = torch.zeros(1, 2, 2, 64)
    for f in (lambda: L.attention(t, t, t), lambda: L.attention_qkv(torch.zeros(1, 2, 192), 1), lambda: L.fused_linear(torch.zeros(2, 8), torch.zeros(4, 8)),
              lambda: L.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))):
        with pytest.raises(CoinHipError):
            f()
