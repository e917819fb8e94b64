"""CPU tests of the host side of the operators next to the decode step: what the C ABI refuses before any
launch, and what their workspaces and plans promise.  No kernel is launched here."""
import ctypes as C

import pytest

from fastforwardattention_amd import capi

P = C.c_void_p(0x100000)


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def pointers(*addresses):
    return (C.c_void_p * len(addresses))(*addresses)


def tokens(n=4, Hq=4, Dh=64, H=4, **kw):
    t = capi.TreeTokens()
    t.tokens, t.q_head_num = n, Hq
    for name, heads in (("q_stride", Hq), ("k_stride", H), ("v_stride", H), ("out_stride", Hq)):
        getattr(t, name)[:] = [n * heads * Dh, Dh, heads * Dh]
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def tree(lib, precision=16, B=2, H=4, Dh=64, Lmax=128, t=100, tok=None, q=P, k=P, v=P, kc=P, vc=P, out=P, ws=None, n_ws=0):
    tok = tokens() if tok is None else tok
    return lib.ffa_attention_tree(precision, B, H, Dh, Lmax, 0.125, t, C.byref(tok) if tok else None, q, k, v, kc, vc, out, ws, n_ws, None)


def test_tree_refusals(lib):
    assert tree(lib, precision=8) == capi.FFA_ERR_DTYPE
    assert tree(lib, Dh=96) == capi.FFA_ERR_HEAD_DIM
    assert tree(lib, B=0) == capi.FFA_ERR_SHAPE
    assert tree(lib, H=-1) == capi.FFA_ERR_SHAPE
    assert tree(lib, B=1 << 12, H=1 << 12) == capi.FFA_ERR_SHAPE
    assert tree(lib, Lmax=1 << 26) == capi.FFA_ERR_SHAPE
    assert tree(lib, t=-1) == capi.FFA_ERR_TIMESTEP
    assert tree(lib, t=128) == capi.FFA_ERR_TIMESTEP
    assert tree(lib, t=125) == capi.FFA_ERR_TREE                        # four tokens do not fit
    assert tree(lib, tok=tokens(n=0)) == capi.FFA_ERR_TREE
    assert tree(lib, t=0, tok=tokens(n=65)) == capi.FFA_ERR_TREE
    assert tree(lib, tok=tokens(Hq=6)) == capi.FFA_ERR_TREE
    assert tree(lib, tok=tokens(Hq=0)) == capi.FFA_ERR_TREE
    assert tree(lib, tok=False) == capi.FFA_ERR_NULL_POINTER
    for name in ("q", "k", "v", "kc", "vc", "out"):
        assert tree(lib, **{name: None}) == capi.FFA_ERR_NULL_POINTER
        assert tree(lib, **{name: C.c_void_p(0x100008)}) == capi.FFA_ERR_ALIGNMENT
    for name in ("parents", "first_keys", "lengths", "counts"):
        assert tree(lib, tok=tokens(**{name: 0x100002})) == capi.FFA_ERR_ALIGNMENT
    for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
        bad = tokens()
        getattr(bad, name)[1] = 68
        assert tree(lib, tok=bad) == capi.FFA_ERR_TREE
    for name in ("k_stride", "v_stride"):
        for step in (-64, (1 << 26) // 2):
            bad = tokens()
            getattr(bad, name)[2] = step
            assert tree(lib, tok=bad) == capi.FFA_ERR_TREE
    # few pairs, a long cache: pieces, and so a workspace
    need = lib.ffa_tree_workspace_bytes(16, 1, 1, 1, 64, 4, 5000)
    one = tokens(Hq=1, H=1)
    assert need > 0
    assert tree(lib, B=1, H=1, Lmax=6000, t=5000, tok=one) == capi.FFA_ERR_WORKSPACE
    assert tree(lib, B=1, H=1, Lmax=6000, t=5000, tok=one, ws=P, n_ws=need - 1) == capi.FFA_ERR_WORKSPACE
    assert tree(lib, B=1, H=1, Lmax=6000, t=5000, tok=one, ws=C.c_void_p(0x100004), n_ws=need) == capi.FFA_ERR_ALIGNMENT


def test_workspace_grows_with_the_step(lib):
    for precision in (16, 32, capi.FFA_PRECISION_BF16):
        for B, H, Hq, Dh, n in ((1, 1, 1, 64, 1), (1, 4, 32, 128, 64), (2, 32, 32, 256, 7), (16, 32, 32, 80, 64)):
            last = last_w = 0
            for t in (0, 1, 100, 255, 256, 257, 1000, 4096, 5000, 33000, 200000):
                now, now_w = lib.ffa_tree_workspace_bytes(precision, B, H, Hq, Dh, n, t), lib.ffa_weights_workspace_bytes(precision, B, H, Hq, Dh, t)
                assert now >= last and now_w >= last_w and now % 256 == 0 and now_w >= 4 * B * Hq * (t + 1)
                last, last_w = now, now_w
    for bad in ((8, 1, 1, 1, 64, 1, 1), (16, 0, 1, 1, 64, 1, 1), (16, 1, 2, 3, 64, 1, 1), (16, 1, 1, 1, 96, 1, 1), (16, 1, 1, 1, 64, 65, 1), (16, 1, 1, 1, 64, 1, -1)):
        assert lib.ffa_tree_workspace_bytes(*bad) == 0


def test_weights_refusals(lib):
    def call(precision=16, B=2, H=4, Hq=8, Dh=64, Lmax=128, t=100, q=P, kw=P, first=None, lengths=None, ws=None, n_ws=0):
        return lib.ffa_attention_weights(precision, B, H, Hq, Dh, Lmax, 0.125, t, q, P, P, P, P, P, kw, first, lengths, ws, n_ws, None)
    assert call(precision=0) == capi.FFA_ERR_DTYPE
    assert call(Dh=32) == capi.FFA_ERR_HEAD_DIM
    assert call(t=128) == capi.FFA_ERR_TIMESTEP
    assert call(Hq=6) == capi.FFA_ERR_TREE
    assert call(q=None) == capi.FFA_ERR_NULL_POINTER
    assert call(kw=None) == capi.FFA_ERR_NULL_POINTER
    assert call(kw=C.c_void_p(0x100002)) == capi.FFA_ERR_ALIGNMENT
    assert call(first=C.c_void_p(0x100001)) == capi.FFA_ERR_ALIGNMENT
    assert call() == capi.FFA_ERR_WORKSPACE


def test_commit_refusals(lib):
    def call(precision=16, k=pointers(0x100000), v=pointers(0x200000), n=1, B=2, H=4, Dh=64, Lmax=128, t=100, path=P, m=4, acc=P, lengths=None):
        return lib.ffa_commit_tree(precision, n, k, v, B, H, Dh, Lmax, t, path, m, acc, lengths, None)
    assert call(precision=1) == capi.FFA_ERR_DTYPE
    assert call(Dh=65) == capi.FFA_ERR_HEAD_DIM
    assert call(n=-1) == capi.FFA_ERR_SHAPE
    assert call(t=128) == capi.FFA_ERR_TIMESTEP
    assert call(m=0) == capi.FFA_ERR_TREE
    assert call(t=0, m=65) == capi.FFA_ERR_TREE
    assert call(t=125) == capi.FFA_ERR_TREE
    assert call(path=None) == capi.FFA_ERR_NULL_POINTER
    assert call(acc=None) == capi.FFA_ERR_NULL_POINTER
    assert call(k=None) == capi.FFA_ERR_NULL_POINTER
    assert call(k=pointers(None)) == capi.FFA_ERR_NULL_POINTER
    assert call(v=pointers(0x200008)) == capi.FFA_ERR_ALIGNMENT
    assert call(lengths=C.c_void_p(0x100002)) == capi.FFA_ERR_ALIGNMENT
    assert call(n=0) == capi.FFA_OK
    # 2 x 4 x 128 slots of 128 bytes: 128 KiB a buffer
    assert call(k=pointers(0x100000), v=pointers(0x110000)) == capi.FFA_ERR_OVERLAP
    assert call(n=2, k=pointers(0x100000, 0x100000), v=pointers(0x200000, 0x300000)) == capi.FFA_ERR_OVERLAP
    assert call(n=2, k=pointers(0x100000, 0x400000), v=pointers(0x200000, 0x11fff0)) == capi.FFA_ERR_OVERLAP


def test_evict_refusals(lib):
    """Two pairs of 64 slots: 16 KiB of K or V and 512 bytes of weights a cache."""
    M = 0x100000

    def call(precision=16, n=1, ks=(1 * M,), vs=(2 * M,), ws=(3 * M,), kd=(4 * M,), vd=(5 * M,), wd=(6 * M,), B=1, H=2, Dh=64, Ls=64, Ld=64,
             t=60, keep=30, recent=10, kept=7 * M):
        arrays = [None if x is None else pointers(*x) for x in (ks, vs, ws, kd, vd, wd)]
        return lib.ffa_evict(precision, n, *arrays, B, H, Dh, Ls, Ld, t, keep, recent, None, None, kept, None)
    assert call(precision=3) == capi.FFA_ERR_DTYPE
    assert call(Dh=48) == capi.FFA_ERR_HEAD_DIM
    assert call(Ld=0) == capi.FFA_ERR_SHAPE
    assert call(t=65) == capi.FFA_ERR_TIMESTEP
    assert call(keep=0) == capi.FFA_ERR_EVICT
    assert call(keep=65) == capi.FFA_ERR_EVICT
    assert call(recent=-1) == capi.FFA_ERR_EVICT
    assert call(recent=31) == capi.FFA_ERR_EVICT
    assert call(ks=None) == capi.FFA_ERR_NULL_POINTER
    assert call(kept=None) == capi.FFA_ERR_NULL_POINTER
    assert call(wd=(None,)) == capi.FFA_ERR_NULL_POINTER
    assert call(kd=(4 * M + 8,)) == capi.FFA_ERR_ALIGNMENT
    assert call(ws=(3 * M + 2,)) == capi.FFA_ERR_ALIGNMENT
    for bad in (dict(kd=(1 * M + 16,)), dict(kd=(2 * M,)), dict(vd=(1 * M,)), dict(vd=(4 * M,)), dict(wd=(3 * M + 4,)), dict(wd=(5 * M,)),
                dict(kept=4 * M + 64), dict(kd=(1 * M,), Ld=72),
                dict(n=2, ks=(1 * M, 8 * M), vs=(2 * M, 9 * M), ws=(3 * M, 10 * M), kd=(1 * M, 1 * M), vd=(2 * M, 9 * M), wd=(3 * M, 10 * M)),
                dict(n=2, ks=(1 * M, 8 * M), vs=(2 * M, 9 * M), ws=(3 * M, 10 * M), kd=(8 * M, 1 * M), vd=(2 * M, 9 * M), wd=(3 * M, 10 * M))):
        assert call(**bad) == capi.FFA_ERR_OVERLAP, bad
    assert call(n=0) == capi.FFA_OK


def test_extension_refuses_cpu_tensors():
    import torch
    from fastforwardattention_amd import FastForwardAttn as F
    kc, vc = torch.zeros(1, 2, 8, 16, 8, dtype=torch.float16), torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    x = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    w = torch.zeros(1, 2, 16)
    for call in (lambda: F.attention_tree(x, x, x, kc, vc, 1.0, 4), lambda: F.attention_weights(x[:, :, 0], x[:, :, 0], x[:, :, 0], kc, vc, 1.0, 4, w),
                 lambda: F.commit_tree([(kc, vc)], 4, torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)),
                 lambda: F.evict([(kc, vc)], [w], 10, 5, 1)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()
