"""Plain 64-bit forms of the operators next to the decode step, input builders and the bounds their
results are held to.  Test infrastructure only."""
from __future__ import annotations

import math

import torch

DEV = "cuda:0"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def pack_k(K, Lmax, fill=0.0):
    """[B,H,L,Dh] -> K cache [B,H,Dh/x,Lmax,x], slots behind L hold `fill`."""
    B, H, L, Dh = K.shape
    x = 16 // K.element_size()
    kc = torch.full((B, H, Dh // x, Lmax, x), fill, dtype=K.dtype, device=K.device)
    kc[:, :, :, :L] = K.view(B, H, L, Dh // x, x).permute(0, 1, 3, 2, 4)
    return kc


def unpack_k(kc):
    B, H, nch, L, x = kc.shape
    return kc.permute(0, 1, 3, 2, 4).reshape(B, H, L, nch * x)


def pack_v(V, Lmax, fill=0.0):
    B, H, L, Dh = V.shape
    vc = torch.full((B, H, Lmax, Dh), fill, dtype=V.dtype, device=V.device)
    vc[:, :, :L] = V
    return vc


def random_parents(g, B, n, reach=5):
    return torch.stack([torch.tensor([max(-1, i - 1 - int(torch.randint(0, reach, (1,), generator=g))) for i in range(n)],
                                     dtype=torch.int32) for _ in range(B)])


def ancestors(parents, i):
    """Node i and its ancestors; a parent that is no earlier node stands for the root."""
    seen = []
    while 0 <= i:
        seen.append(i)
        up = i - 1 if parents is None else int(parents[i])
        i = up if 0 <= up < i else -1
    return seen


def tree_reference(q, k, v, K, V, scale, t, parents=None, first_keys=None, lengths=None, counts=None):
    """float64 on the inputs' device: (out [B,Hq,n,Dh], size [B,Hq,n,Dh] = sum p |v|, logit spread,
    weights: list per sample of [H,G,n,first..length+n]).  K, V [B,H,>=t,Dh]; rows past a sample's count
    are zero.  Only what a node sees is ever touched."""
    B, Hq, n, Dh = q.shape
    H = k.shape[1]
    out, size = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    weights, bound = [], 0.0
    for b in range(B):
        length = t if lengths is None else min(max(int(lengths[b]), 0), t)
        first = 0 if first_keys is None else min(max(int(first_keys[b]), 0), length)
        count = n if counts is None else min(max(int(counts[b]), 0), n)
        par = None if parents is None else parents[b].tolist()
        w = torch.zeros(H, Hq // H, n, length - first + n, dtype=torch.float64, device=q.device)
        for i in range(count):
            mine = sorted(ancestors(par, i))
            kk = torch.cat([K[b, :, first:length].double(), k[b][:, mine].double()], 1)
            vv = torch.cat([V[b, :, first:length].double(), v[b][:, mine].double()], 1)
            for h in range(H):
                hq = slice(h * (Hq // H), (h + 1) * (Hq // H))
                z = q[b, hq, i].double() @ kk[h].t().contiguous() * scale
                bound = max(bound, float((q[b, hq, i].double().abs() @ kk[h].abs().t().contiguous()).nan_to_num(0, 0, 0).max()) * abs(scale))
                p = torch.softmax(z, -1)
                out[b, hq, i] = p @ vv[h]
                size[b, hq, i] = p @ vv[h].abs()
                w[h, :, i, : length - first] = p[:, : length - first]
                w[h, :, i, [length - first + j for j in mine]] = p[:, length - first :]
        weights.append(w)
    return out, size, bound, weights


def tree_tolerance(dtype, want, size, bound, keys, Dh):
    """Elementwise bound.  Half a step of the result's type; weights whose logits are off by the
    rounding of Dh products and of the exponent's argument, twice (numerator and sum); the two-part
    weights of the 16-bit types (2^-20, 2^-14); 2 fp32 additions a key in the sum over the keys."""
    u = 2.0 ** -24
    logit = bound * (Dh + 4) * u + 4 * u
    split = {torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -14, torch.float32: 0.0}[dtype]
    rel = 2 * logit + split + (2 * keys + 64) * u
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
    return torch.finfo(dtype).eps / 2 * want.abs() * (1 + 1e-3) + rel * size + tiny


def assert_close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and not bool((got.isinf() & ~inf).any()), f"{what}: infinities differ"
    ok = ~(want.isnan() | inf)
    over = ((got - want).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: off by {float((got - want)[ok].abs().max())}, {float(over.max())} over its bound"


def evict_reference(w, length, first, keep, recent):
    """Slots that stay of one pair's weights (a list of floats)."""
    if length <= keep:
        return list(range(length))
    tail = length - recent

    def rank(j):
        if j >= tail:
            return (0, 0.0, j)
        if j < first:
            return (2, 0.0, j)
        return (1, math.inf if math.isnan(w[j]) else -w[j], j)      # NaN last of its tier, by slot

    # NaN ranks below every number, -inf included: its own tier between the real keys and padding.
    def full(j):
        a, x, s = rank(j)
        return (1.5, 0.0, s) if a == 1 and math.isnan(w[j]) else (a, x, s)

    return sorted(sorted(range(length), key=full)[:keep])
