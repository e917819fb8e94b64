"""GPU tests in which a few keys have all the weight, so that one key read from a wrong place, lost or counted twice
shows: at offsets beyond 32 bits, and at the ends of tiles, pieces, paddings and lengths."""
import math

import pytest
import torch

from tests.cache_ops_testlib import DEV, DT, pack_k, pack_v, unpack_k
from tests.test_gpu_cache_ops import FFA, NAN, ints

pytestmark = pytest.mark.gpu

HEAVY = 60.0


def plant(K, slots, g):
    """K [..., L, Dh] of small numbers, on any device: with q0 = HEAVY the scores of the heavy slots become HEAVY + 0..1,
    those of all others stay near 0, so that each of them has less than e^-50 of a heavy one's weight."""
    K[..., 0] = 0
    K[..., slots, 0] = 1 + torch.rand(len(slots), generator=g).to(K.device, K.dtype) / 64


def check(got, p, V, dtype, logit, label):
    """got [rows, Dh] against sum p V over the heavy keys (p [rows, m], V [m, Dh], 64 bits).  Bound: half a step of the
    result; scores off by `logit` (numerator and sum); the two 16-bit parts; m + 64 additions of 2^-24 (the light keys'
    weights are 2^20 e^-50 in all).  The test shows itself that a lost, doubled or swapped key is
    outside it."""
    u = 2.0 ** -24
    part = {torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -14, torch.float32: 0.0}[dtype]
    want, size = p @ V, p @ V.abs()
    m = p.shape[1]
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (2 * logit + part + (2 * m + 64) * u) * size + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{label}: {float((err / tol).max())} of its bound"
    assert bool((want.abs() > tol).any(1).all()), label + ": zeros would pass"
    # Without one key, or with its value replaced by that of another slot, some element is out of bounds.
    for r in range(p.shape[0]):
        change = p[r, :, None] * (V - want[r]) / (1 - p[r, :, None]).clamp(min=1e-9)
        assert m == 1 or bool((change.abs() > 2 * tol[r]).any(1).all()), label + ": a lost key would pass"


def logit_error(q, K, scale, Dh):
    return float((q.double().abs() @ K.double().abs().t().contiguous()).max()) * abs(scale) * (Dh + 4) * 2.0 ** -24 + 4 * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_heavy_keys_beyond_four_gigabytes(dtype):
    """Caches of more than 4 GiB; the last pair has heavy keys at both ends and in the middle.  Tree attention, commit, weight-summing step and eviction against its own slots."""
    print("heavy far", dtype, flush=True)
    B, H, Dh, t, n, dt = 2, 16, 128, 590_000, 5, DT[dtype]
    Lmax = t + 16
    g, gh = torch.Generator(device=DEV).manual_seed(90), torch.Generator().manual_seed(91)
    kc = torch.empty(B, H, Dh // 8, Lmax, 8, dtype=dt, device=DEV).normal_(0, 0.01, generator=g)
    vc = torch.empty(B, H, Lmax, Dh, dtype=dt, device=DEV).normal_(generator=g)
    assert kc.numel() * 2 > 4 << 30
    # The last pair lies behind 2^32 bytes as a whole.
    slots = sorted({0, 1, 63, 64, 65, t // 3, t // 2, t // 2 + 1, t - 65, t - 64, t - 2, t - 1, (1 << 19) - 1, 1 << 19, (1 << 19) + 1})
    pair = unpack_k(kc[-1:, -1:])[0, 0]
    plant(pair, slots, gh)
    kc[-1, -1] = pair.view(Lmax, Dh // 8, 8).transpose(0, 1)
    # Every other pair has the same heavy slots with other values, so that a wrong pair's rows are of the same kind.
    kc[:, :, 0, :, 0] = kc[-1, -1, 0, :, 0]
    q, k, v = (torch.empty(B, H, n, Dh, dtype=dt, device=DEV).normal_(generator=g) for _ in range(3))
    q[..., 1:] *= 0.01
    q[..., 0], k[..., 0] = HEAVY, 0
    K, V = pair[slots].clone(), vc[-1, -1, slots].double()
    logit = logit_error(q[-1, -1], K, 1.0, Dh)
    out = FFA().attention_tree(q, k, v, kc, vc, 1.0, t)
    p = torch.softmax(q[-1, -1].double() @ K.double().t().contiguous(), -1)
    check(out[-1, -1], p, V, dt, logit, "tree")
    assert torch.equal(unpack_k(kc[-1:, -1:])[0, 0, t:t + n], k[-1, -1]) and torch.equal(vc[-1, -1, t:t + n], v[-1, -1])
    FFA().commit_tree([(kc, vc)], t, ints([[1, 4]] * B), ints([2] * B))
    assert torch.equal(vc[-1, -1, t:t + 2], v[-1, -1, [1, 4]]) and torch.equal(unpack_k(kc[-1:, -1:])[0, 0, t:t + 2], k[-1, -1, [1, 4]])
    w = torch.zeros(B, H, Lmax, device=DEV)
    out = FFA().attention_weights(q[:, :, 0].contiguous(), k[:, :, 0].contiguous(), v[:, :, 0].contiguous(), kc, vc, 1.0, t + 2, w)
    check(out[-1:, -1], p[:1], V, dt, logit, "weights")
    got = w[-1, -1, slots].double()
    assert bool(((got - p[0]).abs() <= p[0] * (2 * logit + (2 * len(slots) + 64) * 2.0 ** -24)).all())
    rest = w[-1, -1].clone()
    rest[slots] = 0
    assert float(rest.max()) < math.exp(-25)
    # Eviction down to the heavy keys and the last two.
    before = (unpack_k(kc[-1:, -1:])[0, 0].clone(), vc[-1, -1].clone())
    kept = FFA().evict([(kc, vc)], [w], t + 3, len(slots) + 2, 2)[0, -1, -1].long().tolist()
    assert kept == slots + [t + 1, t + 2]
    assert torch.equal(unpack_k(kc[-1:, -1:])[0, 0, :len(kept)], before[0][kept]) and torch.equal(vc[-1, -1, :len(kept)], before[1][kept])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh,H,Hq,n,t", [(64, 2, 2, 4, 9001), (64, 1, 1, 64, 9001), (80, 1, 2, 40, 5003), (128, 1, 8, 24, 7777), (256, 1, 4, 9, 4100),
                                         (128, 2, 2, 3, 130), (64, 40, 40, 33, 1500)])
def test_heavy_keys_in_pieces(dtype, Dh, H, Hq, n, t):
    """Heavy keys at the ends, around multiples of 16, 32 and 64 and at random; left padding and a short sample move the
    visible range's ends onto them."""
    print("heavy pieces", dtype, Dh, H, Hq, n, t, flush=True)
    dt, B, scale = DT[dtype], 2, 1.0
    g = torch.Generator().manual_seed(t + n)
    for run in range(3):
        first, lengths = ([0, 0], [t, t]) if run == 0 else ([t // 3 + run, 0], [t, t - t // 5 - run])
        lo, hi = max(first), min(lengths)
        slots = {first[0], hi - 1, lengths[0] - 1, lo, lo + 1, hi - 2} | {int(x) for x in torch.randint(lo, hi, (12,), generator=g)}
        slots |= {x for m in (16, 32, 64, 1024) for x in (lo // m * m + m - 1, lo // m * m + m) if lo <= x < hi}
        slots = sorted(slots)
        K, V = torch.randn(B, H, t, Dh, generator=g) * 0.01, torch.randn(B, H, t, Dh, generator=g)
        plant(K, slots, g)
        K, V = K.to(dt), V.to(dt)
        Lmax = t + n + 3
        kc, vc = pack_k(K.to(DEV), Lmax, NAN), pack_v(V.to(DEV), Lmax, NAN)
        q, k, v = (torch.randn(B, h, n, Dh, generator=g).to(dt) for h in (Hq, H, H))
        q[..., 1:] *= 0.01
        q[..., 0], k[..., 0] = HEAVY, 0
        out = FFA().attention_tree(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc, scale, t, first_keys=ints(first), lengths=ints(lengths)).cpu()
        w = torch.zeros(B, H, Lmax, device=DEV)
        one = FFA().attention_weights(*(x[:, :, 0].contiguous().to(DEV) for x in (q, k, v)), kc, vc, scale, t, w,
                                      first_keys=ints(first), lengths=ints(lengths)).cpu()
        w = w.cpu().double()
        for b in range(B):
            mine = [s for s in slots if first[b] <= s < lengths[b]]
            for hq in {0, Hq - 1}:
                h = hq // (Hq // H)
                Kh, Vh = K[b, h, mine], V[b, h, mine].double()
                p = torch.softmax(q[b, hq].double() @ Kh.double().t() * scale, -1)
                logit = logit_error(q[b, hq], Kh, scale, Dh)
                check(out[b, hq], p, Vh, dt, logit, f"tree {run} {b} {hq}")
                check(one[b, hq:hq + 1], p[:1], Vh, dt, logit, f"weights {run} {b} {hq}")
            for h in range(H):
                heads = range(h * (Hq // H), (h + 1) * (Hq // H))
                z = torch.stack([q[b, x, 0].double() @ K[b, h, mine].double().t() * scale for x in heads])
                s = torch.softmax(z, -1).sum(0)
                logit = max(logit_error(q[b, x, :1], K[b, h, mine], scale, Dh) for x in heads)
                assert bool(((w[b, h, mine] - s).abs() <= s * (2 * logit + (2 * len(mine) + 64 + len(heads)) * 2.0 ** -24)).all())
                light = w[b, h].clone()
                light[mine] = 0
                assert float(light.max()) < math.exp(-25)
