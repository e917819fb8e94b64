"""GPU tests of what values may do in the tree attention and the weight-summing step: large finite values of
keys without weight, and NaN keys, wherever the cut of the keys puts them."""
import pytest
import torch

from tests.cache_ops_testlib import DEV, DT, pack_k, pack_v, random_parents
from tests.test_gpu_cache_ops import FFA, INF, NAN, ints, make

pytestmark = pytest.mark.gpu

LARGE = {"fp16": 65504.0, "bf16": 3e38, "fp32": 3e38}


def bits(x):
    return x.contiguous().view(torch.int32 if x.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("t,n,G", [(0, 2, 1), (70, 40, 2), (5000, 33, 1), (1300, 64, 4)])
def test_large_values_of_nodes_out_of_sight(dtype, Dh, t, n, G):
    """Rows that do not see a node come out the same, bit for bit, whatever finite value it holds."""
    print("out of sight", dtype, Dh, t, n, G, flush=True)
    H = 2
    g, kc, vc, q, k, v = make(t + n, dtype, 1, H, H * G, Dh, t, n)
    siblings = torch.tensor([[-1] + [0] * (n - 1)], dtype=torch.int32) if n > 2 else torch.tensor([[-1, -1]], dtype=torch.int32)
    hidden = n // 2 if n > 2 else 0
    for parents, rows in ((siblings, [i for i in range(n) if i != hidden]), (None, list(range(n - 1)))):
        node = hidden if parents is not None else n - 1
        got = []
        for value in (0.0, LARGE[dtype], -LARGE[dtype]):
            v2 = v.clone()
            v2[:, :, node] = value
            got.append(FFA().attention_tree(q, k, v2, kc, vc, Dh ** -0.5, t, ints(parents))[:, :, rows])
        assert bool(got[0].isfinite().all())
        assert torch.equal(bits(got[0]), bits(got[1])) and torch.equal(bits(got[0]), bits(got[2])), (parents is None)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("t", [50, 5000])
def test_large_values_of_cached_keys_without_weight(dtype, Dh, t):
    """A cached key whose score lies so far below the others that its weight is 0 in 32 bits (e^-400) adds nothing."""
    print("without weight", dtype, Dh, t, flush=True)
    g, kc, vc, q, k, v = make(t, dtype, 2, 2, 2, Dh, t, 5)
    K = torch.randn(2, 2, t, Dh, generator=g) * 0.1
    K[..., 0] = 0
    K[:, :, 3::7, 0] = -100
    kc = pack_k(K.to(DT[dtype]).to(DEV), kc.shape[3], NAN)
    q[..., 0], k[..., 0] = 4.0, 0.0
    V = vc[:, :, :t].clone()
    par = ints(random_parents(g, 2, 5))
    got, summed = [], []
    for value in (0.0, LARGE[dtype], -LARGE[dtype]):
        V[:, :, 3::7] = value
        vc = pack_v(V, kc.shape[3], NAN)
        got.append(FFA().attention_tree(q, k, v, kc.clone(), vc.clone(), 1.0, t, par))
        w = torch.zeros(2, 2, kc.shape[3], device=DEV)
        summed.append(FFA().attention_weights(q[:, :, 0].contiguous(), k[:, :, 0].contiguous(), v[:, :, 0].contiguous(), kc.clone(), vc, 1.0, t, w))
        assert not bool(w[:, :, 3:t:7].any())
    for x in (got, summed):
        assert bool(x[0].isfinite().all()) and torch.equal(bits(x[0]), bits(x[1])) and torch.equal(bits(x[0]), bits(x[2]))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_infinite_values_of_light_keys(dtype):
    """A visible infinite value shows, also behind a weight whose lower part is zero."""
    print("light", dtype, flush=True)
    _, kc, vc, q, k, v = make(15, dtype, 1, 1, 1, 64, 64, 1)
    kc = pack_k(torch.zeros(1, 1, 64, 64, dtype=DT[dtype], device=DEV), kc.shape[3], NAN)
    k = torch.zeros_like(k)
    for slot in range(0, 64, 9):
        vc2 = vc.clone()
        vc2[0, 0, slot, 5] = INF
        out = FFA().attention_tree(q, k, v, kc, vc2, 0.125, 64)
        assert float(out[0, 0, 0, 5]) == INF and bool(out[0, 0, 0, :5].isfinite().all()) and bool(out[0, 0, 0, 6:].isfinite().all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("where", ["a run of keys", "one key behind padding", "one key before the end"])
def test_nan_scores_show_whatever_piece_they_fill(dtype, where):
    """A row that sees a NaN key is NaN, and so are the weights it gives, also where the keys are cut in pieces
    and all that the row sees of a piece is NaN.  The sample beside it has none."""
    print("NaN piece", dtype, where, flush=True)
    t, H, Dh = 6000, 2, 64
    _, kc, vc, q, k, v = make(16, dtype, 2, H, H, Dh, t, 3)
    first, lengths = [0, 0], [t, t]
    if where == "a run of keys":
        nan = slice(500, 5500)                     # whole pieces, and none of the first and the last
    elif where == "one key behind padding":
        first[0] = t - 200
        nan = slice(first[0], first[0] + 1)
    else:
        lengths[0] = 3001
        nan = slice(3000, 3001)
    for at in {nan.start, nan.stop - 1, (nan.start + nan.stop) // 2}:
        # Every cut: the visible keys of sample 0 end or begin at the NaN ones in one of these.
        for f0, n0 in ((first[0], lengths[0]), (at, lengths[0]), (first[0], at + 1)):
            if not f0 <= at < n0:
                continue
            kc2 = kc.clone()
            kc2[0, 0, :, nan] = NAN
            fk, ln = ints([f0, first[1]]), ints([n0, lengths[1]])
            out = FFA().attention_tree(q, k, v, kc2, vc.clone(), 0.125, t, first_keys=fk, lengths=ln)
            assert bool(out[0, 0].isnan().all()) and bool(out[0, 1].isfinite().all()) and bool(out[1].isfinite().all()), (at, f0, n0)
            w = torch.zeros(2, H, kc.shape[3], device=DEV)
            one = FFA().attention_weights(q[:, :, 0].contiguous(), k[:, :, 0].contiguous(), v[:, :, 0].contiguous(), kc2, vc.clone(), 0.125, t, w,
                                          first_keys=fk, lengths=ln)
            assert bool(one[0, 0].isnan().all()) and bool(one[0, 1].isfinite().all()) and bool(one[1].isfinite().all()), (at, f0, n0)
            assert bool(w[0, 0, f0:n0 + 1].isnan().all()) and bool(w[0, 1].isfinite().all()) and bool(w[1].isfinite().all())
            assert not bool(w[0, 0, :f0].any()) and not bool(w[0, 0, n0 + 1:].any())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_weights_keep_two_16_bit_parts_rounded_to_nearest(dtype):
    """Two keys whose values cancel but for 2^-9 (bf16) of the lighter one's weight p, so that the result's own rounding is
    small.  The heavier key's weight is a power of two and exact.  p = 1.m splits into a part cut after 7 (bf16) or 10
    (fp16) bits of m and the nearest number of 8 or 11 bits to the rest: 2^-16 or 2^-22 of p at most.  The scores are
    single products; their scaling, the exponentials and the sum of the weights are 8 roundings of 2^-24, and the sums
    of products as many."""
    print("two parts", dtype, flush=True)
    B, H, Dh = 4, 64, 64
    g = torch.Generator().manual_seed(17)
    dt = DT[dtype]
    K, V = torch.zeros(B, H, 2, Dh), torch.zeros(B, H, 2, Dh)
    K[:, :, 1, 0] = -0.1 - 0.55 * torch.rand(B, H, generator=g)
    K = K.to(dt)
    p = torch.exp(K[:, :, 1, 0].double())
    V[:, :, 1], V[:, :, 0] = 1.0, -p[..., None].float()
    V = V.to(dt)
    q, k, v = (torch.zeros(B, H, 1, Dh, dtype=dt) for _ in range(3))
    q[..., 0], k[..., 0] = 1.0, -100.0
    want = (V[:, :, 0].double() + p[..., None] * V[:, :, 1].double()) / (1 + p[..., None])
    kc, vc = pack_k(K.to(DEV), 4, NAN), pack_v(V.to(DEV), 4, NAN)
    out = FFA().attention_tree(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc, 1.0, 2)[:, :, 0].double().cpu()
    part = 2.0 ** -16 if dtype == "bf16" else 2.0 ** -22
    tol = torch.finfo(dt).eps / 2 * want.abs() + ((part + 16 * 2.0 ** -24) * p / (1 + p))[..., None]
    assert float(tol.max()) < 2.0 ** -16
    assert bool(((out - want).abs() <= tol).all()), float(((out - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("t,n", [(0, 1), (1, 3), (40, 40), (700, 5), (6000, 17)])
def test_values_of_any_finite_size(dtype, Dh, t, n):
    """All keys alike with weights 1 / keys and one value: the result is that value, also where 4 times the sum of the
    values just fits fp32.  Bound: half a step, the two 16-bit parts, and 2 additions a key in numerator and sum."""
    print("any size", dtype, Dh, t, n, flush=True)
    B, H, dt = 1, 2, DT[dtype]
    q, k = (torch.zeros(B, H, n, Dh, dtype=dt, device=DEV) for _ in range(2))
    kc = pack_k(torch.zeros(B, H, t, Dh, dtype=dt, device=DEV), t + n + 1, NAN)
    tol = torch.finfo(dt).eps / 2 + {"fp16": 2.0 ** -22, "bf16": 2.0 ** -16, "fp32": 0.0}[dtype] + (2 * (t + n) + 64) * 2.0 ** -24
    large = 65504.0 if dtype == "fp16" else 8e37 / (t + n)
    for value in (large, -large, 1.0, 0.01 if dtype == "fp16" else 1e-20):
        V = torch.full((B, H, t + n, Dh), value, dtype=dt, device=DEV)
        vc, v, x = pack_v(V[:, :, :t], t + n + 1, NAN), V[:, :, t:].clone(), float(V[0, 0, 0, 0])
        w = torch.zeros(B, H, t + n + 1, device=DEV)
        outs = [FFA().attention_tree(q, k, v, kc.clone(), vc.clone(), 1.0, t),
                FFA().attention_weights(q[:, :, 0].contiguous(), k[:, :, 0].contiguous(), v[:, :, 0].contiguous(), kc.clone(), vc, 1.0, t, w)]
        for out in outs:
            # A result of fp16 that is rounded up past the largest number is infinite.
            got = out.double().clamp(-65504, 65504) if dtype == "fp16" else out.double()
            assert bool(((got - x).abs() <= tol * abs(x)).all()), (value, float((got - x).abs().max() / abs(x)), tol)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("t,low", [(300, slice(0, 200)), (300, slice(100, 300)), (6000, slice(0, 4000)), (6000, slice(500, 6000)), (6000, slice(1000, 5000))])
def test_large_values_of_a_stretch_without_weight(dtype, Dh, t, low):
    """Whole tiles, waves and pieces whose keys have no weight (e^-400) next to the others: their values, as long as 4
    times their sum fits fp32, change no bit, whichever come first; an infinite one shows."""
    print("stretch", dtype, Dh, t, low, flush=True)
    g, kc, vc, q, k, v = make(t + 1, dtype, 1, 2, 2, Dh, t, 5)
    K = torch.randn(1, 2, t, Dh, generator=g) * 0.1
    K[..., 0] = 0
    K[:, :, low, 0] = -100
    kc = pack_k(K.to(DT[dtype]).to(DEV), kc.shape[3], NAN)
    q[..., 0], k[..., 0] = 4.0, 0.0
    V = vc[:, :, :t].clone()
    got, large = [], 65504.0 if dtype == "fp16" else 8e37 / t
    for value in (0.0, large, -large, INF):
        V[:, :, low] = value
        vc = pack_v(V, kc.shape[3], NAN)
        w = torch.zeros(1, 2, kc.shape[3], device=DEV)
        got.append((FFA().attention_tree(q, k, v, kc.clone(), vc.clone(), 1.0, t),
                    FFA().attention_weights(q[:, :, 0].contiguous(), k[:, :, 0].contiguous(), v[:, :, 0].contiguous(), kc.clone(), vc, 1.0, t, w)))
    for i in range(2):
        assert bool(got[0][i].isfinite().all())
        assert torch.equal(bits(got[0][i]), bits(got[1][i])) and torch.equal(bits(got[0][i]), bits(got[2][i]))
        assert not bool(got[3][i].isfinite().any())
