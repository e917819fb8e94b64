"""GPU tests of the operators next to the decode step -- attention of a tree of drafted tokens, the
move of an accepted path, the weight-summing step, eviction -- against plain forms in 64 bits.  The
slots that nobody may see hold NaN or infinities throughout."""
import math

import pytest
import torch

from tests.cache_ops_testlib import (DEV, DT, assert_close, evict_reference, pack_k, pack_v, random_parents, tree_reference,
                                     tree_tolerance, unpack_k)

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def FFA():
    from fastforwardattention_amd import FastForwardAttn
    return FastForwardAttn


def make(seed, dtype, B, H, Hq, Dh, t, n, Lmax=None, kv=1.0):
    """Inputs on the GPU: caches whose slots from t on hold NaN, and the group's q, k, v."""
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    K, V = ((torch.randn(B, H, t, Dh, generator=g) * kv).to(dt).to(DEV) for _ in range(2))
    Lmax = Lmax or t + n + 3
    q, k, v = (torch.randn(B, n, h, Dh, generator=g).to(dt).to(DEV).transpose(1, 2) for h in (Hq, H, H))
    return g, pack_k(K, Lmax, NAN), pack_v(V, Lmax, NAN), q, k, v


def ints(x):
    return None if x is None else torch.as_tensor(x, dtype=torch.int32).to(DEV)


def run_tree(kc, vc, q, k, v, scale, t, dtype, label, **kw):
    """Calls the operator and checks result and caches; returns the result."""
    K0, V0 = unpack_k(kc).clone(), vc.clone()
    dev = {name: ints(x) for name, x in kw.items()}
    out = FFA().attention_tree(q, k, v, kc, vc, scale, t, **dev)
    torch.cuda.synchronize()
    want, size, bound, _ = tree_reference(q, k, v, K0, V0, scale, t, **kw)
    B, H, n, Dh = k.shape
    assert out.shape == q.shape and out.dtype == q.dtype
    assert_close(out, want, tree_tolerance(q.dtype, want, size, bound, t + n, Dh), label)
    K1, V1 = K0, V0
    for b in range(B):
        at = t if kw.get("lengths") is None else min(max(int(kw["lengths"][b]), 0), t)
        c = n if kw.get("counts") is None else min(max(int(kw["counts"][b]), 0), n)
        K1[b, :, at:at + c], V1[b, :, at:at + c] = k[b, :, :c], v[b, :, :c]
    bits = torch.int32 if q.dtype == torch.float32 else torch.int16
    assert torch.equal(unpack_k(kc).contiguous().view(bits), K1.contiguous().view(bits)), label + ": K cache"
    assert torch.equal(vc.view(bits), V1.view(bits)), label + ": V cache"
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("t,n,G", [(0, 1, 1), (1, 2, 3), (31, 17, 1), (32, 33, 1), (33, 7, 5), (257, 64, 1), (500, 13, 8), (1000, 1, 1)])
def test_tree(dtype, Dh, t, n, G):
    print("tree", dtype, Dh, t, n, G, flush=True)
    B, H = 2, 3
    g, kc, vc, q, k, v = make(t + n, dtype, B, H, H * G, Dh, t, n)
    run_tree(kc, vc, q, k, v, Dh ** -0.5, t, dtype, f"{dtype} {Dh} {t} {n} {G}", parents=random_parents(g, B, n))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
def test_ragged_padded_batch(dtype, Dh):
    """Left padding, samples of different lengths and node counts; what no node sees is NaN or infinite:
    padding and slots past the length in the caches, nodes past the count."""
    print("ragged", dtype, Dh, flush=True)
    B, H, t, n = 6, 2, 300, 40
    g, kc, vc, q, k, v = make(3, dtype, B, H, 2 * H, Dh, t, n)
    lengths, first, counts = [300, 299, 0, 64, 33, 271], [0, 37, 0, 64, 1, 65], [40, 1, 17, 0, 33, 39]
    for b in range(B):
        for cache, dim in ((kc, 3), (vc, 2)):
            cache[b].narrow(dim - 1, 0, first[b]).fill_(INF if b % 2 else NAN)
            cache[b].narrow(dim - 1, lengths[b], t - lengths[b]).fill_(-INF if b % 2 else NAN)
        for x in (q, k, v):
            x[b, :, counts[b]:] = NAN
    out = run_tree(kc, vc, q, k, v, Dh ** -0.5, t, dtype, f"ragged {dtype} {Dh}", parents=random_parents(g, B, n),
                   first_keys=first, lengths=lengths, counts=counts)
    assert all(bool((out[b, :, counts[b]:] == 0).all()) for b in range(B))


@pytest.mark.parametrize("dtype,Dh,H,Hq,n,t", [("fp16", 64, 2, 2, 64, 9001), ("bf16", 128, 1, 8, 24, 7777), ("fp32", 80, 1, 1, 5, 5000),
                                               ("bf16", 256, 1, 4, 64, 4100), ("fp16", 128, 1, 71, 3, 2050)])
def test_long_cache_in_pieces(dtype, Dh, H, Hq, n, t):
    """Few pairs, many keys: the keys are split over workgroups and joined; also left padding that leaves whole pieces empty."""
    print("long", dtype, Dh, H, Hq, n, t, flush=True)
    g, kc, vc, q, k, v = make(5, dtype, 2, H, Hq, Dh, t, n)
    run_tree(kc, vc, q, k, v, Dh ** -0.5, t, dtype, "long chain", first_keys=[0, t - 40])
    run_tree(kc, vc, q, k, v, Dh ** -0.5, t, dtype, "long tree, one sample short", parents=random_parents(g, 2, n), lengths=[t, 100])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_many_workgroups(dtype):
    """More pieces than the chip holds at once, an odd number of them, several row blocks each."""
    print("many", dtype, flush=True)
    B, H, t, n = 37, 5, 96, 33
    _, kc, vc, q, k, v = make(6, dtype, B, H, 2 * H, 64, t, n)
    run_tree(kc, vc, q, k, v, 0.125, t, dtype, "many")


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_nodes_that_are_no_ancestors_have_no_influence(dtype):
    """k and v of one branch are infinite or NaN: the other branches' rows stay finite and right, and the
    branch's own rows show what the formula gives."""
    print("branches", dtype, flush=True)
    B, H, t, n, Dh = 2, 2, 70, 40, 64
    _, kc, vc, q, k, v = make(7, dtype, B, H, H, Dh, t, n)
    parents = torch.tensor([[-1] + [max(-1, i - 3) for i in range(1, n)]] * B, dtype=torch.int32)   # three interleaved branches
    v[0, 0, 3, 5], v[0, 0, 36, 6], v[0, 1, 9, 7] = INF, -INF, NAN
    v[1, :, 33, :] = INF
    k[1, 1, 6] = NAN
    run_tree(kc, vc, q, k, v, 0.125, t, dtype, "branches", parents=parents)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_infinite_values_in_sight(dtype):
    print("visible infinities", dtype, flush=True)
    _, kc, vc, q, k, v = make(8, dtype, 1, 2, 2, 64, 200, 3)
    vc[0, 0, 17, 3], vc[0, 0, 120, 4], vc[0, 1, 5, 5], vc[0, 1, 6, 5] = INF, -INF, INF, -INF
    kc[0, 0, 0, 60, 0] = NAN
    out = run_tree(kc, vc, q, k, v, 0.125, 200, dtype, "one NaN key")
    assert bool(out[0, 0].isnan().all())
    kc[0, 0, 0, 60, 0] = 0.5
    run_tree(kc, vc, q, k, v, 0.125, 200, dtype, "infinite values")


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("order", ["rising", "falling", "equal"])
def test_large_scores(dtype, order):
    """Logits over hundreds, rising or falling along the cache: the reference exponent moves at every tile or never."""
    print("large scores", dtype, order, flush=True)
    B, H, t, n, Dh = 1, 2, 600, 6, 64
    g, kc, vc, q, k, v = make(9, dtype, B, H, H, Dh, t, n)
    K = torch.zeros(B, H, t, Dh)
    ramp = torch.linspace(-100, 100, t) if order != "equal" else torch.full((t,), 100.0)
    K[..., 0] = ramp.flip(0) if order == "falling" else ramp
    kc = pack_k(K.to(DT[dtype]).to(DEV), kc.shape[3], NAN)
    q[..., 0] = 3.0
    k[..., 0] = 1.0
    run_tree(kc, vc, q, k, v, 1.0, t, dtype, f"large {order}")


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_strides_and_alignment(dtype):
    """q, k, v as slices of one fused projection, as [B,heads,n,Dh], as a broadcast over heads, and off any
    16-byte boundary."""
    print("strides", dtype, flush=True)
    B, H, Dh, t, n = 2, 4, 64, 100, 9
    g, kc, vc, _, _, _ = make(10, dtype, B, H, H, Dh, t, n)
    fused = torch.randn(B, n, 3, H, Dh, generator=g).to(DT[dtype]).to(DEV)
    q, k, v = (fused[:, :, i].transpose(1, 2) for i in range(3))
    want = run_tree(kc, vc, q, k, v, 0.125, t, dtype, "fused")
    same = [(q.contiguous(), k.contiguous(), v.contiguous())]
    off = torch.empty(3, B * H * n * Dh + 1, dtype=DT[dtype], device=DEV)
    off[:, 1:] = torch.stack([q, k, v]).reshape(3, -1)
    same.append(tuple(off[i, 1:].view(B, H, n, Dh) for i in range(3)))
    same.append(tuple(x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)))
    for q2, k2, v2 in same:
        assert torch.equal(run_tree(kc, vc, q2, k2, v2, 0.125, t, dtype, "same values"), want)
    run_tree(kc, vc, q, k[:, :1].expand(B, H, n, Dh), v[:, :1].expand(B, H, n, Dh), 0.125, t, dtype, "broadcast")


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-42, -1e-42])
def test_scales_that_are_not_positive(dtype, scale):
    """A negative scale turns the order of the keys, zero makes them all alike; masked keys stay masked."""
    print("scale", dtype, scale, flush=True)
    g, kc, vc, q, k, v = make(13, dtype, 2, 2, 4, 64, 130, 5)
    run_tree(kc, vc, q, k, v, scale, 130, dtype, f"scale {scale}", parents=random_parents(g, 2, 5), first_keys=[0, 40], lengths=[130, 77])


def test_far_apart_tokens_are_copied():
    """A token stride of 64 MiB and more, in a buffer that holds it: the rows are brought together first."""
    _, kc, vc, q, k, v = make(14, "fp16", 1, 1, 1, 64, 40, 2)
    far = torch.empty(1 << 25 | 64, dtype=torch.float16, device=DEV).as_strided((1, 1, 2, 64), (1 << 25, 1 << 25, 1 << 25, 1))
    far.copy_(k)
    run_tree(kc, vc, q, far, v, 0.125, 40, "fp16", "far apart")


def test_wrong_parents_mean_the_root():
    _, kc, vc, q, k, v = make(11, "fp16", 1, 2, 2, 64, 40, 6)
    run_tree(kc, vc, q, k, v, 0.125, 40, "fp16", "wrong parents", parents=torch.tensor([[7, 1, 1, -5, 3, 1 << 30]], dtype=torch.int32))
    run_tree(kc, vc, q, k, v, 0.125, 40, "fp16", "wrong samples", lengths=[99], first_keys=[-3], counts=[77])


def test_one_node_equals_the_decode_step():
    """n = 1 is the engine's own step."""
    g = torch.Generator().manual_seed(12)
    B, H, Dh, L = 3, 4, 128, 333
    K, V = (torch.randn(B, H, L, Dh, generator=g).half().to(DEV) for _ in range(2))
    q, k, v = (torch.randn(B, H, Dh, generator=g).half().to(DEV) for _ in range(3))
    ffa = FFA()(K, V, L + 8, False)
    kc, vc = ffa.get_cache()
    first = ints([0, 7, 200])
    a = ffa.attention(q, k, v, kc, vc, 0.09, L, first, 0.0)
    b = ffa.attention_tree(q[:, :, None], k[:, :, None], v[:, :, None], kc, vc, 0.09, L, first_keys=first)[:, :, 0]
    assert float((a - b).abs().max()) <= 2 * 2 ** -11 * float(a.abs().max())      # each side rounds once


# ------------------------------------------------------------------------------------------------
def commit_reference(K, t, path, accepted, lengths):
    out = K.clone()
    Lmax = K.shape[2]
    for b in range(K.shape[0]):
        at = t if lengths is None else min(max(int(lengths[b]), 0), t)
        for j in range(min(max(int(accepted[b]), 0), path.shape[1])):
            out[b, :, at + j] = K[b, :, at + min(max(int(path[b, j]), 0), Lmax - 1 - at)]
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("n,m,layers", [(1, 1, 1), (8, 3, 2), (64, 64, 1), (64, 31, 35)])
def test_commit(dtype, Dh, n, m, layers):
    print("commit", dtype, Dh, n, m, layers, flush=True)
    B, H, t = 4, 3, 21
    g = torch.Generator().manual_seed(n + m)
    Lmax = t + n + 1
    caches, want = [], []
    path = torch.stack([torch.randperm(n, generator=g)[:m].sort().values for _ in range(B)]).int()
    accepted = torch.tensor([m, 0, (m + 1) // 2, 1])
    lengths = [21, 20, 0, 5]
    for _ in range(layers):
        K, V = (torch.randn(B, H, Lmax, Dh, generator=g).to(DT[dtype]).to(DEV) for _ in range(2))
        caches.append((pack_k(K, Lmax), pack_v(V, Lmax)))
        want.append([commit_reference(x, t, path, accepted, lengths) for x in (K, V)])
    FFA().commit_tree(caches, t, ints(path), ints(accepted), lengths=ints(lengths))
    for (kc, vc), (K, V) in zip(caches, want):
        assert torch.equal(unpack_k(kc), K) and torch.equal(vc, V)


@pytest.mark.parametrize("Dh", [64, 80, 256])
def test_commit_brings_wrong_values_into_range(Dh):
    """Any path is a gather of old slots; entries outside the cache mean its last slot, counts are clamped."""
    g = torch.Generator().manual_seed(1)
    B, H, t, m, Lmax = 3, 2, 10, 5, 16
    K, V = (torch.randn(B, H, Lmax, Dh, generator=g).half().to(DEV) for _ in range(2))
    path = torch.tensor([[4, 3, 2, 1, 0], [2, 2, 2, 2, 2], [1 << 30, -7, 99, 5, 0]])
    accepted = torch.tensor([99, 5, 4])
    kc, vc = pack_k(K, Lmax), pack_v(V, Lmax)
    FFA().commit_tree([(kc, vc)], t, ints(path), ints(accepted), lengths=ints([10, 700, 3]))
    for got, x in ((unpack_k(kc), K), (vc, V)):
        assert torch.equal(got, commit_reference(x, t, path, accepted, [10, 700, 3]))


# ------------------------------------------------------------------------------------------------
def run_weights(kc, vc, q, k, v, scale, t, kw, label, first_keys=None, lengths=None):
    B, Hq, Dh = q.shape
    H = k.shape[1]
    K0, V0, w0 = unpack_k(kc).clone(), vc.clone(), kw.clone()
    out = FFA().attention_weights(q, k, v, kc, vc, scale, t, kw, first_keys=ints(first_keys), lengths=ints(lengths))
    torch.cuda.synchronize()
    want, size, bound, p = tree_reference(q[:, :, None], k[:, :, None], v[:, :, None], K0, V0, scale, t, first_keys=first_keys,
                                          lengths=lengths)
    assert_close(out[:, :, None], want, tree_tolerance(q.dtype, want, size, bound, t + 1, Dh), label)
    u = 2.0 ** -24
    rel = 2 * (bound * (Dh + 4) * u + 4 * u) + (t + 64 + Hq // H) * u
    w1, tol = w0.double(), torch.zeros_like(w0, dtype=torch.float64)
    for b in range(B):
        n = t if lengths is None else lengths[b]
        f = 0 if first_keys is None else min(first_keys[b], n)
        s = p[b].sum((1, 2))
        w1[b, :, f:n] += s[:, :-1]
        w1[b, :, n] = s[:, -1]
        tol[b, :, f:n + 1] = rel * s + u * w1[b, :, f:n + 1].abs()      # the last sum rounds once more
    assert_close(kw, w1, tol, label + ": weights")
    assert torch.equal(kw[tol == 0].nan_to_num(-5), w0[tol == 0].nan_to_num(-5))
    for b in range(B):
        n = t if lengths is None else lengths[b]
        assert torch.equal(unpack_k(kc)[b, :, n], k[b]) and torch.equal(vc[b, :, n], v[b])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Dh", [64, 80, 128, 256])
@pytest.mark.parametrize("t,G", [(0, 1), (1, 4), (33, 1), (300, 20), (2000, 2)])
def test_weights(dtype, Dh, t, G):
    print("weights", dtype, Dh, t, G, flush=True)
    B, H = 2, 2
    g, kc, vc, q, k, v = make(t + G, dtype, B, H, H * G, Dh, t, 1)
    kw = torch.rand(B, H, kc.shape[3], generator=g).to(DEV)
    q, k, v = (x[:, :, 0].contiguous() for x in (q, k, v))
    run_weights(kc, vc, q, k, v, Dh ** -0.5, t, kw, f"weights {dtype} {Dh} {t} {G}")
    if t >= 33:
        lengths, first = [t - 20, t - 1], [t // 2, 0]
        for cache, dim in ((kc, 3), (vc, 2)):
            cache[0].narrow(dim - 1, 0, first[0]).fill_(NAN)
            cache[0].narrow(dim - 1, lengths[0], 20).fill_(INF)
        kw[0, :, :first[0]] = NAN
        run_weights(kc, vc, q, k, v, Dh ** -0.5, t, kw, "ragged", first_keys=first, lengths=lengths)


# ------------------------------------------------------------------------------------------------
def run_evict(seed, dtype, layers, B, H, Dh, t, keep, recent, in_place, lengths=None, first=None, kind="random", label=""):
    g = torch.Generator().manual_seed(seed)
    Lmax, Lto = t + 5, (t + 5 if in_place else keep + 3)
    K, V = (torch.randn(layers, B, H, Lmax, Dh, generator=g).to(DT[dtype]).to(DEV) for _ in range(2))
    w = torch.rand(layers, B, H, Lmax, generator=g)
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float() / 4
        w[torch.rand(w.shape, generator=g) < 0.2] = -0.0
    elif kind == "odd":
        pick = torch.tensor([NAN, INF, -INF, -1.0, 0.0, 1e-45, -1e-45, 3e38, -3e38, 1.0])
        w = pick[torch.randint(0, len(pick), w.shape, generator=g)]
    w = w.to(DEV)
    caches = [(pack_k(K[a], Lmax), pack_v(V[a], Lmax)) for a in range(layers)]
    ws = [x.clone() for x in w]
    if in_place:
        into, to = None, [(k, v, x) for (k, v), x in zip(caches, ws)]
    else:
        to = [(pack_k(torch.full((B, H, Lto, Dh), 7.0, dtype=DT[dtype], device=DEV), Lto),
               torch.full((B, H, Lto, Dh), 7.0, dtype=DT[dtype], device=DEV), torch.full((B, H, Lto), 7.0, device=DEV)) for _ in range(layers)]
        into = to
    old = [(unpack_k(k).clone(), v.clone(), x.clone()) for k, v, x in to]
    kept = FFA().evict(caches, ws, t, keep, recent, first_keys=ints(first), lengths=ints(lengths), into=into)
    torch.cuda.synchronize()
    assert kept.shape == (layers, B, H, keep) and kept.dtype == torch.int32
    wl = w.cpu().tolist()
    for a in range(layers):
        K1, V1, w1 = old[a]
        for b in range(B):
            n = t if lengths is None else lengths[b]
            f = 0 if first is None else first[b]
            for h in range(H):
                stay = evict_reference(wl[a][b][h], n, f, keep, recent)
                assert kept[a, b, h].tolist() == stay + [-1] * (keep - len(stay)), (label, a, b, h)
                K1[b, h, :len(stay)], V1[b, h, :len(stay)] = K[a, b, h, stay], V[a, b, h, stay]
                w1[b, h, :len(stay)] = w[a, b, h, stay]
        assert torch.equal(unpack_k(to[a][0]), K1) and torch.equal(to[a][1], V1), label
        assert torch.equal(to[a][2].nan_to_num(-5), w1.nan_to_num(-5)), label


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype,Dh", [("fp16", 64), ("bf16", 80), ("fp32", 80), ("fp32", 128), ("fp16", 256), ("fp32", 256)])
@pytest.mark.parametrize("t,keep,recent", [(1, 1, 0), (9, 8, 3), (130, 65, 65), (700, 300, 0), (1500, 1400, 200)])
def test_evict(dtype, Dh, t, keep, recent, in_place):
    print("evict", dtype, Dh, t, keep, recent, in_place, flush=True)
    run_evict(t, dtype, 2, 2, 3, Dh, t, keep, recent, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict_ragged_padded(kind, in_place):
    """Samples with fewer slots than stay, none at all, padding that has to stay, ties, zeros of both signs, NaN and infinities."""
    print("evict ragged", kind, in_place, flush=True)
    lengths, first = [0, 1, 99, 100, 101, 400, 377, 400], [0, 1, 50, 0, 101, 350, 13, 0]
    for recent in (0, 20, 100):
        run_evict(3, "fp16", 1, 8, 2, 64, 400, 100, recent, in_place, lengths, first, kind, f"{kind} {recent}")


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_many_caches_and_long(in_place):
    print("evict many", in_place, flush=True)
    run_evict(4, "fp16", 37, 1, 1, 64, 200, 90, 10, in_place)
    run_evict(5, "bf16", 1, 1, 2, 128, 20000, 9000, 1000, in_place, kind="ties")
    run_evict(6, "fp16", 1, 1, 2, 64, 40000, 39000, 100, in_place)


def test_evict_into_the_same_caches_with_other_weights():
    """In place for K and V while the weights go to a buffer of their own."""
    g = torch.Generator().manual_seed(8)
    K, V = (torch.randn(1, 2, 50, 64, generator=g).half().to(DEV) for _ in range(2))
    kc, vc, w = pack_k(K, 50), pack_v(V, 50), torch.rand(1, 2, 50, generator=g).to(DEV)
    w0, w2 = w.clone(), torch.zeros(1, 2, 50, device=DEV)
    kept = FFA().evict([(kc, vc)], [w], 50, 20, 5, into=[(kc, vc, w2)])
    at = kept[0].long()
    assert torch.equal(w, w0) and torch.equal(w2[..., :20], torch.gather(w0, 2, at)) and not bool(w2[..., 20:].any())
    assert torch.equal(vc[:, :, :20], torch.gather(V, 2, at[..., None].expand(1, 2, 20, 64)))


# ------------------------------------------------------------------------------------------------
def test_same_call_twice_gives_the_same_bits():
    g, kc, vc, q, k, v = make(20, "bf16", 2, 3, 6, 128, 3001, 20)
    par = ints(random_parents(g, 2, 20))
    a = FFA().attention_tree(q, k, v, kc, vc, 0.09, 3001, par)
    for _ in range(3):
        assert torch.equal(FFA().attention_tree(q, k, v, kc, vc, 0.09, 3001, par), a)


def test_two_streams_at_once():
    """Two calls that overlap on one device, each with its own workspace."""
    sets = [make(30 + i, "fp16", 1, 2, 2, 64, 9000, 16) for i in range(2)]
    want = [FFA().attention_tree(s[3], s[4], s[5], s[1], s[2], 0.125, 9000) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(FFA().attention_tree(s[3], s[4], s[5], s[1], s[2], 0.125, 9000))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_calls_replay():
    """A whole step of a program -- tree, commit, weight-summing step, eviction -- captured twice in two graphs
    over the same caches, replayed in turn with eager work between: every replay equals the eager run."""
    g, kc, vc, q, k, v = make(40, "fp16", 2, 2, 4, 64, 5000, 12, Lmax=5020)
    par, path, acc = ints(random_parents(g, 2, 12)), ints([[0, 2, 5], [1, 4, 9]]), ints([3, 2])
    w = torch.rand(2, 2, 5020, generator=g).to(DEV)
    q1, k1, v1 = (x[:, :, 0].contiguous() for x in (q, k, v))
    small = (torch.zeros(2, 2, 8, 3000, 8, dtype=torch.float16, device=DEV), torch.zeros(2, 2, 3000, 64, dtype=torch.float16, device=DEV),
             torch.zeros(2, 2, 3000, device=DEV))
    start = [x.clone() for x in (kc, vc, w)]

    def step():
        a = FFA().attention_tree(q, k, v, kc, vc, 0.125, 5000, par)
        FFA().commit_tree([(kc, vc)], 5000, path, acc)
        b = FFA().attention_weights(q1, k1, v1, kc, vc, 0.125, 5002, w)
        c = FFA().evict([(kc, vc)], [w], 5003, 3000, 64, into=[small])
        return a, b, c

    def reset():
        for x, y in zip((kc, vc, w), start):
            x.copy_(y)
        for x in small:
            x.zero_()

    reset()
    want = [x.clone() for x in step()] + [x.clone() for x in (kc, vc, w, *small)]
    graphs, outs = [], []
    for _ in range(2):
        reset()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = step()
        graphs.append(gr)
        outs.append(o)
    for i in range(6):
        reset()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = list(outs[i % 2]) + [kc, vc, w, *small]
        assert all(torch.equal(x.view(torch.int16) if x.dtype == torch.float16 else x, y.view(torch.int16) if y.dtype == torch.float16 else y)
                   for x, y in zip(got, want)), i
        FFA().attention_tree(q, k, v, kc, vc, 0.125, 4000, par)      # eager work of another size between the replays


def test_speculative_decoding_equals_plain_decoding():
    """Draft a tree, attend, accept a path, commit, go on -- ragged, three rounds: the caches and the next
    step are those of a plain decode that was fed the accepted tokens one by one."""
    g = torch.Generator().manual_seed(50)
    B, H, Dh, L, n = 3, 2, 64, 120, 10
    K, V = (torch.randn(B, H, L, Dh, generator=g).half().to(DEV) for _ in range(2))
    kc, vc = FFA()(K, V, L + 60, False).get_cache()
    rows = [[K[b].transpose(0, 1)] for b in range(B)], [[V[b].transpose(0, 1)] for b in range(B)]     # [slots,H,Dh] of each sample
    lengths = torch.full((B,), L, dtype=torch.int32)
    for step in range(3):
        q, k, v = (torch.randn(B, H, n, Dh, generator=g).half().to(DEV) for _ in range(3))
        parents = random_parents(g, B, n)
        t = int(lengths.max())
        FFA().attention_tree(q, k, v, kc, vc, 0.125, t, ints(parents), lengths=ints(lengths))
        path, acc = torch.zeros(B, n, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        for b in range(B):
            node = int(torch.randint(0, n, (1,), generator=g))
            chain = []
            while node >= 0:
                chain.insert(0, node)
                node = int(parents[b, node])
            path[b, :len(chain)] = torch.tensor(chain)
            acc[b] = len(chain) if b or step else 0                    # nothing accepted once
            for new, x in zip(rows, (k, v)):
                new[b].append(x[b, :, chain[: int(acc[b])]].transpose(0, 1))
        FFA().commit_tree([(kc, vc)], t, ints(path), ints(acc), lengths=ints(lengths))
        lengths = lengths + acc
    kt = unpack_k(kc)
    for b in range(B):
        m = int(lengths[b])
        assert torch.equal(kt[b, :, :m], torch.cat(rows[0][b]).transpose(0, 1)) and torch.equal(vc[b, :, :m], torch.cat(rows[1][b]).transpose(0, 1))
    assert len(set(lengths.tolist())) > 1
    q, k, v = (torch.randn(B, H, 1, Dh, generator=g).half().to(DEV) for _ in range(3))
    for x in (kc, vc):
        for b in range(B):
            (x[b].narrow(2 if x is kc else 1, int(lengths[b]), x.shape[3 if x is kc else 2] - int(lengths[b]))).fill_(NAN)
    run_tree(kc, vc, q, k, v, 0.125, int(lengths.max()), "fp16", "after", lengths=lengths.tolist())


def test_bounded_decode_follows_its_definition():
    """Decode with an evicting cache: every step's result is attention over exactly the tokens that the
    definition keeps, tracked on the host by token, three evictions long."""
    g = torch.Generator().manual_seed(60)
    B, H, Dh, L, keep, recent, room = 2, 2, 64, 90, 48, 8, 16
    K, V = (torch.randn(B, H, L, Dh, generator=g).to(DEV) for _ in range(2))
    kc, vc = pack_k(K, L), pack_v(V, L)
    w = (torch.rand(B, H, L, generator=g) * 5).to(DEV)
    small = (torch.zeros(B, H, 16, keep + room, 4, device=DEV), torch.zeros(B, H, keep + room, Dh, device=DEV), torch.zeros(B, H, keep + room, device=DEV))
    alive = [[evict_reference(w[b, h].tolist(), L, 0, keep, recent) for h in range(H)] for b in range(B)]
    FFA().evict([(kc, vc)], [w], L, keep, recent, into=[small])
    kc, vc, w = small
    t = keep
    for step in range(3 * room):
        if t == keep + room:
            before = w.tolist()
            FFA().evict([(kc, vc)], [w], t, keep, recent)
            alive = [[[alive[b][h][j] for j in evict_reference(before[b][h], t, 0, keep, recent)] for h in range(H)] for b in range(B)]
            t = keep
        q, k, v = (torch.randn(B, H, Dh, generator=g).to(DEV) for _ in range(3))
        K, V = torch.cat([K, k[:, :, None]], 2), torch.cat([V, v[:, :, None]], 2)
        out = FFA().attention_weights(q, k, v, kc, vc, 0.125, t, w)
        for b in range(B):
            for h in range(H):
                alive[b][h].append(K.shape[2] - 1)
                kk, vv = K[b, h, alive[b][h]].double(), V[b, h, alive[b][h]].double()
                p = torch.softmax(kk @ q[b, h].double() * 0.125, 0)
                bound = float((kk.abs() @ q[b, h].double().abs()).max()) * 0.125
                want, size = p @ vv, p @ vv.abs()
                assert_close(out[b, h], want, tree_tolerance(torch.float32, want, size, bound, t + 1, Dh), f"step {step}")
        t += 1


@pytest.mark.parametrize("what", ["tree", "weights", "commit", "evict"])
def test_refusals(what):
    """Arguments that do not fit raise before anything is launched."""
    _, kc, vc, q, k, v = make(70, "fp16", 2, 2, 4, 64, 20, 4)
    F, bad = FFA(), lambda f, *a, **kw: pytest.raises(RuntimeError, f, *a, **kw)
    q1, k1, v1 = (x[:, :, 0].contiguous() for x in (q, k, v))
    w = torch.zeros(2, 2, kc.shape[3], device=DEV)
    path, acc = ints([[0, 1], [0, 2]]), ints([1, 2])
    if what == "tree":
        bad(F.attention_tree, q, k, v, kc, vc, 1.0, 24)                                  # 24 + 4 > 27
        bad(F.attention_tree, q, k, v, kc, vc, 1.0, -1)
        bad(F.attention_tree, q[:, :3], k, v, kc, vc, 1.0, 20)                           # 3 query heads on 2
        bad(F.attention_tree, q, k[:, :, :3], v, kc, vc, 1.0, 20)
        bad(F.attention_tree, q.float(), k, v, kc, vc, 1.0, 20)
        bad(F.attention_tree, q.cpu(), k, v, kc, vc, 1.0, 20)
        bad(F.attention_tree, q[:, :, :0], k[:, :, :0], v[:, :, :0], kc, vc, 1.0, 20)
        bad(F.attention_tree, *(x[:, :, :1].expand(-1, -1, 65, -1) for x in (q, k, v)), kc, vc, 1.0, 20)
        for name in ("parents", "first_keys", "lengths", "counts"):
            bad(F.attention_tree, q, k, v, kc, vc, 1.0, 20, **{name: torch.zeros(2, 4 if name == "parents" else 1).to(DEV)})
            bad(F.attention_tree, q, k, v, kc, vc, 1.0, 20, **{name: torch.zeros(3, dtype=torch.int32, device=DEV)})
            bad(F.attention_tree, q, k, v, kc, vc, 1.0, 20, **{name: torch.zeros((2, 4) if name == "parents" else 2, dtype=torch.int32)})
        bad(F.attention_tree, q, k, v, kc[:, :, :, ::2], vc[:, :, ::2], 1.0, 4)
        bad(F.attention_tree, q, k[:, :0], v[:, :0], kc[:, :0].contiguous(), vc[:, :0].contiguous(), 1.0, 4)
    if what == "weights":
        bad(F.attention_weights, q1, k1, v1, kc, vc, 1.0, kc.shape[3], w)
        bad(F.attention_weights, q1, k1, v1, kc, vc, 1.0, 20, w[:, :, :-1])
        bad(F.attention_weights, q1, k1, v1, kc, vc, 1.0, 20, w.double())
        bad(F.attention_weights, q1, k1, v1, kc, vc, 1.0, 20, w.cpu())
        bad(F.attention_weights, q1[:, :3], k1, v1, kc, vc, 1.0, 20, w)
        bad(F.attention_weights, q1, q1, v1, kc, vc, 1.0, 20, w)
    if what == "commit":
        bad(F.commit_tree, [], 20, path, acc)
        bad(F.commit_tree, [(kc, vc)], 26, path, acc)                                    # two slots at 26 of 27
        bad(F.commit_tree, [(kc, vc)], 20, path.float(), acc)
        bad(F.commit_tree, [(kc, vc)], 20, path[:1], acc)
        bad(F.commit_tree, [(kc, vc)], 20, path, acc.cpu())
        bad(F.commit_tree, [(kc, vc), (kc.float(), vc.float())], 20, path, acc)
        bad(F.commit_tree, [(kc, vc), (kc.clone(), vc)], 20, path, acc)                  # one cache twice
    if what == "evict":
        bad(F.evict, [(kc, vc)], [w], 20, 0, 0)
        bad(F.evict, [(kc, vc)], [w], 20, 5, 6)
        bad(F.evict, [(kc, vc)], [w], 20, 5, -1)
        bad(F.evict, [(kc, vc)], [w], 28, 5, 1)
        bad(F.evict, [(kc, vc)], [w], 20, 28, 1)
        bad(F.evict, [(kc, vc)], [], 20, 5, 1)
        bad(F.evict, [(kc, vc)], [w.double()], 20, 5, 1)
        bad(F.evict, [(kc, vc), (kc, vc)], [w, w.clone()], 20, 5, 1)                     # the same cache twice
        bad(F.evict, [(kc, vc)], [w], 20, 5, 1, into=[(kc, vc.clone(), w[:, :, 1:])])
        other = torch.zeros(2, 2, kc.shape[3], 64, dtype=torch.float16, device=DEV)
        bad(F.evict, [(kc, vc)], [w], 20, 5, 1, into=[(kc, kc.view(2, 2, -1, 64), w)])  # V into K's buffer
        F.evict([(kc, vc)], [w], 20, 5, 1, into=[(kc, other, w)])
    torch.cuda.synchronize()


def test_rows_past_the_count_stay_as_they_were():
    """Through the C ABI, which writes only what is there unless it is asked for zeros; one piece and several."""
    import ctypes as C
    from fastforwardattention_amd import capi
    lib = capi.load()
    for t in (50, 9000):
        _, kc, vc, q, k, v = make(80, "fp16", 1, 2, 2, 64, t, 6)
        counts, K0 = ints([4]), kc.clone()
        for zero in (0, 1):
            out = torch.full((1, 6, 2, 64), 7.0, dtype=torch.float16, device=DEV).transpose(1, 2)
            tok = capi.TreeTokens()
            tok.tokens, tok.q_head_num, tok.counts, tok.zero_rest = 6, 2, counts.data_ptr(), zero
            for name, x in (("q_stride", q), ("k_stride", k), ("v_stride", v), ("out_stride", out)):
                getattr(tok, name)[:] = x.stride()[:3]
            n = lib.ffa_tree_workspace_bytes(16, 1, 2, 2, 64, 6, t)
            ws = torch.empty(n + 1, dtype=torch.uint8, device=DEV)
            p = [C.c_void_p(x.data_ptr()) for x in (q, k, v, kc, vc, out, ws)]
            rc = lib.ffa_attention_tree(16, 1, 2, 64, kc.shape[3], 0.125, t, C.byref(tok), *p, n, C.c_void_p(torch.cuda.current_stream().cuda_stream))
            assert rc == capi.FFA_OK
            torch.cuda.synchronize()
            assert bool((out[:, :, 4:] == (0.0 if zero else 7.0)).all()) and not bool((out[:, :, :4] == 7.0).any())
            want = FFA().attention_tree(q, k, v, kc, vc, 0.125, t, counts=counts)
            assert torch.equal(out[:, :, :4], want[:, :, :4])
            assert bool(kc[:, :, :, t + 4:].isnan().all()) and torch.equal(kc[:, :, :, :t], K0[:, :, :, :t])


def test_caches_of_more_than_four_gigabytes():
    """Offsets beyond 32 bits: the last pair's results against its own slots, in all four operators."""
    B, H, Dh, t, n = 2, 16, 128, 590_000, 5
    Lmax = t + 16
    g = torch.Generator(device=DEV).manual_seed(90)
    kc = torch.empty(B, H, Dh // 8, Lmax, 8, dtype=torch.float16, device=DEV).normal_(generator=g)
    vc = torch.empty(B, H, Lmax, Dh, dtype=torch.float16, device=DEV).normal_(generator=g)
    assert kc.numel() * 2 > 4 << 30
    q, k, v = (torch.empty(B, H, n, Dh, dtype=torch.float16, device=DEV).normal_(generator=g) for _ in range(3))
    last = slice(B - 1, B)
    K0, V0 = unpack_k(kc[last, -1:])[:, :, :t].clone(), vc[last, -1:, :t].clone()
    out = FFA().attention_tree(q, k, v, kc, vc, 0.05, t)
    want, size, bound, _ = tree_reference(q[last, -1:], k[last, -1:], v[last, -1:], K0, V0, 0.05, t)
    assert_close(out[last, -1:], want, tree_tolerance(q.dtype, want, size, bound, t + n, Dh), "long tree")
    assert torch.equal(unpack_k(kc[last, -1:])[:, :, t:t + n], k[last, -1:]) and torch.equal(vc[last, -1:, t:t + n], v[last, -1:])
    FFA().commit_tree([(kc, vc)], t, ints([[1, 4]] * B), ints([2] * B))
    assert torch.equal(vc[last, -1:, t:t + 2], v[last, -1:, [1, 4]].view(1, 1, 2, Dh))
    w = torch.rand(B, H, Lmax, generator=g, device=DEV)
    w0 = w[-1, -1].double()
    K1, V1 = unpack_k(kc[last, -1:])[:, :, :t + 2].clone(), vc[last, -1:, :t + 2].clone()
    out = FFA().attention_weights(q[:, :, 0].contiguous(), k[:, :, 0].contiguous(), v[:, :, 0].contiguous(), kc, vc, 0.05, t + 2, w)
    want, size, bound, p = tree_reference(q[last, -1:, :1], k[last, -1:, :1], v[last, -1:, :1], K1, V1, 0.05, t + 2)
    assert_close(out[last, -1:, None], want, tree_tolerance(q.dtype, want, size, bound, t + 3, Dh), "long weights")
    w0[:t + 2] += p[0][0, 0, 0, :-1]
    w0[t + 2] = p[0][0, 0, 0, -1]
    assert float((w[-1, -1, :t + 3].double() - w0[:t + 3]).abs().max()) <= 2.0 ** -23
    keep = t - 1000
    before = (unpack_k(kc[last, -1:])[0, 0].clone(), vc[-1, -1].clone(), w[-1, -1].clone())
    kept = FFA().evict([(kc, vc)], [w], t + 3, keep, 64)[0, -1, -1].long()
    rank = before[2][:t + 3].double()
    rank[t + 3 - 64:] = math.inf
    order = torch.sort(rank, descending=True, stable=True).indices[:keep].sort().values
    assert torch.equal(kept, order)
    assert torch.equal(unpack_k(kc[last, -1:])[0, 0, :keep], before[0][order]) and torch.equal(vc[-1, -1, :keep], before[1][order])
    assert torch.equal(w[-1, -1, :keep], before[2][order])


@pytest.mark.parametrize("in_place", [True, False])
def test_as_many_pairs_as_there_may_be(in_place):
    """2^18 pairs in 33 caches: more threads than one launch can have."""
    B, H, Dh, Lmax, layers = 1024, 256, 64, 2, 33
    g = torch.Generator(device=DEV).manual_seed(91)
    caches = [tuple(torch.empty(shape, dtype=torch.float16, device=DEV).normal_(generator=g)
                    for shape in ((B, H, Dh // 8, Lmax, 8), (B, H, Lmax, Dh))) for _ in range(layers)]
    weights = [torch.rand(B, H, Lmax, generator=g, device=DEV) for _ in range(layers)]
    second = [w[..., 1] > w[..., 0] for w in weights]
    want = [(torch.where(s[..., None, None], k[..., 1, :], k[..., 0, :]),
             torch.where(s[..., None], v[..., 1, :], v[..., 0, :]), w.amax(-1)) for s, (k, v), w in zip(second, caches, weights)]
    if in_place:
        to, to_w = caches, weights
        kept = FFA().evict(caches, weights, Lmax, 1, 0)
    else:
        to = [tuple(torch.zeros_like(x) for x in pair) for pair in caches]
        to_w = [torch.zeros_like(w) for w in weights]
        kept = FFA().evict(caches, weights, Lmax, 1, 0, into=[(k, v, w) for (k, v), w in zip(to, to_w)])
    for i in range(layers):
        assert torch.equal(kept[i, ..., 0], second[i].int())
        assert torch.equal(to[i][0][..., 0, :], want[i][0]), i
        assert torch.equal(to[i][1][..., 0, :], want[i][1]) and torch.equal(to_w[i][..., 0], want[i][2]), i
    one = [tuple(x[..., 1, :].clone() for x in pair) for pair in caches]
    FFA().commit_tree(caches, 0, ints([[1]] * B), ints([1] * B))
    for pair, rows in zip(caches, one):
        for x, row in zip(pair, rows):
            assert torch.equal(x[..., 0, :], row) and torch.equal(x[..., 1, :], row)


@pytest.mark.parametrize("t,keep", [(300, 200), (2500, 1700)])
def test_evict_keys_in_place_and_values_apart(t, keep):
    """One call with both: the keys stay in their cache, values and weights go to others."""
    B, H, Dh = 2, 3, 80
    g = torch.Generator(device=DEV).manual_seed(92)
    kc = torch.empty(B, H, Dh // 8, t, 8, dtype=torch.float16, device=DEV).normal_(generator=g)
    vc = torch.empty(B, H, t, Dh, dtype=torch.float16, device=DEV).normal_(generator=g)
    w = torch.rand(B, H, t, generator=g, device=DEV)
    lengths = ints([t, keep - 3])
    K0, V0, W0 = unpack_k(kc).clone(), vc.clone(), w.clone()
    v2, w2 = torch.full_like(vc, 7), torch.full_like(w, 7)
    kept = FFA().evict([(kc, vc)], [w], t, keep, 20, lengths=lengths, into=[(kc, v2, w2)])[0].long()
    assert torch.equal(vc, V0) and torch.equal(w, W0)
    for b, n in enumerate((keep, keep - 3)):
        assert bool((kept[b, :, n:] == -1).all())
        for h in range(H):
            order = kept[b, h, :n]
            rank = W0[b, h, :int(lengths[b])].double()
            rank[-20:] = math.inf
            want = torch.sort(rank, descending=True, stable=True).indices[:n].sort().values
            assert torch.equal(order, want)
            assert torch.equal(unpack_k(kc)[b, h, :n], K0[b, h, order]) and torch.equal(v2[b, h, :n], V0[b, h, order])
            assert torch.equal(w2[b, h, :n], W0[b, h, order])
        assert bool((v2[b, :, n:] == 7).all()) and bool((w2[b, :, n:] == 7).all())
