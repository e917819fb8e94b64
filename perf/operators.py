"""Workloads of the operators that work on the decode engine's caches: attention of a tree of
drafted tokens, the move of an accepted path, the decode step that sums attention weights, and
eviction by those sums.  Plain torch forms, and the calls of this package (`own`)."""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One user, a small candidate tree verified at the repository's headline prompt length: latency.
        _tree("tree 1x32x64 t1000 n8", "fp16", 1, 32, 32, 64, 1000, 8),
        # The headline batch in speculative decoding; the samples have accepted different numbers of tokens.
        _tree("tree 10x32x64 t1128 n32 ragged", "fp16", 10, 32, 32, 64, 1128, 32, ragged=True, counts=True),
        # Wide heads, a batch that was left-padded at the prompt.
        _tree("tree 8x16x256 t2000 n16 padded", "bf16", 8, 16, 16, 256, 2000, 16, padded=True),
        # Shared key heads over a long context: 4 query heads a key head, 96 query rows a pair.
        _tree("tree 2x8(32)x128 t20001 n24", "bf16", 2, 8, 32, 128, 20001, 24),
        # A chunk of a long prompt (or a long guess by look-up): a chain of 64 tokens on 8192 cached keys.
        _tree("chain 16x32x64 t8192 n64", "fp16", 16, 32, 32, 64, 8192, 64, chain=True),
        # fp32, a head dimension that is no power of two, odd sizes.
        _tree("tree 3x12x80 t777 n5 fp32", "fp32", 3, 12, 12, 80, 777, 5, padded=True),
        # The accepted path of one user in one layer: nothing but latency.
        _commit("commit 1x32x64 one layer", "fp16", 1, 1, 32, 64, 1256, 1000, 8, 5),
        # All layers of the headline model after one verification.
        _commit("commit 24 layers 10x32x64", "fp16", 24, 10, 32, 64, 1256, 1000, 32, 8),
        # One user's decode step under an eviction policy.
        _weights("weights 1x32x64 t1024", "fp16", 1, 32, 32, 64, 1024),
        # The long batch of the pruned sweep's shape.
        _weights("weights 16x32x64 t8192", "fp16", 16, 32, 32, 64, 8192),
        # One layer's prompt of one user halved into a smaller cache.
        _evict("evict 1x32x64 1000 to 500", "fp16", 1, 1, 32, 64, 1000, 500, 100),
        # Four layers of the wide-head shape cut back in place during a decode.
        _evict("evict 4 layers 8x16x256 2256 to 1000", "fp16", 4, 8, 16, 256, 2256, 1000, 200, in_place=True, padded=True),
    ]


def _tree(name, dtype, B, H, Hq, Dh, t, n, chain=False, ragged=False, padded=False, counts=False):
    return {"name": name, "op": "tree", "dtype": dtype, "B": B, "H": H, "Hq": Hq, "Dh": Dh, "t": t, "n": n,
            "chain": chain, "ragged": ragged, "padded": padded, "counts": counts}


def _commit(name, dtype, layers, B, H, Dh, Lmax, t, n, m):
    return {"name": name, "op": "commit", "dtype": dtype, "layers": layers, "B": B, "H": H, "Dh": Dh, "Lmax": Lmax,
            "t": t, "n": n, "m": m}


def _weights(name, dtype, B, H, Hq, Dh, t, ragged=False, padded=False):
    return {"name": name, "op": "weights", "dtype": dtype, "B": B, "H": H, "Hq": Hq, "Dh": Dh, "t": t,
            "ragged": ragged, "padded": padded}


def _evict(name, dtype, layers, B, H, Dh, t, keep, recent, in_place=False, ragged=False, padded=False):
    return {"name": name, "op": "evict", "dtype": dtype, "layers": layers, "B": B, "H": H, "Dh": Dh, "t": t,
            "keep": keep, "recent": recent, "in_place": in_place, "ragged": ragged, "padded": padded}


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(["tree", "tree", "commit", "weights", "evict"])
        dtype, Dh = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"]), rng.choice([64, 80, 128, 256])
        B, H = spread(1, 16), rng.choice([1, 4, 8, 12, 16, 25, 32])
        t = spread(1, 32000)
        flags = {k: rng.random() < 0.4 for k in ("ragged", "padded")}
        if op == "tree":
            c = _tree("", dtype, B, H, H * rng.choice([1, 1, 2, 4, 8]), Dh, t, spread(1, 64), chain=rng.random() < 0.3,
                      counts=rng.random() < 0.3, **flags)
        elif op == "commit":
            n = spread(1, 64)
            c = _commit("", dtype, spread(1, 32), B, H, Dh, t + n + rng.randrange(0, 100), t, n, rng.randint(1, n))
        elif op == "weights":
            c = _weights("", dtype, B, H, H * rng.choice([1, 1, 2, 4, 8]), Dh, t, **flags)
        else:
            t = max(t, 16)
            keep = rng.randint(1, t)
            c = _evict("", dtype, spread(1, 16), B, H, Dh, t, keep, rng.randint(0, keep), in_place=rng.random() < 0.5, **flags)
        w = work(c)
        # As dear as the largest listed case at most, in bytes and in operations, and small enough to hold three times.
        if w["bytes"] <= 1.2e9 and w["flops"] <= 7e10 and _held(c) <= 1e10:
            del c["name"]
            return c


def _held(c):
    """Bytes of the caches."""
    slots = {"tree": c["t"] + c.get("n", 0), "commit": c.get("Lmax"), "weights": c["t"] + 1, "evict": c["t"] + 8}[c["op"]]
    return 2 * c.get("layers", 1) * c["B"] * c["H"] * slots * c["Dh"] * _size(c)


def _size(c):
    return 4 if c["dtype"] == "fp32" else 2


def work(c):
    e, B, H, Dh = _size(c), c["B"], c["H"], c["Dh"]
    row = 2 * B * H * Dh * e      # one slot of every pair, K and V
    if c["op"] == "tree":
        n, t, Hq = c["n"], c["t"], c["Hq"]
        return {"bytes": row * (t + 2 * n) + 2 * B * Hq * n * Dh * e, "flops": 4 * B * Hq * n * (t + n / 2) * Dh}
    if c["op"] == "commit":
        return {"bytes": c["layers"] * 2 * row * (c["m"] + 1) / 2 + 4 * B * (c["m"] + 2), "flops": 0}
    if c["op"] == "weights":
        t, Hq = c["t"], c["Hq"]
        return {"bytes": row * (t + 2) + 2 * B * Hq * Dh * e + 8 * B * H * t, "flops": 4 * B * Hq * t * Dh}
    t, keep = c["t"], c["keep"]
    return {"bytes": c["layers"] * (2 * row * keep + 4 * B * H * (t + 2 * keep)), "flops": 0}


# ----------------------------------------------------------------------------------------------
# What a program has in hand.

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = DTYPES[c["dtype"]], "cuda"
    x = 16 // _size(c)
    B, H, Dh, t, op = c["B"], c["H"], c["Dh"], c["t"], c["op"]

    def randn(*shape, scale=1.0, dtype=dt):
        return torch.empty(shape, device=dev, dtype=dtype).normal_(0.0, scale, generator=g)

    def ints(lo, hi, *shape):     # lo .. hi inclusive
        return torch.randint(lo, hi + 1, shape, generator=g, device=dev, dtype=torch.int32)

    s = {"case": c, "t": t, "scale": 1.0 / math.sqrt(Dh)}
    s["first"] = ints(0, t // 4, B) if c.get("padded") else None
    s["lengths"] = ints(max(0, t - max(1, t // 8)), t, B) if c.get("ragged") else None
    if op in ("tree", "weights"):
        n, Hq = c.get("n", 1), c["Hq"]
        Lmax = -(-(t + n) // 8) * 8
        s["k_cache"], s["v_cache"] = randn(B, H, Dh // x, Lmax, x), randn(B, H, Lmax, Dh)
        # Projections come out token by token, heads side by side.
        s["q"], s["k"], s["v"] = (randn(B, n, h, Dh).transpose(1, 2) for h in (Hq, H, H))
        if op == "tree":
            i = torch.arange(n, device=dev, dtype=torch.int32)
            s["parents"] = None if c["chain"] else (i - 1 - (torch.rand(B, n, generator=g, device=dev) * torch.clamp(i + 1, max=6)).int()).int()
            s["counts"] = ints(max(1, n // 2), n, B) if c["counts"] else None
        else:
            s["q"], s["k"], s["v"] = (y.reshape(B, -1, Dh) for y in (s["q"], s["k"], s["v"]))
            s["key_weights"] = torch.rand(B, H, Lmax, generator=g, device=dev)
        return s
    layers = c["layers"]
    if op == "commit":
        Lmax, n, m = c["Lmax"], c["n"], c["m"]
        # m of the n nodes in order; the samples accepted 1 .. m of them.
        path = torch.argsort(torch.rand(B, n, generator=g, device=dev), dim=1)[:, :m]
        s["path"], s["accepted"] = torch.sort(path, dim=1).values.int().contiguous(), ints(1, m, B)
        s["lengths"] = ints(max(0, t - 16), t, B)
        s["K"], s["V"] = randn(layers, B, H, Dh // x, Lmax, x), randn(layers, B, H, Lmax, Dh)
        return s
    Lmax = -(-(t + 8) // 8) * 8
    s["K"], s["V"] = randn(layers, B, H, Dh // x, Lmax, x), randn(layers, B, H, Lmax, Dh)
    # Sums of attention weights: few heavy keys, a long light tail; a key that was hardly seen may have none at all.
    w = torch.empty(layers, B, H, Lmax, device=dev).exponential_(1.0, generator=g) ** 4
    s["W"] = torch.where(torch.rand(layers, B, H, Lmax, generator=g, device=dev) < 0.05, torch.zeros_like(w), w)
    if c["in_place"]:
        s["K_to"], s["V_to"] = s["K"], s["V"]
    else:
        Lto = -(-(c["keep"] + 8) // 8) * 8
        s["K_to"], s["V_to"] = randn(layers, B, H, Dh // x, Lto, x), randn(layers, B, H, Lto, Dh)
    s["W_to"] = torch.zeros(layers, B, H, s["V_to"].shape[3], device=dev)
    return s


# ----------------------------------------------------------------------------------------------
# One pass.

def run(s):
    return {"tree": _run_tree, "commit": _run_commit, "weights": _run_weights, "evict": _run_evict}[s["case"]["op"]](s)


def _run_tree(s):
    if own:
        from fastforwardattention_amd import FastForwardAttn
        out = FastForwardAttn.attention_tree(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["scale"], s["t"],
                                             s["parents"], first_keys=s["first"], lengths=s["lengths"], counts=s["counts"])
    else:
        out = _plain_tree(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["scale"], s["t"], s["parents"], s["first"],
                          s["lengths"], s["counts"])[0]
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_weights(s):
    if own:
        from fastforwardattention_amd import FastForwardAttn
        out = FastForwardAttn.attention_weights(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["scale"], s["t"],
                                                s["key_weights"], first_keys=s["first"], lengths=s["lengths"])
    else:
        t, B = s["t"], s["q"].shape[0]
        out, p = _plain_tree(s["q"][:, :, None], s["k"][:, :, None], s["v"][:, :, None], s["k_cache"], s["v_cache"],
                             s["scale"], t, None, s["first"], s["lengths"], None)
        out = out[:, :, 0]
        p, w = p.sum(2), s["key_weights"]            # [B,H,t+1]: cached slots, then the new token
        at = _per_sample(s["lengths"], t, B, w.device)[:, None, None].expand(B, w.shape[1], 1).long()
        w[:, :, :t] += p[:, :, :t]
        w.scatter_(2, at, p[:, :, t:])
    return {"out": out, "key_weights": s["key_weights"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_commit(s):
    if own:
        from fastforwardattention_amd import FastForwardAttn
        FastForwardAttn.commit_tree(list(zip(s["K"].unbind(0), s["V"].unbind(0))), s["t"], s["path"], s["accepted"],
                                    lengths=s["lengths"])
    else:
        K, V, m = s["K"], s["V"], s["path"].shape[1]
        B = K.shape[1]
        b = torch.arange(B, device=K.device)[:, None]
        j = torch.arange(m, device=K.device)[None]
        base = s["lengths"].long()[:, None]
        to, at = base + j, base + torch.where(j < s["accepted"][:, None], s["path"].long(), j)
        k, v = K.permute(1, 4, 0, 2, 3, 5), V.permute(1, 3, 0, 2, 4)      # [B, slot, ...]
        k[b, to] = k[b, at]
        v[b, to] = v[b, at]
    return {"K": s["K"], "V": s["V"]}


def _run_evict(s):
    c = s["case"]
    if own:
        from fastforwardattention_amd import FastForwardAttn
        kept = FastForwardAttn.evict(list(zip(s["K"].unbind(0), s["V"].unbind(0))), list(s["W"].unbind(0)), s["t"], c["keep"],
                                     c["recent"], first_keys=s["first"], lengths=s["lengths"],
                                     into=list(zip(s["K_to"].unbind(0), s["V_to"].unbind(0), s["W_to"].unbind(0))))
    else:
        t, keep, K, V = s["t"], c["keep"], s["K"], s["V"]
        N, B, H = K.shape[:3]
        j = torch.arange(t, device=K.device)
        length = _per_sample(s["lengths"], t, B, K.device)[None, :, None, None]
        first = _per_sample(s["first"], 0, B, K.device)[None, :, None, None]
        # Classes from the top: the last `recent`, real keys by weight, padding, slots behind the sample's length.
        rank = torch.where(j < first, -1.0, s["W"][..., :t])
        rank = torch.where(j >= length - c["recent"], math.inf, rank)
        rank = torch.where(j >= length, -2.0, rank)
        order = torch.sort(rank, dim=3, descending=True, stable=True).indices[..., :keep]
        order = torch.sort(order, dim=3).values
        there = order < length
        kept = torch.where(there, order, -1).int()
        Dh, x, nch = V.shape[4], K.shape[5], K.shape[3]
        k = torch.gather(K, 4, order[:, :, :, None, :, None].expand(N, B, H, nch, keep, x))
        v = torch.gather(V, 3, order[..., None].expand(N, B, H, keep, Dh))
        w = torch.gather(s["W"], 3, order)
        s["K_to"][:, :, :, :, :keep] = torch.where(there[:, :, :, None, :, None], k, s["K_to"][:, :, :, :, :keep])
        s["V_to"][:, :, :, :keep] = torch.where(there[..., None], v, s["V_to"][:, :, :, :keep])
        s["W_to"][..., :keep] = torch.where(there, w, s["W_to"][..., :keep])
    return {"kept": kept, "K": s["K_to"], "V": s["V_to"], "W": s["W_to"]}


def _per_sample(x, value, B, device):
    return torch.full((B,), value, device=device, dtype=torch.int32) if x is None else x


def _plain_tree(q, k, v, k_cache, v_cache, scale, t, parents, first, lengths, counts):
    """out [B,Hq,n,Dh] in q's type, weights [B,H,G*n,t+n] in 32 bits; appends k and v."""
    B, Hq, n, Dh = q.shape
    H, dev = k.shape[1], q.device
    G = Hq // H
    first, length = _per_sample(first, 0, B, dev), _per_sample(lengths, t, B, dev)
    count = _per_sample(counts, n, B, dev)
    i = torch.arange(n, device=dev)
    if parents is None:
        seen = (i[:, None] >= i[None]).expand(B, n, n)
    else:   # ancestors by squaring the parent relation: 64 nodes are at most 63 steps from the root
        seen = (i[None, :, None] == i[None, None]) | (parents[:, :, None] == i[None, None])
        for _ in range(6):
            seen = torch.matmul(seen.float(), seen.float()) > 0
    key = torch.arange(t, device=dev)
    old = (key >= first[:, None]) & (key < length[:, None])                               # [B,t]
    mask = torch.cat([old[:, None].expand(B, n, t), seen], 2)[:, None, None].expand(B, H, G, n, t + n).reshape(B, H, G * n, t + n)
    qf = q.float().reshape(B, H, G * n, Dh)
    kt = k_cache[:, :, :, :t].permute(0, 1, 2, 4, 3).float().reshape(B, H, Dh, t)
    kt = torch.cat([kt, k.float().transpose(2, 3)], 3)
    z = (torch.matmul(qf, kt) * scale).masked_fill_(~mask, -math.inf)
    z = torch.exp(z - z.amax(3, keepdim=True))
    z = z / z.sum(3, keepdim=True)
    vf = torch.cat([v_cache[:, :, :t].float(), v.float()], 2)
    out = torch.matmul(z, vf).reshape(B, Hq, n, Dh)
    out = torch.where((i < count[:, None])[:, None, :, None], out, 0.0).to(q.dtype)
    b, slot = torch.arange(B, device=dev)[:, None], length.long()[:, None] + i
    real = (i < count[:, None])[:, :, None, None]
    kc, vc = k_cache.permute(0, 3, 1, 2, 4), v_cache.permute(0, 2, 1, 3)                   # [B,slot,...]
    kn = k.transpose(1, 2).reshape(B, n, H, kc.shape[3], kc.shape[4])
    kc[b, slot] = torch.where(real[..., None], kn, kc[b, slot])
    vc[b, slot] = torch.where(real, v.transpose(1, 2), vc[b, slot])
    return out, z


# ----------------------------------------------------------------------------------------------
# The definitions in 64 bits, sample by sample.

def exact(c, seed):
    s = prepare(c, seed)
    op, B, t, n = c["op"], c["B"], c["t"], c.get("n", 1)
    if op == "commit":
        K, V = s["K"].double(), s["V"].double()
        K0, V0 = K.clone(), V.clone()
        for b in range(B):
            at = int(s["lengths"][b])
            for j, node in enumerate(s["path"][b, : int(s["accepted"][b])].tolist()):
                K[:, b, :, :, at + j], V[:, b, :, at + j] = K0[:, b, :, :, at + node], V0[:, b, :, at + node]
        return {"K": K, "V": V}
    if op == "evict":
        return None if c["layers"] * B * c["H"] * t > 4e6 else _exact_evict(c, s)
    q, k, v = (y.double() if y.dim() == 4 else y[:, :, None].double() for y in (s["q"], s["k"], s["v"]))
    H, G = c["H"], c["Hq"] // c["H"]
    out = torch.zeros_like(q)
    w = s["key_weights"].double() if op == "weights" else None
    for b in range(B):
        length = t if s["lengths"] is None else int(s["lengths"][b])
        first = 0 if s["first"] is None else int(s["first"][b])
        first = min(first, length)
        nodes = n if s.get("counts") is None else int(s["counts"][b])
        up = list(range(-1, n - 1)) if s.get("parents") is None else s["parents"][b].tolist()
        blocked = torch.ones(n, n, dtype=torch.bool)
        for i in range(n):
            a = i
            while a >= 0:
                blocked[i, a] = False
                a = up[a]
        K = s["k_cache"][b, :, :, first:length].permute(0, 2, 1, 3).reshape(H, length - first, -1).double()
        K, V = torch.cat([K, k[b]], 1), torch.cat([s["v_cache"][b, :, first:length].double(), v[b]], 1)
        z = torch.bmm(q[b].reshape(H, G * n, -1), K.transpose(1, 2).contiguous()) * s["scale"]
        z = z.view(H, G, n, -1)
        z[..., length - first:] = z[..., length - first:].masked_fill(blocked.to(z.device), -math.inf)
        p = torch.softmax(z, -1)
        out[b, :, :nodes] = torch.bmm(p.view(H, G * n, -1), V).view(H * G, n, -1)[:, :nodes]
        if w is not None:
            total = p.sum((1, 2))
            w[b, :, first:length] += total[:, :-1]
            w[b, :, length] = total[:, -1]
    if op == "weights":
        return {"out": out[:, :, 0], "key_weights": w, "k_cache": None, "v_cache": None}
    return {"out": out, "k_cache": None, "v_cache": None}


def _exact_evict(c, s):
    """Each pair by itself, on the host: a list of (class, weight, slot), sorted."""
    import numpy as np
    K, V, W = s["K_to"].double(), s["V_to"].double(), s["W_to"].double()
    weights = s["W"].cpu().numpy().astype(np.float64)
    for b in range(c["B"]):
        length = c["t"] if s["lengths"] is None else int(s["lengths"][b])
        first = 0 if s["first"] is None else int(s["first"][b])
        slot = np.arange(length)
        tier = np.where(slot >= length - c["recent"], 2, np.where(slot < first, 0, 1))
        for a in range(c["layers"]):
            for h in range(c["H"]):
                w = np.where(tier == 1, weights[a, b, h, :length], 0.0)
                chosen = np.sort(np.lexsort((slot, -w, -tier))[: c["keep"]])
                at = torch.from_numpy(chosen).to(K.device)
                K[a, b, h, :, : len(chosen)] = s["K"][a, b, h][:, at].double()
                V[a, b, h, : len(chosen)] = s["V"][a, b, h][at].double()
                W[a, b, h, : len(chosen)] = s["W"][a, b, h][at].double()
    return {"kept": None, "K": K, "V": V, "W": W}
