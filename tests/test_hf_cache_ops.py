"""Hugging Face hook: passes of several tokens after the prompt, cropping, prompt-lookup and assisted
decoding, and the bounded cache with eviction.  On the CPU a plain float64 stand-in answers for the
engine's operators (it checks the hook's bookkeeping); the GPU tests run the real extension."""
import math

import pytest
import torch

from tests.cache_ops_testlib import evict_reference, tree_reference
from tests.test_hf_shim import OracleEngine, padded_batch, small_gptj, teacher_forced_logits, tiny_gptj, tiny_opt

transformers = pytest.importorskip("transformers")
from fastforwardattention_amd import hf  # noqa: E402


def as_rows(kc):
    B, H, nch, L, x = kc.shape
    return kc.permute(0, 1, 3, 2, 4).reshape(B, H, L, nch * x)


class PlainEngine(OracleEngine):
    """The operators next to the decode step in their plain form, on CPU tensors."""

    calls_of_groups = 0

    @staticmethod
    def _append(kc, vc, t, k, v):
        n = k.shape[2]
        assert t + n <= vc.shape[2]
        kc[:, :, :, t:t + n] = k.reshape(*k.shape[:3], kc.shape[2], kc.shape[4]).permute(0, 1, 3, 2, 4)
        vc[:, :, t:t + n] = v

    @staticmethod
    def attention_tree(q, k, v, kc, vc, scale, t, parents=None, first_keys=None, lengths=None, counts=None):
        assert k.shape[2] <= 64
        PlainEngine.calls_of_groups += 1
        out = tree_reference(q, k, v, as_rows(kc), vc, scale, t, parents, first_keys, lengths, counts)[0]
        PlainEngine._append(kc, vc, t, k, v)
        return out.to(q.dtype)

    @staticmethod
    def attention_weights(q, k, v, kc, vc, scale, t, w, first_keys=None, lengths=None):
        B, H, Dh = kc.shape[0], kc.shape[1], vc.shape[3]
        q, k, v = (x.reshape(B, -1, 1, Dh) for x in (q, k, v))
        out, _, _, p = tree_reference(q, k, v, as_rows(kc), vc, scale, t, first_keys=first_keys)
        PlainEngine._append(kc, vc, t, k, v)
        for b in range(B):
            f = 0 if first_keys is None else min(int(first_keys[b]), t)
            s = p[b].sum((1, 2)).to(w.dtype)
            w[b, :, f:t] += s[:, :-1]
            w[b, :, t] = s[:, -1]
        return out[:, :, 0].to(q.dtype)

    @staticmethod
    def evict(caches, weights, t, keep, recent, first_keys=None, lengths=None, into=None):
        into = [(k, v, w) for (k, v), w in zip(caches, weights)] if into is None else into
        for (k, v), w, (k2, v2, w2) in zip(caches, weights, into):
            for b in range(w.shape[0]):
                for h in range(w.shape[1]):
                    stay = evict_reference(w[b, h].tolist(), t, 0 if first_keys is None else min(int(first_keys[b]), t), keep, recent)
                    n = len(stay)
                    k2[b, h, :, :n], v2[b, h, :n], w2[b, h, :n] = k[b, h][:, stay].clone(), v[b, h, stay].clone(), w[b, h, stay].clone()


def chunked_logits(model, ids, mask, pieces, cache):
    """Feeds ids in pieces; the logits of every position, padding included."""
    out, at, logits = None, 0, []
    with torch.no_grad():
        for n in pieces:
            part, m = ids[:, at:at + n], mask[:, :at + n]
            pos = (m.long().cumsum(-1) - 1).clamp(min=0)[:, -n:]
            kw = {"position_ids": pos} if "GPTJ" in type(model).__name__ else {}
            out = model(input_ids=part, attention_mask=m, past_key_values=cache, use_cache=True, **kw)
            cache = out.past_key_values
            logits.append(out.logits.float())
            at += n
    return torch.cat(logits, 1), cache


def long_ids(device="cpu", length=40):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(3, 96, (2, length), generator=g).to(device)
    mask = torch.ones_like(ids)
    ids[1, :4] = 1
    mask[1, :4] = 0
    return ids, mask


def check_chunks(model, ids, mask, pieces, engine, tol):
    want, _ = chunked_logits(model, ids, mask, [ids.shape[1]], None)
    hf.enable(model)
    got, cache = chunked_logits(model, ids, mask, pieces, hf.FFACache(max_new_tokens=ids.shape[1] - pieces[0], **engine))
    hf.disable(model)
    real = mask.bool()
    assert float((got - want)[real].abs().max()) < tol
    assert cache.get_seq_length() == ids.shape[1]
    return cache


@pytest.mark.parametrize("family", ["opt", "gptj"])
def test_prompt_in_chunks(family):
    model = tiny_opt() if family == "opt" else tiny_gptj()
    ids, mask = long_ids()
    for pieces in ([9, 31], [9, 1, 2, 20, 8]):
        check_chunks(model, ids, mask, pieces, dict(engine=PlainEngine), 2e-4)


def test_group_of_more_than_64_tokens_is_cut():
    model = small_gptj()
    ids, mask = long_ids(length=150)
    PlainEngine.calls_of_groups = 0
    check_chunks(model, ids, mask, [10, 140], dict(engine=PlainEngine), 2e-4)
    assert PlainEngine.calls_of_groups == 2 * 3          # 64 + 64 + 12, in two layers


def test_crop_and_go_on():
    """Tokens that are taken back leave no trace."""
    model = tiny_opt()
    ids, mask = long_ids()
    want, _ = chunked_logits(model, ids, mask, [40], None)
    hf.enable(model)
    cache = hf.FFACache(max_new_tokens=35, engine=PlainEngine)
    wrong = ids.clone()
    wrong[:, 20:] = 50
    _, cache = chunked_logits(model, wrong[:, :26], mask[:, :26], [9, 17], cache)
    cache.crop(20)
    with torch.no_grad():
        out = model(input_ids=ids[:, 20:], attention_mask=mask, past_key_values=cache, use_cache=True)
    assert float((out.logits.float() - want[:, 20:]).abs().max()) < 2e-4
    cache.crop(-1)
    assert cache.get_seq_length() == 39
    with torch.no_grad():
        out = model(input_ids=ids[:, 39:], attention_mask=mask, past_key_values=cache, use_cache=True)
    assert float((out.logits[:, -1].float() - want[:, 39]).abs().max()) < 2e-4
    hf.disable(model)


def check_assisted(device, engine, dtype=torch.float32, **kw):
    model = tiny_opt(dtype).to(device)
    ids = torch.tensor([[5, 6, 7, 8, 5, 6, 7, 9, 10, 5, 6, 7]], device=device)
    common = dict(attention_mask=torch.ones_like(ids), max_new_tokens=16, do_sample=False, pad_token_id=1, eos_token_id=None)
    want = model.generate(ids, **common)
    if "assistant_model" in kw:
        kw["assistant_model"] = tiny_opt(dtype).to(device)
    hf.enable(model)
    cache = hf.FFACache(max_new_tokens=24, **engine)
    got = model.generate(ids, past_key_values=cache, **common, **kw)
    hf.disable(model)
    assert torch.equal(got, want)
    return cache


@pytest.mark.parametrize("how", ["lookup", "assistant"])
def test_speculative_generate_equals_greedy(how):
    PlainEngine.calls_of_groups = 0
    check_assisted("cpu", dict(engine=PlainEngine), **({"prompt_lookup_num_tokens": 4} if how == "lookup" else {"assistant_model": True}))
    assert PlainEngine.calls_of_groups > 0


# ------------------------------------------------------------------------------------------------
class BoundedReference:
    """Attention over full histories with, per layer, sample and head, a list of living tokens and their
    weights: the eviction policy by its definition, without any cache of slots."""

    def __init__(self, keep, recent, evict_every, first):
        self.keep, self.recent, self.cap, self.first = keep, recent, keep + evict_every, first
        self.layers = {}

    def __call__(self, module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kw):
        scale = query.shape[-1] ** -0.5 if scaling is None else scaling
        B, H, n, Dh = query.shape
        K, V = key.double(), value.double()               # the model's own cache hands over the whole history
        T = K.shape[2]
        if id(module) not in self.layers:
            z = query.double() @ K.transpose(-1, -2) * scale
            z = z + attention_mask.double()
            p = torch.softmax(z, -1)
            alive = [[None] * H for _ in range(B)]
            for b in range(B):
                for h in range(H):
                    w = p[b, h, self.first[b]:].sum(0).tolist()
                    stay = evict_reference(w, T, self.first[b], self.keep, self.recent)
                    alive[b][h] = [[j, w[j]] for j in stay]
            self.layers[id(module)] = alive
            return (p @ V).to(query.dtype).transpose(1, 2).contiguous(), None
        alive, out = self.layers[id(module)], torch.zeros(B, 1, H, Dh, dtype=torch.float64)
        for b in range(B):
            for h in range(H):
                a = alive[b][h]
                if len(a) == self.cap:
                    pads = sum(1 for j, _ in a if j < self.first[b])
                    a = alive[b][h] = [a[j] for j in evict_reference([w for _, w in a], len(a), pads, self.keep, self.recent)]
                a.append([T - 1, 0.0])
                use = [x for x in a if x[0] >= self.first[b]]
                at = [j for j, _ in use]
                p = torch.softmax(K[b, h, at] @ query[b, h, 0].double() * scale, 0)
                for x, w in zip(use, p.tolist()):
                    x[1] += w
                out[b, 0, h] = p @ V[b, h, at]
        return out.to(query.dtype), None


def check_bounded(device, engine, tol, dtype=torch.float32, keep=8, recent=3, evict_every=4, steps=24):
    model = tiny_opt(dtype).to(device)
    ids, mask = padded_batch(device)
    from transformers.masking_utils import AttentionMaskInterface, eager_mask
    from transformers.modeling_utils import AttentionInterface
    ref = BoundedReference(keep, recent, evict_every, [0, 4])
    AttentionInterface.register("bounded_reference", lambda module, q, k, v, m, **kw: tuple(
        x if x is None else x.to(device) for x in ref(module, q.cpu(), k.cpu(), v.cpu(), None if m is None else m.cpu(), **kw)))
    AttentionMaskInterface.register("bounded_reference", eager_mask)
    before = model.config._attn_implementation
    model.config._attn_implementation = "bounded_reference"
    want, _ = teacher_forced_logits(model, ids, mask, steps, None)
    model.config._attn_implementation = before
    hf.enable(model)
    got, cache = teacher_forced_logits(model, ids, mask, steps,
                                       hf.FFACache(max_new_tokens=steps, keep=keep, recent=recent, evict_every=evict_every, **engine))
    hf.disable(model)
    assert float((got - want).abs().max()) < tol
    layer = cache.layers[0]
    assert cache.get_seq_length() == ids.shape[1] + steps and layer.bounded[1].shape[2] == keep + evict_every
    assert keep < layer.t <= keep + evict_every
    return layer


def test_bounded_cache_follows_its_definition():
    layer = check_bounded("cpu", dict(engine=PlainEngine), 2e-4)
    assert layer.first_key.tolist() == [0, 0]             # the short sample's padding went first


def test_bounded_cache_with_room_for_all_is_exact():
    for make in (tiny_opt, tiny_gptj):
        model = make()
        ids, mask = padded_batch()
        want, _ = teacher_forced_logits(model, ids, mask, 6, None)
        hf.enable(model)
        got, cache = teacher_forced_logits(model, ids, mask, 6, hf.FFACache(max_new_tokens=6, engine=PlainEngine, keep=9, evict_every=6))
        hf.disable(model)
        assert float((got - want).abs().max()) < 2e-4


def test_bounded_cache_refusals():
    for bad in (dict(keep=0), dict(keep=4, recent=5), dict(keep=4, recent=-1), dict(keep=4, evict_every=0), dict(keep=4, num_beams=2),
                dict(keep=4, prob_thresh=0.1)):
        with pytest.raises(ValueError):
            hf.FFALayer(4, **bad)
    model = tiny_opt()
    ids, mask = padded_batch()
    hf.enable(model)
    with pytest.raises(NotImplementedError, match="keep="), torch.no_grad():
        model(input_ids=ids, attention_mask=mask, past_key_values=hf.FFACache(max_new_tokens=4, engine=OracleEngine, keep=4), use_cache=True)
    # several tokens at once: not with an engine that has no attention_tree, nor with a bounded cache
    for kw in (dict(engine=OracleEngine), dict(engine=PlainEngine, keep=4)):
        cache = hf.FFACache(max_new_tokens=8, **kw)
        with torch.no_grad():
            model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True)
            with pytest.raises(NotImplementedError, match="several tokens"):
                model(input_ids=torch.full((2, 3), 40), attention_mask=torch.cat([mask, torch.ones(2, 3, dtype=mask.dtype)], 1),
                      past_key_values=cache, use_cache=True)
    with pytest.raises(NotImplementedError):
        cache.crop(3)
    # more tokens than the cache has room for
    cache = hf.FFACache(max_new_tokens=2, engine=PlainEngine)
    with torch.no_grad():
        model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True)
        with pytest.raises(RuntimeError, match="cache full"):
            model(input_ids=torch.full((2, 3), 40), attention_mask=torch.cat([mask, torch.ones(2, 3, dtype=mask.dtype)], 1),
                  past_key_values=cache, use_cache=True)
    hf.disable(model)


# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("family,dtype,tol", [("opt", torch.float32, 2e-4), ("gptj", torch.float32, 2e-4), ("opt", torch.float16, 3e-2),
                                               ("gptj", torch.float16, 3e-2)])
def test_prompt_in_chunks_with_hip_engine(family, dtype, tol):
    print("chunks", family, dtype, flush=True)
    model = (tiny_opt(dtype) if family == "opt" else tiny_gptj(dtype)).to("cuda:0")
    ids, mask = long_ids("cuda:0")
    for pieces in ([9, 31], [9, 1, 2, 20, 8]):
        check_chunks(model, ids, mask, pieces, {}, tol)
    if family == "gptj":
        ids, mask = long_ids("cuda:0", 700)
        check_chunks(small_gptj(dtype).to("cuda:0"), ids, mask, [300, 400], {}, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["lookup", "assistant"])
def test_speculative_generate_with_hip_engine(how):
    print("speculative generate", how, flush=True)
    check_assisted("cuda:0", {}, **({"prompt_lookup_num_tokens": 4} if how == "lookup" else {"assistant_model": True}))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4)])
def test_bounded_cache_with_hip_engine(dtype, tol):
    print("bounded", dtype, flush=True)
    check_bounded("cuda:0", {}, tol, dtype)
    for make in (tiny_opt, tiny_gptj):
        model = make(dtype).to("cuda:0")
        ids, mask = padded_batch("cuda:0")
        want, _ = teacher_forced_logits(model, ids, mask, 6, None)
        hf.enable(model)
        got, cache = teacher_forced_logits(model, ids, mask, 6, hf.FFACache(max_new_tokens=6, keep=9, evict_every=6))
        hf.disable(model)
        assert float((got - want).abs().max()) < tol
