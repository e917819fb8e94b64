"""Hugging Face hook: the attention mask of a pass of several tokens after the prompt.  Left padding may be as
long as the first chunk and longer; a mask that is not left padding and causal order is refused.  On the CPU the
plain stand-in of tests/test_hf_cache_ops.py answers for the engine."""
import pytest
import torch

from tests.test_hf_cache_ops import PlainEngine, check_chunks, chunked_logits, long_ids
from tests.test_hf_shim import OracleEngine, padded_batch, small_gptj, tiny_gptj, tiny_opt

transformers = pytest.importorskip("transformers")
from fastforwardattention_amd import hf  # noqa: E402

MAKE = {"opt": tiny_opt, "gptj": tiny_gptj}


def padded_ids(pad, device="cpu", length=40):
    ids, _ = long_ids(device, length)
    mask = torch.ones_like(ids)
    ids[1, :pad], mask[1, :pad] = 1, 0
    return ids, mask


@pytest.mark.parametrize("family", ["opt", "gptj"])
@pytest.mark.parametrize("pad", [8, 9, 10, 14, 39])
def test_padding_longer_than_the_first_chunk(family, pad):
    model = MAKE[family]()
    ids, mask = padded_ids(pad)
    for pieces in ([9, 31], [9, 1, 2, 20, 8], [9, 3, 3, 25], [9] + [1] * 31, [1] * 40):
        check_chunks(model, ids, mask, pieces, dict(engine=PlainEngine), 2e-4)


def test_padding_longer_than_64_tokens_of_a_chunk():
    model = small_gptj()
    ids, mask = padded_ids(100, length=150)
    for pieces in ([10, 140], [10, 64, 76], [100, 50]):
        check_chunks(model, ids, mask, pieces, dict(engine=PlainEngine), 2e-4)


@pytest.mark.parametrize("family", ["opt", "gptj"])
def test_generate_with_a_prompt_in_chunks(family):
    """generate(prefill_chunk_size=...) on a batch whose short sample begins behind the first chunk."""
    model = MAKE[family]()
    ids, mask = padded_ids(14, length=24)
    common = dict(attention_mask=mask, max_new_tokens=8, do_sample=False, pad_token_id=1, eos_token_id=None)
    want = model.generate(ids, **common)
    hf.enable(model)
    got = model.generate(ids, past_key_values=hf.FFACache(max_new_tokens=24 - 9 + 8, engine=PlainEngine), prefill_chunk_size=9, **common)
    hf.disable(model)
    assert torch.equal(got, want)


@pytest.mark.parametrize("family", ["opt", "gptj"])
def test_crop_into_the_padding(family):
    """After a crop the short sample has no real token left (its first were at 4 and 5); the next come behind more padding."""
    model = MAKE[family]()
    ids, mask = padded_ids(12)
    want, _ = chunked_logits(model, ids, mask, [40], None)
    hf.enable(model)
    for at, pieces in ((4, [36]), (4, [1] * 36), (3, [1, 36])):
        other = mask.clone()
        other[1, 4:] = 1                                     # at first its tokens began at 4
        _, cache = chunked_logits(model, ids[:, :14], other[:, :14], [8, 6], hf.FFACache(max_new_tokens=36, engine=PlainEngine))
        cache.crop(at)
        logits, done = [], at
        for n in pieces:
            pos = (mask[:, :done + n].long().cumsum(-1) - 1).clamp(min=0)[:, -n:]
            kw = {"position_ids": pos} if family == "gptj" else {}
            with torch.no_grad():
                out = model(input_ids=ids[:, done:done + n], attention_mask=mask[:, :done + n], past_key_values=cache, use_cache=True, **kw)
            logits.append(out.logits.float())
            done += n
        assert float((torch.cat(logits, 1) - want[:, at:])[mask[:, at:].bool()].abs().max()) < 2e-4
    hf.disable(model)


def test_second_turn_padded_behind_the_first_is_refused():
    """Padding between a sample's keys cannot be left out by the engine; the cache goes on without that turn."""
    for make in (tiny_opt, tiny_gptj):
        model = make()
        ids, mask = long_ids()
        want, _ = chunked_logits(model, ids[:, :20], mask[:, :20], [20], None)
        hf.enable(model)
        _, cache = chunked_logits(model, ids[:, :12], mask[:, :12], [9, 3], hf.FFACache(max_new_tokens=31, engine=PlainEngine))
        for hole in (slice(12, 15), slice(17, 20), slice(13, 14)):
            m = mask[:, :20].clone()
            m[0, hole] = 0
            with pytest.raises(NotImplementedError, match="left padding"), torch.no_grad():
                model(input_ids=ids[:, 12:20], attention_mask=m, past_key_values=cache, use_cache=True)
        pos = (mask[:, :20].long().cumsum(-1) - 1).clamp(min=0)[:, 12:]
        with torch.no_grad():
            out = model(input_ids=ids[:, 12:20], attention_mask=mask[:, :20], past_key_values=cache, use_cache=True,
                        **({"position_ids": pos} if make is tiny_gptj else {}))
        assert float((out.logits.float() - want[:, 12:])[mask[:, 12:20].bool()].abs().max()) < 2e-4
        hf.disable(model)


def layer_after_prompt(t=6, B=2, H=2, Dh=64):
    g = torch.Generator().manual_seed(4)
    layer = hf.FFALayer(16, engine=PlainEngine)
    k, v = (torch.randn(B, H, t, Dh, generator=g) for _ in range(2))
    k, v = layer.update(k, v)
    causal = torch.ones(t, t).tril().bool()[None, None].expand(B, 1, t, t)
    hf.ffa_attention_forward(None, k.clone(), k, v, causal)
    return g, layer


def group(g, layer, n, mask, B=2, H=2, Dh=64):
    q, k, v = (torch.randn(B, H, n, Dh, generator=g) for _ in range(3))
    k, v = layer.update(k, v)
    return hf.ffa_attention_forward(None, q, k, v, mask)[0]


def causal_mask(t, n, B=2, dtype=torch.bool):
    seen = (torch.arange(t + n)[None] <= t + torch.arange(n)[:, None])[None, None].expand(B, 1, n, t + n).clone()
    if dtype == torch.bool:
        return seen
    return torch.zeros(seen.shape, dtype=dtype).masked_fill(~seen, torch.finfo(dtype).min)


def test_masks_that_are_no_chain_are_refused():
    for name in ("tree", "window", "bias", "noncausal", "heads", "short", "2-d", "bool tree"):
        g, layer = layer_after_prompt()
        before = [x.clone() for x in layer.engine.get_cache()]
        m = causal_mask(6, 4, dtype=torch.float32)
        low = torch.finfo(torch.float32).min
        if name == "tree":
            m[:, :, 2, 7] = low                              # nodes 1 and 2 are siblings
        elif name == "bool tree":
            m = m == 0
            m[1, :, 3, 8] = False
        elif name == "window":
            m[:, :, 3, :2] = low
        elif name == "bias":
            m[0, 0, 1, 3] = -0.5
        elif name == "noncausal":
            m[:, :, 0, 7] = 0
        elif name == "heads":
            m = m.expand(2, 2, 4, 10)
        elif name == "short":
            m = m[..., :-1]
        else:
            m = m[0, 0]
        with pytest.raises(NotImplementedError, match="left padding"):
            group(g, layer, 4, m)
        assert layer.t == layer.seen == 6 and all(torch.equal(a, b) for a, b in zip(layer.engine.get_cache(), before)), name
        group(g, layer, 4, causal_mask(6, 4))                # and the layer goes on
        assert layer.t == 10


@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.float16, torch.bfloat16])
def test_masks_of_any_type(dtype):
    got = []
    for m in (None, causal_mask(6, 4, dtype=dtype), causal_mask(6, 4, B=1, dtype=dtype)):
        g, layer = layer_after_prompt()
        got.append(group(g, layer, 4, m))
        assert layer.first_key.tolist() == [0, 0]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_bounded_cache_wants_a_real_token_of_every_sample():
    model = tiny_opt()
    ids, mask = padded_batch()
    mask = mask.clone()
    mask[1] = 0
    hf.enable(model)
    with pytest.raises(NotImplementedError, match="real token"), torch.no_grad():
        model(input_ids=ids, attention_mask=mask, past_key_values=hf.FFACache(max_new_tokens=4, engine=PlainEngine, keep=4), use_cache=True)
    hf.disable(model)


def test_refused_prompt_leaves_the_bounded_cache_empty():
    model = tiny_opt()
    ids, mask = padded_batch()
    gone = mask.clone()
    gone[1] = 0
    hf.enable(model)
    cache = hf.FFACache(max_new_tokens=4, engine=PlainEngine, keep=9)
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="real token"):
            model(input_ids=ids, attention_mask=gone, past_key_values=cache, use_cache=True)
        assert cache.get_seq_length() == 0
        got = model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True).logits
        hf.disable(model)
        want = model(input_ids=ids, attention_mask=mask).logits
    assert float((got - want)[mask.bool()].abs().max()) < 2e-4


def test_engine_without_group_attention_still_takes_single_tokens():
    """A sample that is all padding so far, on an engine without attention_tree: its keys begin behind the prompt."""
    model = tiny_opt()
    ids, mask = padded_ids(9, length=14)
    check_chunks(model, ids, mask, [9] + [1] * 5, dict(engine=OracleEngine), 2e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["opt", "gptj"])
def test_padding_longer_than_the_first_chunk_with_hip_engine(family):
    print("padded chunks", family, flush=True)
    model = MAKE[family]().to("cuda:0")
    for pad, pieces in ((9, [9, 31]), (14, [9, 1, 2, 20, 8])):
        ids, mask = padded_ids(pad, "cuda:0")
        check_chunks(model, ids, mask, pieces, {}, 2e-4)
    if family == "gptj":
        ids, mask = padded_ids(100, "cuda:0", 150)
        check_chunks(small_gptj().to("cuda:0"), ids, mask, [10, 64, 76], {}, 2e-4)
