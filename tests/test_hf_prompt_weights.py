"""Hugging Face hook: what a bounded cache takes from the prompt as its keys' weights, against 64 bits."""
import pytest
import torch

from tests.cache_ops_testlib import pack_k, pack_v
from tests.test_hf_cache_ops import PlainEngine
from tests.test_hf_shim import tiny_gptj, tiny_opt

transformers = pytest.importorskip("transformers")
from fastforwardattention_amd import hf  # noqa: E402


class AnyTypeEngine(PlainEngine):
    """The stand-in with caches of any type."""

    def __init__(self, K, V, max_len, use_default_kernel_launch):
        self.kc, self.vc = pack_k(K, max_len), pack_v(V, max_len)

    def get_cache(self):
        return self.kc, self.vc


def prompt(dtype, L, first, B=2, H=3, Dh=64):
    g = torch.Generator().manual_seed(L)
    q, k, v = (torch.randn(B, H, L, Dh, generator=g).to(dtype) for _ in range(3))
    seen = (torch.arange(L)[None] <= torch.arange(L)[:, None])[None] & (torch.arange(L) >= torch.tensor(first)[:, None])[:, None]
    return q, k, v, seen[:, None]


def sums_in_64_bits(q, k, seen, first, scale):
    z = (q.double() @ k.double().transpose(-1, -2) * scale).masked_fill(~seen, float("-inf"))
    p = torch.softmax(z, -1).nan_to_num(0.0)              # rows of padding see nothing
    return p.sum(2), float((q.double().abs() @ k.double().abs().transpose(-1, -2)).max()) * scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("family", ["opt", "gptj"])
@pytest.mark.parametrize("L", [1, 7, 300])
def test_prompt_weights_are_summed_in_32_bits(dtype, family, L):
    """The scores, probabilities and sums are 32-bit numbers whatever the model's type.  Bound: a score is off by
    Dh + 4 roundings of its products' sizes, a probability by twice that and by the roundings of its row's sum, the
    sum over L rows by L more, each of 2^-24."""
    Dh = 64 if family == "opt" else 128
    first, scale = [0, L // 3], Dh ** -0.5
    q, k, v, seen = prompt(dtype, L, first, Dh=Dh)
    mask = torch.zeros(seen.shape, dtype=dtype).masked_fill(~seen, torch.finfo(dtype).min)
    layer = hf.FFALayer(4, engine=AnyTypeEngine, keep=L + 1)
    tagged, _ = layer.update(k, v)
    if family == "opt":
        hf.ffa_attention_forward(None, q, tagged, v, mask, scaling=scale)
    else:
        model = tiny_gptj().eval()
        hf.enable(model)
        attn = model.transformer.h[0].attn
        assert abs(float(attn.scale_attn) - Dh ** 0.5) < 1e-5
        attn._attn(q, tagged, v, mask)
        hf.disable(model)
    want, size = sums_in_64_bits(q, k, seen, first, scale)
    got = layer.bounded[2][:, :, :L].double()
    u = 2.0 ** -24
    rel = 2 * (size * (Dh + 4) * u) + (2 * L + 8) * u
    assert bool(((got - want).abs() <= rel * want).all()), float(((got - want) / want.clamp(min=1e-30)).abs().max())
    assert not bool(layer.bounded[2][:, :, L:].any())


def test_prompt_weights_over_several_blocks_of_rows(monkeypatch):
    """The rows are taken a block at a time; the blocks add up."""
    q, k, v, seen = prompt(torch.float32, 300, [0, 100])
    got = []
    for rows in (1 << 30, 300, 7, 1):
        monkeypatch.setattr(hf, "_WEIGHT_ROWS", rows)
        got.append(hf._prompt_weights(q, k, seen, 0.125, torch.tensor([0, 100])))
    assert all(float((x - got[0]).abs().max()) <= 300 * 2.0 ** -24 * float(got[0].max()) for x in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bounded_cache_in_16_bits_with_hip_engine(dtype):
    """A bounded cache with room for all gives the logits of the model's own cache, to the model's type."""
    print("bounded", dtype, flush=True)
    from tests.test_hf_shim import padded_batch, teacher_forced_logits
    for make in (tiny_opt, tiny_gptj):
        model = make(dtype).to("cuda:0")
        ids, mask = padded_batch("cuda:0")
        want, _ = teacher_forced_logits(model, ids, mask, 6, None)
        hf.enable(model)
        got, cache = teacher_forced_logits(model, ids, mask, 6, hf.FFACache(max_new_tokens=6, keep=9, evict_every=6))
        hf.disable(model)
        assert float((got - want).abs().max()) < (3e-2 if dtype == torch.float16 else 0.25)
        w = cache.layers[0].bounded[2]
        assert w.dtype == torch.float32 and bool(w.isfinite().all())
        real = (mask.sum(1) + 6).float().cpu()
        total = w.sum(2).cpu()                            # every query of every sample hands out a weight of 1
        assert bool(((total - real[:, None]).abs() <= 64 * 2.0 ** -24 * 32 * real[:, None]).all()), (total, real)
