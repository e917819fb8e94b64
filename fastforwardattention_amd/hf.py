"""Hugging Face decoder hook: routes the one-token decode steps of OPT- and GPT-J-style
attention layers through `FastForwardAttn`.

Stands where the reference patches transformers' model files in place (modeling_opt.py:196-226,
modeling_gptj.py:252-281): the prompt pass runs ordinary attention and builds one
`FastForwardAttn` per layer from the prompt's keys and values; every later call with a single
query token goes to `attention(q, k, v, k_cache, v_cache, scale, t, seq_lens, p)` with
`seq_lens` = index of the first real key of each left-padded sample (modeling_opt.py:222,
modeling_gptj.py:274) and `t` = number of keys cached so far, carried per layer.

Written against the installed transformers (5.x) instead of a patched copy of its files:

* `FFACache` is a `transformers.Cache` whose layers own the engines.  Its `update` hands the
  new token's key/value through (tagged with the layer that owns them) instead of returning
  the concatenated history.
* models that dispatch through transformers' attention-function registry (OPT) select the
  registered function `"ffa"`; GPT-J, which calls its own `_attn`, gets that method wrapped.
* GPT-J's rotary embedding of the new token's q and k, which the reference leaves to torch
  ahead of the call (modeling_gptj.py:231-247), is taken over by the engine on decode steps
  (`attention_ex(..., rotary_dim, ...)`: the FasterTransformer feature of attention.cu:874-882):
  the layer's forward is wrapped and skips the torch-side sin/cos gather, split, rotate and
  concatenate.  `enable(model, fused_rotary=False)` keeps the reference's arrangement.
* beam search (`generate(num_beams=n, past_key_values=FFACache(..., num_beams=n))`): where the
  reference's models copy every layer's caches along the batch axis after each step
  (`_reorder_cache`, modeling_opt.py:1072-1075, modeling_gptj.py:911-918), the cache keeps one
  small table per layer -- for every sample and slot, the beam of the group whose caches hold
  that slot -- permutes its rows when beams are re-parented, and hands it to the engine
  (`attention_ex(..., cache_indir, beam_width)`: the FasterTransformer feature of
  attention.cu:1024-1033 that the reference switches off).  Keys and values never move.

* passes of several tokens after the prompt (a prompt in chunks, assisted and prompt-lookup
  decoding), which the reference's models cannot run, go to `attention_tree` as chains of up to 64
  tokens; `crop` takes rejected tokens back.  Their mask may hold left padding, also of more than the
  first chunk, and causal order; any other is refused.
* a cache of bounded size (`FFACache(..., keep=n, recent=m)`): every step goes to
  `attention_weights`, which sums the attention each key receives, starting from the prompt's own;
  whenever evict_every tokens have come on top of `keep`, `evict` keeps the last `recent` tokens
  and the heaviest of the others, per head.

    from fastforwardattention_amd import hf
    hf.enable(model)
    out = model.generate(ids, attention_mask=mask, max_new_tokens=n,
                         past_key_values=hf.FFACache(max_new_tokens=n))

The reference's environment switches are honoured by `FFACache.from_env()`:
`max_tokens`, `use_ffa_default_kl`, `prob_thresh` (summarize.py:77-96)."""
from __future__ import annotations

import functools
import os
import types

import torch
from transformers.cache_utils import Cache, CacheLayerMixin
from transformers.masking_utils import AttentionMaskInterface, eager_mask
from transformers.modeling_utils import AttentionInterface

ATTN_NAME = "ffa"
_TAG = "_ffa_layer"


def _default_engine():
    from . import FastForwardAttn  # raises ImportError when the HIP extension is not built
    return FastForwardAttn


class FFALayer(CacheLayerMixin):
    """One decoder layer's cache: a `FastForwardAttn` built at the prompt pass (or the bounded caches
    filled from it), the number of keys it holds, and the left-padding offsets of the batch."""

    is_sliding = False
    is_compileable = False

    def __init__(self, max_new_tokens: int, prob_thresh: float = 0.0,
                 use_default_kernel_launch: bool = False, engine=None, num_beams: int = 1,
                 keep: int | None = None, recent: int | None = None, evict_every: int = 64):
        super().__init__()
        if keep is not None:
            recent = keep // 2 if recent is None else recent
            if keep < 1 or not 0 <= recent <= keep or evict_every < 1:
                raise ValueError("eviction wants keep >= 1, 0 <= recent <= keep and evict_every >= 1")
            if num_beams != 1 or prob_thresh != 0.0:
                raise ValueError("eviction goes with neither beam search nor a pruning threshold")
        self.keep, self.recent, self.evict_every = keep, recent, int(evict_every)
        self.bounded = None         # (k_cache, v_cache, key_weights) of keep + evict_every slots
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be >= 1")
        if num_beams < 1:
            raise ValueError("num_beams must be >= 1")
        self.num_beams = int(num_beams)
        self.beam_table = None      # int32 [B, max_len]: beam of the group whose caches hold the slot
        self.max_new_tokens = int(max_new_tokens)
        self.prob_thresh = float(prob_thresh)
        self.use_default_kernel_launch = bool(use_default_kernel_launch)
        self._engine_cls = engine
        self.engine = None
        self.t = 0                  # keys cached = slot of the next token
        self.seen = 0               # tokens so far: more than t once some were evicted
        self.max_len = 0
        self.first_key = None       # int32 [B]: first real key of each left-padded sample
        self.max_first = 0          # its largest entry: t or more while a sample has no real key yet
        self._hooked = False        # the attention hook has seen this layer's prompt pass
        self._pending = False       # a decode token was handed out and not yet attended

    # -- transformers.Cache protocol -----------------------------------------------------
    def lazy_initialization(self, key_states, value_states):
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def update(self, key_states, value_states, *args, **kwargs):
        if self.engine is None:
            return self._prompt_pass(key_states, value_states)
        n = key_states.shape[-2]
        if n > 1:
            self._check_group_pass()
        if not self._hooked:
            raise RuntimeError("FFACache: the model's attention does not go through the 'ffa' hook; "
                               "call fastforwardattention_amd.hf.enable(model) first")
        if self._pending:
            raise RuntimeError("FFACache: the previous decode token of this layer was never attended")
        self._check_room(n)
        self._pending = True
        setattr(key_states, _TAG, self)
        return key_states, value_states

    def _check_room(self, n):
        if self.seen + n > self.max_len:
            raise RuntimeError(f"FFACache: cache full ({self.max_len} slots = first pass + max_new_tokens, which counts the rest of "
                               "a prompt in chunks and guesses too)")

    def _check_group_pass(self):
        if self.beam_table is not None or self.bounded is not None or not hasattr(self.engine, "attention_tree"):
            raise NotImplementedError("FFACache: passes of several tokens after the prompt need an engine with attention_tree "
                                      "and go with neither beam search nor eviction")

    def get_seq_length(self) -> int:
        return self.seen

    def get_mask_sizes(self, query_length: int):
        return self.seen + query_length, 0

    def get_max_length(self) -> int:
        return -1

    def reset(self):
        self.engine, self.t, self.max_len, self.first_key, self.beam_table = None, 0, 0, None, None
        self.max_first = 0
        self.seen, self.bounded = 0, None
        self._hooked = self._pending = False

    def reorder_cache(self, beam_idx):
        """Beam search re-parents the samples: sample b continues sample beam_idx[b] of its own
        group.  Its history becomes the parent's -- a row copy in the table -- and the slot
        the parent wrote last (t - 1) is found in the parent's own caches."""
        if self.engine is None:
            return
        if self.num_beams == 1:
            raise NotImplementedError("FFACache: beam search needs FFACache(..., num_beams=n) with generate's "
                                      "num_beams (the caches are not copied between samples)")
        beam_idx = beam_idx.to(self.beam_table.device)
        B = self.beam_table.shape[0]
        own = torch.arange(B, device=beam_idx.device)
        if beam_idx.numel() != B or bool(((beam_idx // self.num_beams) != (own // self.num_beams)).any()):
            raise ValueError("FFACache: a beam can only continue a beam of its own group")
        table = self.beam_table.index_select(0, beam_idx)
        table[:, self.t - 1] = (beam_idx % self.num_beams).to(torch.int32)
        self.beam_table = table

    def crop(self, max_length: int):
        """Forgets the tokens from `max_length` on (zero or negative: that many of the last, as transformers'
        own caches take it): their slots are written again by the tokens that come instead."""
        if self.engine is None or self.beam_table is not None or self.bounded is not None:
            raise NotImplementedError("FFACache: cropping needs a prompt and goes with neither beam search nor eviction")
        max_length = int(max_length)
        if max_length <= 0:
            max_length = max(0, self.seen + max_length)
        self.t = self.seen = min(self.seen, max_length)
        self._pending = False

    def _unsupported(self, *a, **k):
        raise NotImplementedError("FFACache holds the reference's fixed-layout caches: no batch reshaping")

    batch_repeat_interleave = batch_select_indices = offload = prefetch = _unsupported

    # -- the two passes -------------------------------------------------------------------
    def _prompt_pass(self, key_states, value_states):
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        cls = self._engine_cls or _default_engine()
        prompt_len = key_states.shape[-2]
        self.max_len = prompt_len + self.max_new_tokens
        if self.keep is not None and not (hasattr(cls, "attention_weights") and hasattr(cls, "evict")):
            raise NotImplementedError("FFACache: this engine has no attention_weights and evict, which keep= needs")
        # A bounded cache is filled from the prompt's once the prompt's attention is known.
        slots = prompt_len if self.keep is not None else self.max_len
        self.engine = cls(key_states.contiguous(), value_states.to(key_states.dtype).contiguous(),
                          slots, self.use_default_kernel_launch)
        self.t = self.seen = prompt_len
        if self.num_beams > 1:
            B = key_states.shape[0]
            if B % self.num_beams:
                raise ValueError(f"FFACache: batch {B} is not a multiple of num_beams = {self.num_beams}")
            if not hasattr(self.engine, "attention_ex"):
                raise NotImplementedError("FFACache: this engine has no attention_ex, which beam search needs")
            own = (torch.arange(B, device=key_states.device) % self.num_beams).to(torch.int32)
            self.beam_table = own[:, None].expand(B, self.max_len).contiguous()   # every slot in the sample's own caches
        setattr(key_states, _TAG, self)
        return key_states, value_states

    def note_prompt_mask(self, attention_mask):
        """Left-padding offsets from the prompt pass's mask, as the reference takes them:
        index of the first maximum of the last query row (modeling_opt.py:222).  A sample whose last
        row sees nothing is all padding so far: its first real key lies behind the prompt."""
        self._hooked = True
        self.first_key, self.max_first = None, 0
        if attention_mask is None:
            return
        row = attention_mask[:, :, -1, :]
        none = ~_visible(row).any(dim=-1)
        if row.dtype == torch.bool:
            row = row.to(torch.int8)
        first = torch.where(none, row.shape[-1], torch.max(row, dim=-1).indices)
        self.first_key = first.reshape(-1).to(torch.int32).contiguous()
        self.max_first = int(self.first_key.max())
        if self.keep is not None and self.max_first >= self.t:
            self.reset()
            raise NotImplementedError("FFACache: a bounded cache wants a real token of every sample in the prompt")

    def takes_group(self, n: int) -> bool:
        """Whether a pass of n tokens goes to attend_group: several tokens, or a sample that has no real
        key yet, so that the pass's mask has to say whether its token is one."""
        return n > 1 or (self.t <= self.max_first and self.first_key is not None and self.bounded is None
                         and self.beam_table is None and hasattr(self.engine, "attention_tree"))

    def _note_group_mask(self, mask, n: int):
        """Left-padding offsets from the mask [B,1,n,t+n] of a pass of n tokens; returns the tokens' parents
        (None: a chain).  The engine attends to the keys from a sample's first real one up to the token
        itself, so any other mask is refused; rows of padding may hold anything."""
        if mask is None:
            return None
        B, T = self.engine.get_cache()[1].shape[0], self.t + n
        fits = mask.dim() == 4 and mask.shape[0] in (1, B) and tuple(mask.shape[1:]) == (1, n, T)
        if fits:
            mask = mask[:, 0].expand(B, n, T)
            key = torch.arange(T, device=mask.device)
            last = _visible(mask[:, -1])
            first = torch.where(last.any(dim=-1), torch.max(last.to(torch.int8), dim=-1).indices, T)
            wrong = torch.zeros((), dtype=torch.bool, device=mask.device)
            for i in range(0, n, 256):      # bounds the temporaries
                part, at = mask[:, i:i + 256], key[None, self.t + i:self.t + min(n, i + 256), None]
                seen, since = _visible(part), first[:, None, None]
                differs = seen != ((key >= since) & (key <= at))
                if part.dtype.is_floating_point:
                    differs |= seen & (part != 0)       # a bias
                wrong |= (differs & (at >= since)).any()
            wrong, max_first = torch.stack([wrong.to(first.dtype), first.max()]).tolist()
            fits = not wrong
        if not fits:
            self._pending = False
            raise NotImplementedError("FFACache: a pass of several tokens wants a mask [B,1,n,keys] of left padding and causal "
                                      "order, the same for all heads; trees, windows, biases and padding behind a sample's "
                                      "first token are not supported")
        self.first_key, self.max_first = first.to(torch.int32).contiguous(), int(max_first)
        if self.max_first <= self.t:
            return None
        # A sample that begins within the pass: its first real token sees no padding.
        node = torch.arange(n, device=mask.device)
        return torch.where(node == first[:, None] - self.t, -1, node - 1).to(torch.int32)

    def note_prompt_weights(self, query, key, attention_mask, scaling):
        """What each key of the prompt received from real queries, for a bounded cache.  Moves the prompt
        into the bounded caches."""
        if self.keep is None:
            return
        w = _prompt_weights(query, key, attention_mask, scaling, self.first_key)
        k, v = self.engine.get_cache()
        cap = self.keep + self.evict_every
        self.bounded = (k.new_empty((*k.shape[:3], cap, k.shape[4])), v.new_empty((*v.shape[:2], cap, v.shape[3])),
                        w.new_zeros((*w.shape[:2], cap)))
        self.engine = type(self.engine)     # its caches are not needed any more
        self._evict([(k, v)], [w], [self.bounded])

    def _evict(self, caches, weights, into):
        self.engine.evict(caches, weights, self.t, self.keep, self.recent, first_keys=self.first_key, into=into)
        gone = max(0, self.t - self.keep)
        if self.first_key is not None:      # padding goes first
            self.first_key = (self.first_key - gone).clamp_(min=0)
        self.t -= gone

    def attend_group(self, query, key, value, scale: float, attention_mask=None):
        """A pass of n tokens after the prompt: [B,H,n,Dh] q/k/v -> [B,H,n,Dh]; appends them from slot t on."""
        if not self._pending:
            raise RuntimeError("FFACache: attend_group() without pending tokens")
        dt, n = self.dtype, key.shape[-2]
        parents = self._note_group_mask(attention_mask, n)
        q, k, v = query.to(dt), key.to(dt), value.to(dt)
        k_cache, v_cache = self.engine.get_cache()
        outs = []
        for i in range(0, n, 64):
            part = slice(i, min(n, i + 64))
            outs.append(self.engine.attention_tree(q[:, :, part], k[:, :, part], v[:, :, part], k_cache, v_cache,
                                                   float(scale), self.t + i, None if parents is None else parents[:, part] - i,
                                                   first_keys=self.first_key))
        self.t += n
        self.seen += n
        self._pending = False
        return outs[0] if len(outs) == 1 else torch.cat(outs, dim=2)

    def attend(self, query, key, value, scale: float):
        """One decode step: [B,H,1,Dh] q/k/v -> [B,H,Dh]; appends k, v at slot t."""
        if not self._pending:
            raise RuntimeError("FFACache: attend() without a pending decode token")
        dt = self.dtype
        q, k, v = query.to(dt), key.to(dt), value.to(dt)
        if self.bounded is not None:
            k_cache, v_cache, w = self.bounded
            if self.t == w.shape[2]:
                self._evict([(k_cache, v_cache)], [w], None)
            out = self.engine.attention_weights(q, k, v, k_cache, v_cache, float(scale), self.t, w,
                                                first_keys=self.first_key)
            self.t += 1
            self.seen += 1
            self._pending = False
            return out
        k_cache, v_cache = self.engine.get_cache()
        if self.beam_table is not None:
            out = self.engine.attention_ex(q, k, v, k_cache, v_cache, float(scale), self.t, self.first_key,
                                           self.prob_thresh, 0, None, None, None,
                                           cache_indir=self.beam_table, beam_width=self.num_beams)
        elif self.first_key is None:
            out = self.engine.attention(q, k, v, k_cache, v_cache, float(scale), self.t, self.prob_thresh)
        else:
            out = self.engine.attention(q, k, v, k_cache, v_cache, float(scale), self.t, self.first_key,
                                        self.prob_thresh)
        self.t += 1
        self.seen += 1
        self._pending = False
        return out

    def attend_rotary(self, query, key, value, scale: float, rotary_dim: int):
        """One decode step on un-rotated q, k: [B,H,Dh] each -> [B,H,Dh].  The engine rotates q
        and k at position t - first_key[b] (the sample's real tokens so far, which is what
        transformers passes as position_ids for a left-padded batch) and appends."""
        if not self._hooked:
            raise RuntimeError("FFACache: the prompt pass did not go through the 'ffa' hook")
        self._check_room(1)
        dt = self.dtype
        k_cache, v_cache = self.engine.get_cache()
        beams = {} if self.beam_table is None else dict(cache_indir=self.beam_table, beam_width=self.num_beams)
        out = self.engine.attention_ex(query.to(dt), key.to(dt), value.to(dt), k_cache, v_cache, float(scale), self.t,
                                       self.first_key, self.prob_thresh, int(rotary_dim), None, None, None, **beams)
        self.t += 1
        self.seen += 1
        return out


class FFACache(Cache):
    """`past_key_values` object that keeps every layer's keys and values inside a
    `FastForwardAttn` (cache layouts [B,H,Dh/x,Lmax,x] / [B,H,Lmax,Dh], Lmax = prompt +
    max_new_tokens, which counts every token after the first pass: also the rest of a prompt fed in
    chunks, and guesses that are taken back).  `engine` replaces the `FastForwardAttn` class (same constructor and
    methods); tests use it to run the bookkeeping without a GPU.  num_beams: generate's num_beams
    when beam search is used (samples are grouped num_beams at a time, as generate lays them out).
    keep: bound the cache: keep + evict_every slots a head; when they are full, `keep` stay: the last
    `recent` tokens (default keep // 2) and of the others those that received the most attention, by
    head.  Memory and step time then do not grow with the sequence."""

    def __init__(self, max_new_tokens: int, prob_thresh: float = 0.0,
                 use_default_kernel_launch: bool = False, engine=None, num_beams: int = 1,
                 keep: int | None = None, recent: int | None = None, evict_every: int = 64):
        super().__init__(layer_class_to_replicate=functools.partial(
            FFALayer, max_new_tokens, prob_thresh, use_default_kernel_launch, engine, num_beams, keep, recent, evict_every))

    @classmethod
    def from_env(cls, engine=None):
        """The reference's switches (summarize.py:77-96; modeling_opt.py:196-199)."""
        return cls(int(os.environ["max_tokens"]), float(os.environ.get("prob_thresh", "0")),
                   int(os.environ.get("use_ffa_default_kl", "0")) == 1, engine)


def enabled_by_env() -> bool:
    """`use_ffa=1` in the environment, the reference's master switch (modeling_opt.py:196)."""
    return int(os.environ.get("use_ffa", "0")) == 1


# -- attention hooks --------------------------------------------------------------------------
def _visible(mask):
    """Where an attention mask lets a key through: True, a whole number other than 0, or a float that is no
    large negative number (transformers masks with the type's lowest)."""
    if mask.dtype == torch.bool:
        return mask
    return mask > -1e4 if mask.dtype.is_floating_point else mask != 0


def _masked(w, mask):
    if mask is None:
        return w
    return w + mask if mask.dtype != torch.bool else w.masked_fill(~mask, float("-inf"))


def _plain_attention(query, key, value, attention_mask, scaling):
    """Ordinary masked softmax attention for the prompt pass: [B,H,Lq,Dh]."""
    w = _masked(torch.matmul(query, key.transpose(-1, -2)) * scaling, attention_mask)
    w = torch.softmax(w, dim=-1, dtype=torch.float32).to(value.dtype)
    return torch.matmul(w, value)


_WEIGHT_ROWS = 256      # queries at a time: bounds the scores held at once


def _prompt_weights(query, key, attention_mask, scaling, first_key):
    """The attention each key of the prompt receives, summed over the queries: float32 [B,H,Lk].  Scores and
    probabilities are float32 too, as in the steps that add to these sums."""
    q, kt = query.float(), key.float().transpose(-1, -2)
    total = q.new_zeros((*q.shape[:2], kt.shape[-1]))
    for i in range(0, q.shape[2], _WEIGHT_ROWS):
        part = slice(i, min(i + _WEIGHT_ROWS, q.shape[2]))
        mask = attention_mask if attention_mask is None or attention_mask.shape[-2] == 1 else attention_mask[..., part, :]
        w = torch.softmax(_masked(torch.matmul(q[:, :, part], kt) * scaling, mask), dim=-1)
        if first_key is not None:           # the rows of padding say nothing
            real = torch.arange(part.start, part.stop, device=w.device)[None] >= first_key[:, None]
            w = torch.where(real[:, None, :, None], w, 0.0)
        total += w.sum(2)
    return total


def ffa_attention_forward(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kwargs):
    """Attention function for transformers' registry (`attn_implementation="ffa"`).
    Returns ([B, Lq, H, Dh], None) like the built-in ones."""
    if scaling is None:
        scaling = query.shape[-1] ** -0.5
    layer = getattr(key, _TAG, None)
    if layer is not None and layer._pending:
        if layer.takes_group(query.shape[-2]):
            return layer.attend_group(query, key, value, scaling, attention_mask).transpose(1, 2).contiguous(), None
        return layer.attend(query, key, value, scaling).unsqueeze(1), None
    if layer is not None:
        layer.note_prompt_mask(attention_mask)
    out = _plain_attention(query, key, value, attention_mask, scaling)
    if layer is not None:
        layer.note_prompt_weights(query, key, attention_mask, scaling)
    return out.transpose(1, 2).contiguous(), None


def _gptj_attn(self, query, key, value, attention_mask=None, *rest):
    """Replacement for GPTJAttention._attn (modeling_gptj.py:252-281): ([B,H,Lq,Dh], weights)."""
    layer = getattr(key, _TAG, None)
    if layer is not None and layer._pending:
        if layer.takes_group(query.shape[-2]):
            return layer.attend_group(query, key, value, 1.0 / self.scale_attn, attention_mask), None
        return layer.attend(query, key, value, 1.0 / self.scale_attn).unsqueeze(2), None
    if layer is not None:
        layer.note_prompt_mask(attention_mask)
    out, weights = self._ffa_original_attn(query, key, value, attention_mask, *rest)
    if layer is not None:
        layer.note_prompt_weights(query, key, attention_mask, 1.0 / self.scale_attn)
    return out, weights


def _gptj_forward(self, hidden_states, layer_past=None, attention_mask=None, position_ids=None, use_cache=False,
                  output_attentions=False, **kwargs):
    """Replacement for GPTJAttention.forward on one-token steps with an FFACache: projections,
    then the engine (rotary embedding, append, attention), then the output projection.  Every
    other call goes to the layer's own forward."""
    layer = None
    if isinstance(layer_past, FFACache) and self.layer_idx is not None and len(layer_past.layers) > self.layer_idx:
        layer = layer_past.layers[self.layer_idx]
    # The engine rotates by the slot's distance from the first key: not the token's position after an eviction.
    if (layer is None or layer.engine is None or layer.bounded is not None or layer.takes_group(hidden_states.shape[1])
            or output_attentions or not hasattr(layer.engine, "attention_ex")):
        return self._ffa_original_forward(hidden_states, layer_past, attention_mask, position_ids, use_cache,
                                          output_attentions, **kwargs)
    B, H, Dh = hidden_states.shape[0], self.num_attention_heads, self.head_dim
    q = self.q_proj(hidden_states).view(B, H, Dh)
    k = self.k_proj(hidden_states).view(B, H, Dh)
    v = self.v_proj(hidden_states).view(B, H, Dh)
    out = layer.attend_rotary(q, k, v, 1.0 / float(self.scale_attn), self.rotary_dim if self.rotary_dim is not None else Dh)
    out = self.out_proj(out.reshape(B, 1, H * Dh).to(hidden_states.dtype))
    return self.resid_dropout(out), None


def register():
    """Make `"ffa"` known to transformers' attention and mask registries (idempotent)."""
    AttentionInterface.register(ATTN_NAME, ffa_attention_forward)
    AttentionMaskInterface.register(ATTN_NAME, eager_mask)


def enable(model, fused_rotary=True):
    """Route `model`'s decode steps through FastForwardAttn.  Pass an `FFACache` as
    `past_key_values` afterwards; with any other cache the model behaves as before.
    fused_rotary: GPT-J's rotary embedding of the new token runs inside the engine's call
    instead of in torch (no effect on models without one)."""
    register()
    wrapped = 0
    for mod in model.modules():
        if type(mod).__name__.startswith("GPTJ") and hasattr(mod, "_attn") and hasattr(mod, "scale_attn"):
            if not hasattr(mod, "_ffa_original_attn"):
                mod._ffa_original_attn = mod._attn
                mod._attn = types.MethodType(_gptj_attn, mod)
            if fused_rotary and not hasattr(mod, "_ffa_original_forward") and hasattr(mod, "rotary_dim"):
                mod._ffa_original_forward = mod.forward
                mod.forward = types.MethodType(_gptj_forward, mod)
            wrapped += 1
    if wrapped == 0:
        model._ffa_previous_attn = model.config._attn_implementation
        model.config._attn_implementation = ATTN_NAME
    return model


def disable(model):
    """Undo `enable`."""
    for mod in model.modules():
        if hasattr(mod, "_ffa_original_attn"):
            del mod.__dict__["_attn"]          # the class's own method shows through again
            del mod._ffa_original_attn
        if hasattr(mod, "_ffa_original_forward"):
            del mod.__dict__["forward"]
            del mod._ffa_original_forward
    prev = getattr(model, "_ffa_previous_attn", None)
    if prev is not None:
        model.config._attn_implementation = prev
        del model._ffa_previous_attn
    return model
