"""The GPU attention block in place of a Llama-family model's attention module.

    from insitu_amd.adapters.torch_llama import graft

    model = AutoModelForCausalLM.from_pretrained(...)
    graft(model, layers=[10], quant=QuantConfig(key_bits=3, value_bits=2))

The names, arguments and behaviour are those of adapters/torch_llama.py of the
reference (KernelAttention, build_from_layer, graft, ungraft,
compare_against_original), with AttentionBlock (the whole block on the GPU:
fp16 projections, scale, RoPE and the cast to the wire, then rotate, append,
attend on the codes and W_o') in place of the numpy AttentionKernel. The
hidden states stay on the device; nothing crosses to numpy on the way.

The contract a decoder layer calls (transformers' LlamaAttention) is kept as
the reference keeps it:

  * `position_ids` give the tokens' positions (`cache_position` is the older
    spelling); without either the block counts from its own cache length.
  * `past_key_values` is advanced with zero K/V of the right shape, so the
    model's own length bookkeeping stays right; it is never read back: the
    compressed cache is the block's own.
  * a sequence that has begun can change sides: graft(..., past_key_values=cache) takes a dense cache's rows
    into the blocks' own, ungraft(..., past_key_values=cache) writes the blocks' rows where the zeros are. A
    cache whose tensors have room behind the sequence (a static one that is not full) is refused. A layer with a sliding window is grafted as one with window="layer"; by default the block attends every row.
  * `attention_mask` and `position_embeddings` are ignored: the block is causal
    by construction and applies RoPE itself. A batch of more than one sequence
    is refused rather than attended across.

Differences from the reference, by construction: the host half runs its fp32
GEMVs on the GPU, so a wire row can differ from the reference's numpy float
order by up to 2 Q8.16 LSB in a few lanes (below the seam everything is
bit-exact for the same wire rows); the dense fp16 baseline (compressed=False),
the reference's hardware model (hw) and norms of queries and keys that are not an
RMS norm of each head are refused with NotImplementedError rather than approximated.
"""

from __future__ import annotations

import dataclasses
import sys

import numpy as np
import torch
import torch.nn as nn

from ..block import AttentionBlock
from ..config import FixedFormat, ModelConfig, QuantConfig
from ..host import Weights


class KernelAttention(nn.Module):
    """torch_llama.py:58-155: a module with the shape of a Llama attention module,
    holding an AttentionBlock."""

    def __init__(self, kernel: AttentionBlock, layer_idx: int = 0, dtype=None, device=None) -> None:
        super().__init__()
        self.kernel = kernel
        self.layer_idx = layer_idx
        self._dtype = dtype
        self._device = device
        self.last_report = None

    def forward(self, hidden_states, *args, **kwargs):
        """(batch, seq, hidden) or (seq, hidden) in, (output of the same shape, None) out."""
        x = hidden_states
        squeeze = x.dim() == 2
        if squeeze:
            x = x.unsqueeze(0)
        if x.shape[0] != 1:
            raise NotImplementedError(
                f"batch of {x.shape[0]}: this adapter holds one sequence's cache and ignores "
                f"attention_mask, so a padded batch would silently attend across sequences. "
                f"Run one sequence at a time.")
        positions = kwargs.get("position_ids")
        if positions is None:
            positions = kwargs.get("cache_position")
        pos = None
        if positions is not None:
            pos = positions.reshape(-1).detach().cpu().numpy().astype(np.int64)
        y, report = self.kernel.forward(x[0].detach(), pos)
        self.last_report = report
        self._advance_hf_cache(kwargs.get("past_key_values"), x)
        out = y.to(device=x.device, dtype=self._dtype or hidden_states.dtype)
        return (out if squeeze else out.unsqueeze(0)), None

    def _advance_hf_cache(self, cache, x) -> None:
        """torch_llama.py:137-159: bookkeeping only, so that
        past_key_values.get_seq_length() stays the truth."""
        if cache is None:
            return
        m = self.kernel.model
        filler = torch.zeros((x.shape[0], m.num_kv_heads, x.shape[1], m.head_dim),
                             dtype=x.dtype, device=x.device)
        try:
            cache.update(filler, filler, self.layer_idx)
        except Exception as e:
            raise RuntimeError(
                f"could not advance past_key_values ({type(cache).__name__}) for layer "
                f"{self.layer_idx}; positions after the first token would be wrong. Pass "
                f"past_key_values=None, or update this shim.") from e

    def take(self, past_key_values) -> int:
        """The rows that a dense cache holds of this layer into the block's own, which is empty: a graft in
        the middle of a sequence goes on where the model was. Returns their number. A cache that keeps
        a window's rows alone is taken over with those, where the block's window needs no others."""
        k, v = _dense(past_key_values, self.layer_idx)
        name = type(past_key_values).__name__
        n = 0 if k is None else int(k.shape[2])
        written = int(past_key_values.get_seq_length(self.layer_idx))
        if not written and not n:
            return 0
        if k is not None and k.shape[0] != 1:
            raise NotImplementedError(f"batch of {k.shape[0]}: this adapter holds one sequence's cache")
        if self.kernel.cache.length:
            raise ValueError(f"the block's cache holds {self.kernel.cache.length} rows already")
        if n > written:
            raise NotImplementedError(f"{name}: room for {n} rows, {written} of them written")
        window = self.kernel.window
        if n < written and (not n or not _sliding(past_key_values, self.layer_idx) or window is None or n < window - 1):
            raise NotImplementedError(f"{name}: {n} of {written} rows in its tensors, and the block's queries see "
                                      f"{'all' if window is None else window}")
        self.kernel.take(k[0].detach().transpose(0, 1), v[0].detach().transpose(0, 1), first=written - n)
        return n

    def give(self, past_key_values) -> int:
        """The block's rows into a dense cache, in the place of the last it holds of this layer (which
        _advance_hf_cache filled with zeros): the model goes on without the graft. Returns their number."""
        n = self.check_give(past_key_values)
        if not n:
            return 0
        k, v = _dense(past_key_values, self.layer_idx)
        types = (torch.float32, torch.float16, torch.bfloat16)
        rows = self.kernel.cache.read_float(self.kernel.cache.length - n, n, seq=0,
                                            dtype=k.dtype if k.dtype in types else torch.float32)
        with torch.no_grad():
            for dense, x in zip((k, v), rows):
                dense[0, :, -n:].copy_(x.transpose(0, 1))
        return n

    def check_give(self, past_key_values) -> int:
        """How many rows give writes; raises where it cannot. They go to the end of the layer's tensors, which
        therefore end with the sequence, and what they do not hold is what a window has left."""
        k, _ = _dense(past_key_values, self.layer_idx)
        length = self.kernel.cache.length
        if not length:
            return 0
        written = int(past_key_values.get_seq_length(self.layer_idx))
        if written != self.kernel.first + length or (k is not None and k.shape[0] != 1):
            raise ValueError(f"past_key_values is not of the block's sequence of {length} rows")
        rows = 0 if k is None else int(k.shape[2])
        if rows > written:
            raise NotImplementedError(f"{type(past_key_values).__name__}: room for {rows} rows, {written} of them written")
        if rows < written and not _sliding(past_key_values, self.layer_idx):
            raise NotImplementedError(f"{type(past_key_values).__name__}: {rows} of {written} rows in its tensors")
        return min(rows, length)

    def reset(self) -> None:
        self.kernel.reset()


def _dense(past_key_values, layer_idx: int):
    """A transformers cache's (keys, values) of a layer, each (batch, n_kv_heads, tokens, d), or Nones where it holds
    none yet."""
    layers = getattr(past_key_values, "layers", None)
    if layers is not None:
        if layer_idx >= len(layers):
            return None, None
        k, v = getattr(layers[layer_idx], "keys", None), getattr(layers[layer_idx], "values", None)
    elif hasattr(past_key_values, "key_cache"):           # the older spelling
        if layer_idx >= len(past_key_values.key_cache):
            return None, None
        k, v = past_key_values.key_cache[layer_idx], past_key_values.value_cache[layer_idx]
    else:
        raise TypeError(f"{type(past_key_values).__name__} is no cache whose layers hold keys and values")
    if not isinstance(k, torch.Tensor) or k.dim() != 4 or not k.numel():
        return None, None
    return k, v


def _sliding(past_key_values, layer_idx: int) -> bool:
    """Whether a transformers cache keeps the last rows of a layer alone, as a window needs them."""
    layers = getattr(past_key_values, "layers", None)
    return layers is not None and bool(getattr(layers[layer_idx], "is_sliding", False))


def _window(attn_module, model_config, layer_idx: int):
    """The layer's sliding window, or None: the module's own `sliding_window`, else the configuration's where its
    layer_types (if there are any) say so of this layer."""
    get = (lambda k: model_config.get(k)) if isinstance(model_config, dict) else (lambda k: getattr(model_config, k, None))
    if hasattr(attn_module, "sliding_window"):
        w = attn_module.sliding_window
    else:
        kinds = get("layer_types")
        w = get("sliding_window")
        if kinds is not None and layer_idx < len(kinds) and kinds[layer_idx] != "sliding_attention":
            w = None
        if get("use_sliding_window") is False:
            w = None
    return None if w is None or int(w) < 1 else int(w)


def _head_norms(attn_module, m: ModelConfig):
    """The module's q_norm and k_norm as (weights or None, weights or None, eps). Each has to be
    x / sqrt(mean(x^2) + eps) * weight over a head's channels, which one row shows: there are norms
    with a mean, a bias, 1 + weight or a whole projection's width."""
    weights, eps = [], []
    for name in ("q_norm", "k_norm"):
        norm = getattr(attn_module, name, None)
        if norm is None:
            weights.append(None)
            continue
        w = getattr(norm, "weight", None)
        e = next((float(getattr(norm, a)) for a in ("variance_epsilon", "eps") if getattr(norm, a, None) is not None),
                 None)
        if w is None or tuple(w.shape) != (m.head_dim,) or e is None or not e > 0:
            raise NotImplementedError(f"QK-norm: {name} ({type(norm).__name__}) is not an RMS norm of each head")
        x = torch.linspace(-1.0, 2.0, m.head_dim, dtype=torch.float32)
        with torch.no_grad():
            got = norm(x.to(device=w.device, dtype=w.dtype)).float().cpu()
        want = x.to(w.dtype).float()
        want = want * torch.rsqrt(want.square().mean() + e) * w.detach().float().cpu()
        if not torch.allclose(got, want, rtol=8 * torch.finfo(w.dtype).eps, atol=8 * torch.finfo(w.dtype).eps):
            raise NotImplementedError(f"QK-norm: {name} ({type(norm).__name__}) is not an RMS norm of each head")
        weights.append(w)
        eps.append(e)
    if len(set(eps)) > 1:
        raise NotImplementedError(f"QK-norm: queries and keys with different eps {eps}")
    return weights[0], weights[1], eps[0] if eps else m.qk_norm_eps


def _interleaved(attn_module, rotary_dim: int) -> bool:
    """Whether the module's file turns channel 2 j with 2 j + 1 (else j with j + rotary_dim / 2), as its own
    apply_rotary_pos_emb shows: a turn by a quarter (cos 0, sin 1, the same for every pair) takes channel 0 to its
    partner. Half pairs where the file has no such function."""
    turn = getattr(sys.modules.get(type(attn_module).__module__), "apply_rotary_pos_emb", None)
    if turn is None:
        return False
    x = torch.zeros(1, 1, 1, rotary_dim)
    x[..., 0] = 1.0
    for width in (rotary_dim, rotary_dim // 2):       # (a channel's angle, or a pair's)
        try:
            y = turn(x, x, torch.zeros(1, 1, width), torch.ones(1, 1, width))[0].reshape(-1)
        except Exception:
            continue
        at = torch.nonzero(y.abs() > 0.5).reshape(-1).tolist()
        if at == [rotary_dim // 2]:
            return False
        if at == [1]:
            return True
    raise NotImplementedError(f"rotary positions of {type(attn_module).__name__}: which channels its "
                              f"apply_rotary_pos_emb pairs up cannot be seen; give rope_interleaved")


def build_from_layer(attn_module, model_config, *, quant: QuantConfig | None = None,
                     fmt: FixedFormat | None = None, hw=None, capacity: int = 4096,
                     compressed: bool = True, layer_idx: int = 0, softmax: str = "two_pass",
                     rope_interleaved: bool | None = None, window: int | str | None = None, sinks: int = 0,
                     ctx=None) -> KernelAttention:
    """torch_llama.py:172-203: a KernelAttention from an attention module's weights.

    softmax defaults to the reference AttentionKernel's default, "two_pass";
    "online" is the hardware's order and the single fused launch per decode step.
    rope_interleaved: rotary pairs of channels (2 j, 2 j + 1) instead of (j, j + rotary_dim / 2);
    None takes the module's own (_interleaved). window: rows that a query sees, its own the last,
    and sinks: first rows that stay visible beside them; None is all rows, whatever the layer did, and "layer"
    the layer's own sliding_window.
    """
    if not compressed:
        raise NotImplementedError("compressed=False is the reference's fp16 dense baseline; "
                                  "this build runs the compressed block only")
    if hw is not None:
        raise NotImplementedError("hw configures the reference's systolic-array model; the GPU "
                                  "block has no counterpart")
    m = ModelConfig.from_hf(model_config)
    m = dataclasses.replace(m, rope_interleaved=_interleaved(attn_module, m.rotary_dim) if rope_interleaved is None
                            else bool(rope_interleaved))
    q_norm, k_norm, eps = _head_norms(attn_module, m)
    m = dataclasses.replace(m, qk_norm_eps=eps)
    if window == "layer":
        window = _window(attn_module, model_config, layer_idx)
    block = AttentionBlock(m, quant or QuantConfig(), fmt, capacity=capacity, softmax=softmax, window=window, sinks=sinks,
                           ctx=ctx)

    def w(name):
        return getattr(attn_module, f"{name}_proj").weight

    def b(name):
        return getattr(attn_module, f"{name}_proj").bias

    block.weights = Weights(w("q"), w("k"), w("v"), w("o"), m, block.rotation,
                            q_bias=b("q"), k_bias=b("k"), v_bias=b("v"), o_bias=b("o"),
                            q_norm=q_norm, k_norm=k_norm, ctx=block.ctx)
    return KernelAttention(block, layer_idx=layer_idx)


def graft(model, layers, *, past_key_values=None, **kw) -> dict:
    """torch_llama.py:206-219: replace model.model.layers[i].self_attn for each i;
    returns the replaced modules, so the graft can be undone. past_key_values: a dense cache of a
    sequence that has begun, whose rows the blocks take over."""
    original, blocks = {}, {}
    for i in layers:
        original[i] = model.model.layers[i].self_attn
        blocks[i] = build_from_layer(original[i], model.config, layer_idx=i, **kw)
        if past_key_values is not None:
            blocks[i].take(past_key_values)
    for i, block in blocks.items():                   # (all of them or, where one is refused, none)
        model.model.layers[i].self_attn = block
    return original


def ungraft(model, original: dict, *, past_key_values=None) -> None:
    """past_key_values: the sequence's dense cache, which receives the blocks' rows for the model to go on with."""
    if past_key_values is not None:
        blocks = [model.model.layers[i].self_attn for i in original]
        for block in blocks:                          # (all of them or, where one is refused, none)
            block.check_give(past_key_values)
        for block in blocks:
            block.give(past_key_values)
    for i, module in original.items():
        model.model.layers[i].self_attn = module


def compare_against_original(model, layer_idx: int, hidden_states, **kw):
    """torch_llama.py:226-253: one layer both ways on the same input, and the difference."""
    layer = model.model.layers[layer_idx]
    with torch.no_grad():
        ref = layer.self_attn(hidden_states, **kw)
        ref = ref[0] if isinstance(ref, tuple) else ref
    adapter = build_from_layer(layer.self_attn, model.config, layer_idx=layer_idx)
    with torch.no_grad():
        got = adapter(hidden_states, **kw)[0]
    a = ref.detach().cpu().float().numpy()
    b = got.detach().cpu().float().numpy()
    denom = max(float(np.abs(a).max()), 1e-9)
    return {
        "max_abs": float(np.abs(a - b).max()),
        "relative": float(np.abs(a - b).max() / denom),
        "cosine": float((a.ravel() @ b.ravel()) / (np.linalg.norm(a) * np.linalg.norm(b) + 1e-30)),
        "report": adapter.last_report,
    }
