"""Attention entry point registered with Hugging Face's attention interface.

Mirrors ``shareprefill_attention_forward`` / ``shareprefill_attention_core``
(attn/shareprefill_attn.py:87-184): same signature, same ``(attn_output[B,N,H,D],
attn_weights)`` return.  Differences that do not change results: K/V are never repeated to
the query head count (the kernels map a query head to its KV head) and q/k/v are consumed
through their strides instead of being copied to ``[B,N,H,D]``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import native


def _token_major(x: torch.Tensor) -> torch.Tensor:
    """``[H,N,D]`` (any strides) -> ``[N,H,D]`` view usable by the kernels, copying only if
    the head dimension is not contiguous or rows are not 16-byte aligned."""
    v = x.transpose(0, 1)
    ok = v.stride(2) == 1 and v.stride(0) % 8 == 0 and v.stride(1) % 8 == 0 and v.data_ptr() % 16 == 0
    return v if ok else v.contiguous()


def sparse_prefill_attention(sharing, q, k, v, layer_idx: int, num_heads: int, config, scale: float):
    """One layer of prefill for batch element views q ``[N,H,D]``, k/v ``[N,Hkv,D]``."""
    block_size = config.block_size
    min_budget = 1 if config.min_budget is None else config.min_budget
    max_budget = 2**31 - 1 if config.max_budget is None else config.max_budget
    pat, use_dense = sharing.get_active_blocks(
        q, k, layer_idx, num_heads, block_size,
        math.ceil(min_budget / block_size), math.ceil(max_budget / block_size),
        config.pattern_threshold, config.similarity_threshold, config.fallback_threshold,
        config.queryaware_threshold, False)
    # layers without a head in a shared cluster cannot elect a pivot: no block-mass pass for them
    state = sharing.state if pat.info.get("can_share", True) else None
    out = native.sparse_attention(q, k, v, pat.bitmap, block_size, scale, pat.flags, pat.slot_of_head, state)
    sharing._mark("attention")
    sharing.update_pivotal_attns(layer_idx, None, use_dense, config.pattern_threshold)
    return out, pat


def shareprefill_attention_core(module, query_states, key_states, value_states, *,
                                gqa_interleave: bool = False):
    bsz, num_heads, q_len, head_dim = query_states.shape
    config = module.config
    softmax_scale = getattr(module, "scaling", 1.0 / math.sqrt(head_dim))
    if gqa_interleave:
        raise NotImplementedError("gqa_interleave=True is not supported by the B200 kernels")

    if q_len != 1:
        if not query_states.is_cuda:
            raise native.SpfError("sparse prefill needs CUDA tensors: there is no CPU fallback")
        assert query_states.dtype == torch.bfloat16
        assert q_len == key_states.shape[2]
        if bsz != 1:
            raise NotImplementedError("the sharing state assumes batch size 1")
        q = _token_major(query_states[0])
        k = _token_major(key_states[0])
        v = _token_major(value_states[0])
        out, pat = sparse_prefill_attention(module.attention_sharing, q, k, v, module.layer_idx,
                                            num_heads, config, softmax_scale)
        attn_weights = None
        if getattr(config, "output_attentions", False):
            attn_weights = dense_avg_attn(module.attention_sharing, pat, num_heads)
        return out[None], attn_weights

    # decode step (one query token): dense attention over the cache with the split-K decode kernel;
    # the reference calls flash_attn_func here (attn/shareprefill_attn.py:146-153), which takes bf16 /
    # fp16 only and applies attention dropout in training mode.  This path has one kernel and no
    # library fallback: dropout (training with attention_dropout > 0) and other dtypes are refused.
    dropout = float(getattr(module, "attention_dropout", 0.0) or 0.0) if module.training else 0.0
    if (query_states.is_cuda and query_states.dtype == torch.bfloat16 and dropout == 0.0
            and head_dim in (64, 128)):
        outs = []
        for b in range(bsz):
            outs.append(native.decode_attention(query_states[b, :, 0, :], _token_major(key_states[b]),
                                                _token_major(value_states[b]), softmax_scale))
        return torch.stack(outs)[:, None], None
    raise native.SpfError(
        "decode step: the B200 kernel needs CUDA bfloat16 tensors, head_dim 64 or 128 and no attention "
        f"dropout (got {query_states.dtype} on {query_states.device}, head_dim {head_dim}, dropout {dropout})")


def sliding_window_attention(module, query_states, key_states, value_states, window: int) -> torch.Tensor:
    """A layer with a sliding window: ``[1,H,N,D]`` -> ``[1,N,H,D]``, every token sees the last ``window`` keys up to its
    own.  The reference refuses such layers (attn/shareprefill_attn.py:160-184); they need no block selection.  A prompt brings
    all its keys, a decode step one query and the keys that its cache kept (all, or at least the last ``window``).
    Batch 1: padding is not visible at this interface.  Refused are more keys than tokens were seen, as far as a patched
    model knows their number: buffers of a fixed size that are not full yet."""
    bsz, _, q_len, head_dim = query_states.shape
    if bsz != 1:
        raise NotImplementedError("sliding-window layers are served with batch size 1")
    if q_len != 1 and q_len != key_states.shape[2]:
        raise native.SpfError(f"sliding window: {q_len} queries with {key_states.shape[2]} keys is neither a prompt nor a decode step")
    dropout = float(getattr(module, "attention_dropout", 0.0) or 0.0) if module.training else 0.0
    if dropout != 0.0:
        raise native.SpfError(f"sliding window: the B200 kernels have no attention dropout (got {dropout})")
    if window < 1:
        raise native.SpfError(f"sliding window must be at least 1 (got {window})")
    tokens = getattr(getattr(module, "attention_sharing", None), "tokens_so_far", None)
    if tokens is not None and key_states.shape[2] > tokens:
        raise NotImplementedError(f"sliding window: {key_states.shape[2]} keys of {tokens} tokens; a cache whose buffer has places that no "
                                  "token has filled (a static cache) is not supported by windowed layers")
    out = native.window_attention(_token_major(query_states[0]), _token_major(key_states[0]), _token_major(value_states[0]),
                                  getattr(module, "scaling", 1.0 / math.sqrt(head_dim)), window)
    return out[None]


def dense_avg_attn(sharing, pat, num_heads: int) -> torch.Tensor:
    """The reference's ``avg_attn [1,H,nb,nb]`` (zeros except for this layer's pivots)."""
    nb = pat.num_blocks
    out = torch.zeros(1, num_heads, nb, nb, dtype=torch.float32, device=pat.bitmap.device)
    st = sharing.state
    if st is not None and st.n_slots:
        piv = torch.nonzero(pat.flags & native.HEAD_PIVOT).flatten().tolist()
        slots = pat.slot_of_head.tolist()
        attn = st.field("pivot_attn")
        for h in piv:
            out[0, h] = attn[slots[h]]
    return out


def shareprefill_attention_forward(module, query_states, key_states, value_states,
                                   attention_mask: Optional[torch.Tensor], *, scaling: float = None,
                                   dropout: float = 0.0, **kwargs) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Hugging Face attention interface: q ``[B,H,N,D]``, k/v ``[B,Hkv,N,D]`` ->
    ``(attn_output [B,N,H,D] contiguous, attn_weights or None)``.  ``attention_mask``,
    ``scaling`` and ``dropout`` are ignored as in the reference (the scale is read from
    ``module.scaling``).  Layers that pass ``sliding_window`` go to ``sliding_window_attention``; they refuse a mask."""
    sliding_window = kwargs.pop("sliding_window", None)
    gqa_interleave = kwargs.pop("gqa_interleave", False)
    if sliding_window is not None:
        if gqa_interleave:
            raise NotImplementedError("gqa_interleave=True is not supported by the B200 kernels")
        for name in ("s_aux", "softcap"):      # what some models with windowed layers change the softmax by
            if kwargs.get(name) is not None:
                raise NotImplementedError(f"{name} is not supported by the B200 kernels")
        causal = kwargs.get("is_causal")
        if attention_mask is not None or not (getattr(module, "is_causal", True) if causal is None else causal):
            raise NotImplementedError("windowed layers are causal and take no attention mask")
        return sliding_window_attention(module, query_states, key_states, value_states, int(sliding_window)), None
    return shareprefill_attention_core(module, query_states, key_states, value_states,
                                       gqa_interleave=gqa_interleave)
