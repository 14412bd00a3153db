"""Drop-in ``do_sdpa_attn`` (laprune/attention.py:21-73).

Same signature, argument meaning and errors as the reference: post-RoPE
query/key/value ``[B, H, T, D]``, optional down-projections, an optional
mask, native GQA, output ``[B, T, H*D]`` through ``out_proj`` when given.

A single query without a mask or down-projections (decode; the reference's
``num_queries == 1`` branch, :62-65) runs the split-K flash-decode kernel
(``lap_dense_attn_decode``): fp16/bf16, head dim 64/128/256, 1/2/4/8 query
heads per KV head, K/V rows 16-byte aligned.  Several queries without a mask
(prefill, with the causal or tail-causal mask of :66-73) run the prompt
kernel (``lap_prompt_attention``) on rows of the same kind when no gradient is
needed and the caller chose no backend (``sdpa_kernel``).  Every other case (an explicit mask, shapes outside the kernels'
contract) runs ``scaled_dot_product_attention`` exactly as the reference does.

:func:`prompt_attention` is that kernel for packed prompts of different lengths
over their caches.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from ._ops import ops, untraced


def _tail_causal_mask(num_queries: int, num_keys: int, dtype, device) -> torch.Tensor:
    """Additive mask for queries at the last positions of the cache
    (laprune/attention.py:6-18): query i sees keys up to num_keys - nq + i."""
    if num_queries > num_keys:
        raise ValueError(f"num_queries={num_queries} exceeds num_keys={num_keys}")
    allowed = torch.ones(num_queries, num_keys, dtype=torch.bool, device=device).tril(
        diagonal=num_keys - num_queries)
    mask = torch.zeros(1, 1, num_queries, num_keys, dtype=torch.float32, device=device)
    mask.masked_fill_(~allowed, torch.finfo(dtype).min)
    return mask.to(dtype=dtype)


def _decode_kernel_fits(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> bool:
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        return False
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[2] != 1:
        return False
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        return False
    B, Hq, _, D = q.shape
    Hkv = k.shape[1]
    if k.shape[0] != B or k.shape[3] != D or D not in (64, 128, 256) or k.shape[2] < 1:
        return False
    if Hq % Hkv or not 1 <= Hq // Hkv <= 8:
        return False
    if q.stride(3) != 1 or k.stride(3) != 1 or v.stride(3) != 1:
        return False
    for t in (k, v):  # rows are read as 16-byte vectors
        if t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:3]):
            return False
    return True


def _needs_grad(*ts: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def _rows16(t: torch.Tensor) -> bool:
    """Rows of contiguous values that start at multiples of 16 bytes."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and
            all(s % 8 == 0 for s in t.stride()[:-1]))


def _any_backend() -> bool:
    """Whether no caller chose among the library's attention kernels (sdpa_kernel(...) or
    the flags that it sets)."""
    b = torch.backends.cuda
    return b.flash_sdp_enabled() and b.mem_efficient_sdp_enabled() and b.math_sdp_enabled()


def _prompt_kernel_fits(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> bool:
    """Several queries [B, Hq, Tq, D] at the end of [B, Hkv, Tk, D] keys, for the
    prompt kernel."""
    return (q.is_cuda and k.is_cuda and v.is_cuda and q.dim() == 4 and k.dim() == 4 and
            v.shape == k.shape and q.dtype in (torch.float16, torch.bfloat16) and
            k.dtype == q.dtype and v.dtype == q.dtype and q.device == k.device == v.device and
            q.shape[0] == k.shape[0] > 0 and k.shape[1] > 0 and q.shape[3] == k.shape[3] and
            q.shape[3] in (64, 128, 256) and q.shape[1] > 0 and q.shape[1] % k.shape[1] == 0 and
            q.shape[1] // k.shape[1] <= 128 and 0 < q.shape[2] <= k.shape[2] and
            all(type(t) in (torch.Tensor, torch.nn.Parameter) and _rows16(t) for t in (q, k, v)) and
            k.shape[2] < 1 << 30 and
            # a launch takes less than 2^24 workgroups, each 128 // group tokens of a KV head
            q.shape[0] * k.shape[1] * -(-q.shape[2] // (128 * k.shape[1] // q.shape[1])) < 1 << 24 and
            max(k.stride(2), v.stride(2)) <= 1 << 24 and untraced() and _any_backend() and
            not torch.is_autocast_enabled(q.device.type) and not _needs_grad(q, k, v))


def prompt_attention(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, plan,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts over their caches.

    query [n, Hq, D]: the packed tokens' post-RoPE queries; keys, values
    [B, Hkv, T, D]: each sequence's cache, the new tokens' rows included (any strides
    between rows); plan: :func:`laprune_amd.packed.pack_prompts` of the n tokens with
    these head counts.  A token at position p of its sequence sees cache rows
    [0, p].  Returns [n, Hq, D] (``out`` if given; rows of no sequence are left as
    they are).  scale: 1/sqrt(D) by default.  fp16/bf16, D 64/128/256; no gradients.

    Softmax and sums are fp32; a weight enters the product with the values in the
    tensors' dtype, relative to a running maximum that may lag by up to 2^8 (error of the
    outputs 1.2 to 1.3 times that of their own rounding, 1.15 to 1.2 with exact maxima)."""
    q, k, v = query, keys, values
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("prompt_attention: tensors must be on CUDA (ROCm) devices")
    if _needs_grad(q, k, v):
        raise RuntimeError("prompt_attention computes no gradients: call it under no_grad, or "
                           "do_sdpa_attn for tensors that require them")
    if q.dim() != 3 or k.dim() != 4 or v.shape != k.shape:
        raise RuntimeError("prompt_attention: query [n, Hq, D], keys and values [B, Hkv, T, D]")
    if plan.heads is None:
        raise RuntimeError("prompt_attention: the plan was made without head counts")
    if plan.heads != (q.shape[1], k.shape[1], q.shape[2]) or q.shape[2] != k.shape[3]:
        raise RuntimeError(f"prompt_attention: the plan is for (Hq, Hkv, D) = {plan.heads}, got "
                           f"({q.shape[1]}, {k.shape[1]}, {q.shape[2]})")
    if plan.total != q.shape[0] or plan.B != k.shape[0]:
        raise RuntimeError(f"prompt_attention: a plan of {plan.total} tokens of {plan.B} sequences, "
                           f"got {q.shape[0]} of {k.shape[0]}")
    if plan.lens is not None and plan.longest > k.shape[2] and plan.total:
        raise RuntimeError(f"prompt_attention: {plan.longest} keys exceed the {k.shape[2]} rows "
                           "of the caches")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise RuntimeError("prompt_attention: out must be like query")
    if plan.total:
        bt, _, nsplit = plan.shape
        ops().prompt_attention(q, k, v, plan.tiles, bt, nsplit, plan.max_keys,
                               1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale), out)
    return out


def do_sdpa_attn(query, key, value, cos=None, sin=None, out_proj=None, query_down_proj=None,
                 key_down_proj=None, mask=None, already_rope: bool = False):
    """Attention over post-RoPE Q/K with native GQA caches."""
    if not already_rope:
        raise ValueError("LAPrune attention expects post-RoPE query and key tensors")
    q, k, v = query, key, value
    num_heads = int(q.shape[1])
    num_queries = int(q.shape[-2])
    if query_down_proj is not None:
        q = q.transpose(1, 2).flatten(2) @ query_down_proj
        q = q.unflatten(-1, (num_heads, -1)).transpose(1, 2)
    if key_down_proj is not None:
        k = k.transpose(1, 2).flatten(2) @ key_down_proj
        k = k.unflatten(-1, (num_heads, -1)).transpose(1, 2)
    enable_gqa = int(q.shape[1]) != int(k.shape[1])
    if enable_gqa and int(q.shape[1]) % int(k.shape[1]) != 0:
        raise ValueError(f"invalid GQA head counts: Hq={q.shape[1]}, Hkv={k.shape[1]}")

    if (mask is None and num_queries == 1 and query_down_proj is None
            and key_down_proj is None and _decode_kernel_fits(q, k, v)):
        from .aq_kernels import _impl
        output = _impl.dense_attn_decode(q, k, v)
    elif mask is None and num_queries > 1 and _prompt_kernel_fits(q, k, v):
        from .packed import prompt_shape
        B, Hq, Tq, D = q.shape
        heads = Hq, k.shape[1], D
        n = B * -(-Tq // prompt_shape(Tq, 1, k.shape[2], *heads)[0])
        bt, _, nsplit = prompt_shape(B * Tq, B, k.shape[2], *heads, n)
        output = q.new_empty((B, Tq, Hq, D))
        ops().prompt_attention(q.transpose(1, 2), k, v, None, bt, nsplit, k.shape[2],
                               1.0 / math.sqrt(D), output)
        output = output.transpose(1, 2)
    elif mask is not None:
        output = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=False,
                                                enable_gqa=enable_gqa)
    else:
        num_keys = int(k.shape[-2])
        if num_keys == num_queries:
            output = F.scaled_dot_product_attention(q, k, v, attn_mask=None, is_causal=True,
                                                    enable_gqa=enable_gqa)
        elif num_queries == 1:
            output = F.scaled_dot_product_attention(q, k, v, attn_mask=None, is_causal=False,
                                                    enable_gqa=enable_gqa)
        else:
            causal = _tail_causal_mask(num_queries, num_keys, q.dtype, q.device)
            output = F.scaled_dot_product_attention(q, k, v, attn_mask=causal, is_causal=False,
                                                    enable_gqa=enable_gqa)
    output = output.transpose(1, 2).flatten(2)
    return out_proj(output) if out_proj is not None else output
