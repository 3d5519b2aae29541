# Copyright 2026. Licensed under the Apache License, Version 2.0.
"""Transformer training operators: attention over packed sequences, layer
norm over a dropped-out residual join, and dropout whose mask is never stored.

``packed_attention``  softmax(scale q k^T) v inside each sequence of a batch
                      without padding; causal, grouped heads, dropout
``layer_norm``        LayerNorm(residual + dropout(x)) with its gradients
``counter_dropout``   x * keep / (1 - p)

Masks come from Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, SC
2011), key = ``seed``, 16 bits to an element: element i of a tensor takes
value i % 8 of the call with counter (i // 8 % 2**32, i // 8 // 2**32, 0,
offset); the probability of (head h, packed row t, key j of the row's sequence)
takes value (j // 8 % 2) * 4 + j % 4 of the call with counter
(j // 16 * 2 + j // 4 % 2, t, h, offset). An element is kept if its value is
at least t = min(65535, floor(65536 p + 0.5)) and then scaled by
65536 / (65536 - t); a dropped element counts as 0 whatever it holds. So p is
held to 16 bits (below 2**-17 nothing is dropped), a mask repeats for the same
seed and offset, and the backward pass computes it again.

GPU tensors (f32, f16, bf16) run gfx950 kernels and raise if the native
extension is missing; CPU tensors (f64 too) run the torch code below. The
results are differentiable once: ``create_graph=True`` and forward mode raise
on the GPU, as do tensors without memory (fakes, freed storages). Results do
not depend on the order of atomics: there are none.

``seed`` is an int, or one int64 on the device, which a captured graph reads
at every replay; ``None`` draws one from torch's generator, so
``torch.manual_seed`` governs it. ``offset`` (0 <= offset < 2**32) tells apart
the masks of one seed: give every call of a step its own.
"""

import math
import operator
from typing import Optional, Union

import torch

from bluefog_amd.ops import hip_ext

__all__ = ["packed_attention", "layer_norm", "counter_dropout"]

Seed = Union[None, int, torch.Tensor]
_CPU_TYPES = (torch.float32, torch.float64, torch.float16, torch.bfloat16)
_M32 = 0xFFFFFFFF


def packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    causal: bool = False,
    scale: Optional[float] = None,
    dropout_p: float = 0.0,
    seed: Seed = None,
    offset: int = 0,
) -> torch.Tensor:
    """Attention inside each sequence of a packed batch.

    ``q`` is [tokens, heads, dim], ``k`` and ``v`` are [tokens, kv_heads, dim]
    with heads (at most 65535) a multiple of kv_heads and dim at most 128; rows may be strided
    (slices of one projection). Sequence b is rows ``cu_seqlens[b]`` to
    ``cu_seqlens[b + 1]``; ``cu_seqlens`` is int32 on the same device, starts
    with 0 and does not decrease (a GPU kernel cannot raise on its values: it
    only guarantees to stay inside the tensors). Empty sequences are allowed.
    A GPU call has room for fewer than 2**24 / heads tiles, of which a sequence
    takes one to every 128 tokens or part of them (2**23 / kv_heads if gradients
    are needed of half types with dim above 64).
    Rows behind the last sequence give zeros and take no part, whatever they
    hold; their gradients are zero.

    ``scale`` defaults to 1 / sqrt(dim). Scores, softmax and sums are held in
    32 bits; probabilities are rounded to the input's type once, in front of
    the product with v. Returns [tokens, heads, dim], dense.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() == 3 and q.shape[-1] else 1.0
    if q.is_cuda and hip_ext._require_ext("packed_attention"):
        seed, value = _seed(seed, q, dropout_p)
        return hip_ext._C.packed_attention(
            q, k, v, cu_seqlens, scale, causal, dropout_p, seed, value, offset
        )
    _check(q, dropout_p, offset)
    if not (q.dim() == k.dim() == v.dim() == 3):
        raise ValueError("q, k and v have to be [tokens, heads, dim]")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k and v have to be of one type")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("shapes of q, k and v do not match")
    if not 1 <= q.shape[2] <= 128:
        raise ValueError(f"head dimensions of 1 to 128 are supported, got {q.shape[2]}")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1] or q.shape[1] > 65535:
        raise ValueError("the number of query heads has to be a multiple of the key/value heads")
    if cu_seqlens.dtype != torch.int32:
        raise TypeError("cu_seqlens has to be int32")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.device != q.device:
        raise ValueError("cu_seqlens has to be a dense vector on the same device")
    if cu_seqlens.numel() > 1 << 24:
        raise ValueError("too many sequences")
    kept = _held(scale, q.dtype)
    if not (kept > 0 and math.isfinite(kept)):
        raise ValueError(f"scale has to be positive and finite in 32 bits, got {scale}")
    ends = cu_seqlens.tolist()
    if ends[0] != 0 or ends[-1] > q.shape[0] or any(a > b for a, b in zip(ends, ends[1:])):
        raise ValueError("cu_seqlens has to rise from 0 to at most the number of tokens")
    seed, value = _seed(seed, q, dropout_p)
    key = value if seed is None else int(seed)
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    wide = q.dtype if q.dtype == torch.float64 else torch.float32
    parts = []
    for begin, end in zip(ends, ends[1:]):
        n = end - begin
        if n == 0:
            continue
        # [heads, n, dim]
        sq = q[begin:end].to(wide).transpose(0, 1)
        sk, sv = (
            x[begin:end].to(wide).repeat_interleave(group, 1).transpose(0, 1) for x in (k, v)
        )
        score = torch.matmul(sq, sk.transpose(1, 2)) * scale
        if causal:
            i = torch.arange(n, device=q.device)
            score = score.masked_fill(i > i[:, None], -math.inf)
        prob = torch.softmax(score, 2)
        if dropout_p:
            prob = _masked(prob, _attention_bits(heads, begin, n, key, offset, q.device), dropout_p)
        if causal and not _all_finite(sv):
            # a masked probability of 0 times such a value would be no number
            out = [torch.matmul(prob[:, i : i + 1, : i + 1], sv[:, : i + 1]) for i in range(n)]
            out = torch.cat(out, 1)
        else:
            out = torch.matmul(prob, sv)
        parts.append(out.transpose(0, 1).to(q.dtype))
    # zeros behind the last sequence, tied to the inputs for the case that no
    # sequence has a row
    rest = q[ends[-1]:].masked_fill(torch.ones((), dtype=torch.bool, device=q.device), 0.0)
    parts.append(rest + k[:0].sum() + v[:0].sum())
    return torch.cat(parts)


def layer_norm(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    *,
    residual: Optional[torch.Tensor] = None,
    dropout_p: float = 0.0,
    seed: Seed = None,
    offset: int = 0,
) -> torch.Tensor:
    """LayerNorm(residual + dropout(x)) over the last dimension, of any width
    to 2**26.

    ``residual`` has x's shape and is of x's type or f32 (a 32-bit residual
    stream under half-precision layers); the result has the residual's type,
    or x's without one. ``weight`` and ``bias`` are vectors of x's type or
    f32, each optional. The sum, mean, variance and the sums over rows of the
    gradients of weight and bias are held in 32 bits.
    """
    if x.is_cuda and hip_ext._require_ext("layer_norm"):
        seed, value = _seed(seed, x, dropout_p)
        return hip_ext._C.layer_norm(
            x, weight, bias, eps, residual, dropout_p, seed, value, offset
        )
    _check(x, dropout_p, offset)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 1 << 26:
        raise ValueError("layer_norm needs a tensor with a last dimension of 1 to 2^26")
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != x.shape[-1:] or t.device != x.device:
            raise ValueError("weight and bias have to be vectors of the last dimension")
        if t.dtype not in (torch.float32, x.dtype):
            raise TypeError("weight and bias have to be f32 or of the input's type")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias have to be of one type")
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError("residual has to have the input's shape")
        if residual.dtype not in (torch.float32, x.dtype):
            raise TypeError("residual has to be f32 or of the input's type")
    kept = _held(eps, x.dtype)
    if not ((eps == 0 or kept > 0) and math.isfinite(kept)):
        raise ValueError(f"eps has to be finite and not negative, in 32 bits, got {eps}")
    seed, value = _seed(seed, x, dropout_p)
    wide = x.dtype if x.dtype == torch.float64 else torch.float32
    z = x.to(wide)
    if dropout_p:
        z = _masked(z, _flat_bits(x, value if seed is None else int(seed), offset), dropout_p)
    if residual is not None:
        z = z + residual.to(wide)
    z = z - z.mean(-1, keepdim=True)
    y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(wide)
    if bias is not None:
        y = y + bias.to(wide)
    return y.to(x.dtype if residual is None else residual.dtype)


def counter_dropout(x: torch.Tensor, p: float, seed: Seed = None, offset: int = 0) -> torch.Tensor:
    """x with a share p of its elements set to 0 and the others scaled by
    1 / (1 - p). The mask depends on seed, offset and the place of an element
    in row-major order, not on x's strides. A GPU call takes fewer than 2**35
    elements."""
    if x.is_cuda and hip_ext._require_ext("counter_dropout"):
        seed, value = _seed(seed, x, p)
        return hip_ext._C.counter_dropout(x, p, seed, value, offset)
    _check(x, p, offset)
    seed, value = _seed(seed, x, p)
    bits = _flat_bits(x, value if seed is None else int(seed), offset)
    wide = x.dtype if x.dtype == torch.float64 else torch.float32
    return _masked(x.to(wide), bits, p).to(x.dtype)


# ---------------------------------------------------------------------------
# shared
# ---------------------------------------------------------------------------


def _seed(seed: Seed, like: torch.Tensor, p: float):
    """(tensor or None, int): a seed as the kernels take it."""
    if seed is None:
        if not p:
            return None, 0
        return torch.randint(1 << 62, (1,), device=like.device), 0
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != like.device:
            raise ValueError("seed has to be an int or one int64 on the input's device")
        return seed, 0
    try:
        seed = operator.index(seed)
    except TypeError:
        raise ValueError("seed has to be an int or one int64 on the input's device") from None
    if not -(1 << 63) <= seed < 1 << 63:
        raise ValueError(f"seed has to fit 64 bits, got {seed}")
    return None, seed


def _held(value: float, dtype: torch.dtype) -> float:
    """A number as the sums of this type hold it."""
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    return torch.tensor(value, dtype=wide).item()


def _check(x: torch.Tensor, p: float, offset: int) -> None:
    if x.dtype not in _CPU_TYPES:
        raise TypeError(f"f32, f64, f16 or bf16 tensors are supported, got {x.dtype}")
    if not 0 <= p < 1:
        raise ValueError(f"dropout probability has to be in [0, 1), got {p}")
    if not 0 <= offset <= _M32:
        raise ValueError(f"offset has to be in [0, 2^32), got {offset}")


def _all_finite(x: torch.Tensor) -> bool:
    try:
        return bool(torch.isfinite(x).all())
    except RuntimeError:  # inside torch.vmap, where no value can be asked for
        return True


def _philox(c0, c1, c2, c3, key: int) -> torch.Tensor:
    """[..., 8] 16-bit values of Philox4x32-7 for int64 counters."""
    k0, k1 = key & _M32, (key >> 32) & _M32
    for _ in range(7):
        # the products' low 64 bits are exact, their sign does not matter
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (
            ((b >> 32) & _M32) ^ c1 ^ k0,
            b & _M32,
            ((a >> 32) & _M32) ^ c3 ^ k1,
            a & _M32,
        )
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).flatten(-2)


def _flat_bits(x: torch.Tensor, key: int, offset: int) -> torch.Tensor:
    n = x.numel()
    block = torch.arange((n + 7) // 8, device=x.device)
    zero = torch.zeros_like(block)
    bits = _philox(block & _M32, block >> 32, zero, zero + offset, key)
    return bits.flatten()[:n].view(x.shape)


def _attention_bits(heads: int, begin: int, n: int, key: int, offset: int, device) -> torch.Tensor:
    """[heads, n, n] for the sequence that starts in row ``begin``."""
    call = torch.arange(2 * ((n + 15) // 16), device=device)
    row = begin + torch.arange(n, device=device)[:, None]
    head = torch.arange(heads, device=device)[:, None, None]
    bits = _philox(call, row, head, torch.full_like(call, offset), key)
    # [.., 16 keys, quad parity, (key // 8 % 2, key % 4)] -> keys in order
    bits = bits.unflatten(3, (2, 4)).unflatten(2, (-1, 2)).transpose(3, 4)
    return bits.flatten(2)[:, :, :n]


def _masked(x: torch.Tensor, bits: torch.Tensor, p: float) -> torch.Tensor:
    t = min(65535, int(p * 65536 + 0.5))
    return torch.where(bits >= t, x * (65536 / (65536 - t)), 0.0)
