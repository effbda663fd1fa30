"""A KV cache held in 4 bits: writing, reading and single-token attention over
it (``tf_kv4_write``, ``tf_rope_kv4_write``, ``tf_kv4_read``,
``tf_kv4_decode_attention``, ``tf_kv4_decode_attention_rope``).

Format: each cached row (one token's key or value of one kv head) keeps its D
channels as codes 0..15, two per byte (byte j: channel 2j low, 2j + 1 high),
and per group of 64 or 128 channels a (scale, zero point) pair in the model's
dtype; a channel's value is (code - zero) * scale. It is the weight format of
``quant`` with the group's range widened to hold zero, so that a group of one
sign keeps its values. No counterpart in the reference, whose cache is
transformers' DynamicCache in the model dtype.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from .prompt_attention import _offsets, _rows


class KV4Cache(NamedTuple):
    """The tensors of a cache for B sequences of up to t_max positions (a
    multiple of 16): codes uint8 [B, Hkv, t_max, D/2] and parameters
    [B, Hkv, t_max, D/group, 2] (scale, zero point), all contiguous."""

    k: torch.Tensor
    k_params: torch.Tensor
    v: torch.Tensor
    v_params: torch.Tensor

    @classmethod
    def empty(cls, batch: int, kv_heads: int, max_len: int, head_dim: int, group_size: int = 64,
              dtype: torch.dtype = torch.bfloat16, device=None) -> "KV4Cache":
        """A cache for at least `max_len` positions (rounded up to 16), zeroed."""
        if head_dim not in (64, 128) or group_size not in (64, 128) or group_size > head_dim:
            raise ValueError(f"head_dim {head_dim} with groups of {group_size}: both 64 or 128, the group no larger")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"cache dtype must be fp16/bf16, got {dtype}")
        device = device or torch.device("cuda", torch.cuda.current_device())
        t_max = -(-max_len // 16) * 16
        codes = [torch.zeros(batch, kv_heads, t_max, head_dim // 2, dtype=torch.uint8, device=device) for _ in "kv"]
        params = [torch.zeros(batch, kv_heads, t_max, head_dim // group_size, 2, dtype=dtype, device=device)
                  for _ in "kv"]
        return cls(codes[0], params[0], codes[1], params[1])

    def layout(self) -> tuple[int, int, int, int, int, int]:
        """(B, Hkv, D, group, t_max, dtype code) after checking that the four tensors fit together."""
        k, kp, v, vp = self
        shape, params = k.shape, kp.shape
        if len(shape) != 4 or len(params) != 5:
            raise ValueError(f"not a 4-bit cache: codes {tuple(shape)}, parameters {tuple(params)}")
        b, h, t, half = shape
        groups = params[3]
        if params != (b, h, t, groups, 2):
            raise ValueError(f"not a 4-bit cache: codes {tuple(shape)}, parameters {tuple(params)}")
        if v.shape != shape or vp.shape != params:
            raise ValueError("the key and value sides of the cache differ in shape")
        dtype = kp.dtype
        if k.dtype is not torch.uint8 or v.dtype is not torch.uint8 or vp.dtype is not dtype:
            raise ValueError("cache codes must be uint8, its parameters of one dtype")
        if not (k.is_contiguous() and kp.is_contiguous() and v.is_contiguous() and vp.is_contiguous()):
            raise ValueError("cache tensors must be contiguous")
        if groups < 1 or 2 * half % groups:
            raise ValueError(f"{groups} groups do not divide {2 * half} channels")
        return b, h, 2 * half, 2 * half // groups, t, _lib.dtype_code(dtype)

    def pointers(self) -> tuple[int, int, int, int]:
        k, kp, v, vp = self
        return k.data_ptr(), kp.data_ptr(), v.data_ptr(), vp.data_ptr()


def _index(t: torch.Tensor | None, n: int, name: str) -> int | None:
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _side(t: torch.Tensor, h: int, d: int, dtype: torch.dtype, name: str) -> int:
    """Tokens of `t`, which must be [tokens, h, d]."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != h or shape[2] != d or t.dtype is not dtype:
        raise ValueError(f"{name} must be [tokens, {h}, {d}] of {dtype}, got {tuple(shape)} {t.dtype}")
    return shape[0]


def _rope_rows(qkv: torch.Tensor, q_heads: int, cos: torch.Tensor, sin: torch.Tensor, cache: KV4Cache, h: int, d: int,
               t_max: int) -> int:
    """The row stride of projection rows that fit the cache and the tables."""
    width = (q_heads + 2 * h) * d
    if qkv.ndim != 2 or qkv.shape[1] != width or qkv.stride(1) != 1 or qkv.dtype != cache.k_params.dtype:
        raise ValueError(f"qkv must be rows of {width} {cache.k_params.dtype}, got {tuple(qkv.shape)} {qkv.dtype}")
    if qkv.stride(0) < width and qkv.shape[0] > 1:
        raise ValueError("qkv rows overlap")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.ndim != 2 or t.shape[0] < t_max or t.shape[1] != d or t.dtype != qkv.dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [>= {t_max}, {d}] of {qkv.dtype}, got {tuple(t.shape)}")
    return qkv.stride(0) if qkv.shape[0] > 1 else width


def kv4_write(k: torch.Tensor, v: torch.Tensor, cache: KV4Cache, cu_seqlens: torch.Tensor,
              start: torch.Tensor | None = None, slots: torch.Tensor | None = None) -> None:
    """Quantise packed keys and values [T, Hkv, D] into the cache: token i of
    sequence s (cu_seqlens int32 [S + 1] on the device) goes to position
    start[s] + i (start defaults to 0) of cache row slots[s] (defaults to s).
    Tokens whose position or row lies outside the cache are left out, as are
    rows that belong to no sequence (from cu_seqlens[S] on: padding)."""
    b, h, d, g, t_max, dt = cache.layout()
    S = _offsets(cu_seqlens)
    dtype = cache.k_params.dtype
    total = _side(k, h, d, dtype, "k")
    if _side(v, h, d, dtype, "v") != total:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    dev = _lib.require_cuda(k, v, *cache, cu_seqlens, start, slots)
    (k, k_at, k_t, k_h), (v, v_at, v_t, v_h) = _rows(k), _rows(v)
    rc = _lib.load().tf_kv4_write(
        k_at, k_t, k_h, v_at, v_t, v_h, *cache.pointers(), cu_seqlens.data_ptr(), _index(start, S, "start"),
        _index(slots, S, "slots"), S, total, b, h, d, g, t_max, dt, _lib.stream_ptr(dev))
    _lib.check(rc, "kv4_write")


def rope_kv4_write(qkv: torch.Tensor, q_heads: int, cos: torch.Tensor, sin: torch.Tensor, cache: KV4Cache,
                   cu_seqlens: torch.Tensor, start: torch.Tensor | None = None,
                   slots: torch.Tensor | None = None) -> None:
    """Rotate the q and k heads of packed projection rows qkv [T, (Hq + 2 Hkv) D]
    in place (rotary tables cos/sin [>= t_max of the positions, D], transformers'
    roundings) and quantise the rotated keys and the values into the cache, as
    kv4_write places them. What kv4_write leaves out is neither rotated nor written."""
    b, h, d, g, t_max, dt = cache.layout()
    S = _offsets(cu_seqlens)
    ld = _rope_rows(qkv, q_heads, cos, sin, cache, h, d, t_max)
    dev = _lib.require_cuda(qkv, cos, sin, *cache, cu_seqlens, start, slots)
    rc = _lib.load().tf_rope_kv4_write(
        qkv.data_ptr(), ld, cos.data_ptr(), sin.data_ptr(), *cache.pointers(),
        cu_seqlens.data_ptr(), _index(start, S, "start"), _index(slots, S, "slots"), S, qkv.shape[0], b, q_heads, h, d,
        g, t_max, dt, _lib.stream_ptr(dev))
    _lib.check(rc, "rope_kv4_write")


def kv4_read(cache: KV4Cache, cu_seqlens: torch.Tensor, total: int, start: torch.Tensor | None = None,
             slots: torch.Tensor | None = None, *,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [total, Hkv, D] in the cache's dtype: the values held at the
    positions where kv4_write with the same cu_seqlens, start and slots would
    place packed tokens; zeros for what it would leave out."""
    b, h, d, g, t_max, dt = cache.layout()
    S = _offsets(cu_seqlens)
    dev = _lib.require_cuda(*cache, cu_seqlens, start, slots)
    dtype = cache.k_params.dtype
    if out is None:
        k = torch.empty_strided((total, h, d), (h * d, d, 1), dtype=dtype, device=dev)
        v = torch.empty_strided((total, h, d), (h * d, d, 1), dtype=dtype, device=dev)
        k_t = v_t = h * d
        k_h = v_h = d
    else:
        k, v = out
        for name, t in (("k", k), ("v", v)):
            if _side(t, h, d, dtype, name) != total or t.stride(2) != 1 or t.device != dev:
                raise ValueError(f"out {name} must be [{total}, {h}, {d}] on {dev} with contiguous channels")
        (k_t, k_h, _), (v_t, v_h, _) = k.stride(), v.stride()
    rc = _lib.load().tf_kv4_read(
        *cache.pointers(), k.data_ptr(), k_t, k_h, v.data_ptr(), v_t, v_h, cu_seqlens.data_ptr(),
        _index(start, S, "start"), _index(slots, S, "slots"), S, total, b, h, d, g, t_max, dt, _lib.stream_ptr(dev))
    _lib.check(rc, "kv4_read")
    return k, v


def kv4_decode_attention(q: torch.Tensor, cache: KV4Cache, lens: torch.Tensor, *, scale: float | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one query token per sequence over the cache: q [B, Hq, D],
    lens int32 [B] on the device (positions attended, clamped to the cache;
    none gives zeros) -> [B, Hq, D]. `scale` is positive and defaults to D**-0.5."""
    b, h, d, g, t_max, dt = cache.layout()
    shape, dtype = q.shape, cache.k_params.dtype
    if len(shape) != 3 or shape[0] != b or shape[2] != d or q.dtype is not dtype:
        raise ValueError(f"q must be [{b}, heads, {d}] of {dtype}, got {tuple(shape)} {q.dtype}")
    hq = shape[1]
    if hq < 1 or hq % h:
        raise ValueError(f"{hq} query heads are not a multiple of {h} kv heads")
    if scale is not None and not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive, got {scale}")
    dev = _lib.require_cuda(q, *cache, lens)
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty_strided(shape, (hq * d, d, 1), dtype=dtype, device=dev)
    elif out.shape != shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be contiguous, of q's shape and dtype")
    lib = _lib.load()
    ws = _lib.kv4_workspaces.get(dev, lib.tf_kv4_attention_workspace_bytes())
    rc = lib.tf_kv4_decode_attention(
        q.data_ptr(), *cache.pointers(), out.data_ptr(), _index(lens, b, "lens"), b, hq, h, d, g, t_max,
        d ** -0.5 if scale is None else scale, dt, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "kv4_decode_attention")
    return out


def kv4_decode_attention_rope(qkv: torch.Tensor, q_heads: int, cos: torch.Tensor, sin: torch.Tensor, cache: KV4Cache,
                              pos: torch.Tensor, *, scale: float | None = None,
                              out: torch.Tensor | None = None) -> torch.Tensor:
    """A decode step's attention in one launch: projection rows qkv
    [B, (Hq + 2 Hkv) D] of one new token per sequence at position pos[b] (int32
    [B] on the device); q and the new key are rotated (tables cos/sin
    [>= t_max, D]), key and value quantised into the cache, and the token attends
    over pos[b] + 1 positions -> [B, Hq, D]. The same results, bit for bit, as
    rope_kv4_write followed by kv4_decode_attention; qkv is only read. A sequence
    whose position lies outside the cache writes nothing and gets zeros."""
    b, h, d, g, t_max, dt = cache.layout()
    ld = _rope_rows(qkv, q_heads, cos, sin, cache, h, d, t_max)
    if qkv.shape[0] != b:
        raise ValueError(f"{qkv.shape[0]} rows for a cache of {b} sequences")
    if q_heads < 1 or q_heads % h:
        raise ValueError(f"{q_heads} query heads are not a multiple of {h} kv heads")
    if scale is not None and not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive, got {scale}")
    dev = _lib.require_cuda(qkv, cos, sin, *cache, pos)
    if out is None:
        out = torch.empty_strided((b, q_heads, d), (q_heads * d, d, 1), dtype=qkv.dtype, device=dev)
    elif out.numel() != b * q_heads * d or out.dtype != qkv.dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be contiguous, [B, Hq, D] or [B, Hq * D] of qkv's dtype")
    lib = _lib.load()
    ws = _lib.kv4_workspaces.get(dev, lib.tf_kv4_attention_workspace_bytes())
    rc = lib.tf_kv4_decode_attention_rope(
        qkv.data_ptr(), ld, cos.data_ptr(), sin.data_ptr(), *cache.pointers(),
        _index(pos, b, "pos"), out.data_ptr(), b, q_heads, h, d, g, t_max, d ** -0.5 if scale is None else scale, dt,
        ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "kv4_decode_attention_rope")
    return out
