"""Paged 8-bit key / value cache: rotary positions, quantised writes, reads and attention.

One layer's cache holds int8 codes ``[pages, kv_heads, page_size, head_dim]``
and one fp32 scale per (page, kv head), for k and v each (value = code *
scale).  A serving loop keeps one ``KVCache`` per layer, one page table for all
layers, and per step

    q = kv_write(cache, k, v, page_table, kv_lens, cu_q, q=q, cos_sin=table)
    o = attention(q, cache, page_table, kv_lens, cu_q, max_q_len)

where the step's tokens of sequence ``s`` are rows ``cu_q[s] .. cu_q[s + 1]`` of
q, k, v and are that sequence's last tokens: ``kv_lens[s]`` counts them.  The
lengths, offsets and the page table are read on the device, so a captured
CUDA graph follows their contents; a page id outside the cache means "no
page" (not written, not attended to, read as zeros), and so does a length past the
table's columns for the tokens there.

Argument checks raise ``RuntimeError``; kernels run on the current stream of
the tensors' device, whichever device is current.  The reference has no counterpart (its serving stack keeps a
bf16 cache); there is no CPU implementation.
"""
from __future__ import annotations

import ctypes
import math
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from .ops import _check, _launch, _stream_of, workspace

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


class KVCache:
    """One layer's cache: four tensors, checked once, and their C descriptor."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page_size", "head_dim", "device", "_index", "_desc",
                 "_ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        _check(k.is_cuda, "KVCache: needs CUDA tensors (there is no CPU implementation)")
        _check(k.dim() == 4 and v.shape == k.shape, "KVCache: k and v must be [pages, kv_heads, page_size, head_dim]")
        _check(k.dtype == torch.int8 and v.dtype == torch.int8, "KVCache: k and v must be int8")
        P, H, S, D = k.shape
        _check(S in PAGE_SIZES, f"KVCache: page_size must be one of {PAGE_SIZES}; got {S}")
        _check(D in HEAD_DIMS, f"KVCache: head_dim must be one of {HEAD_DIMS}; got {D}")
        for t in (k_scale, v_scale):
            _check(t.dtype == torch.float32 and tuple(t.shape) == (P, H), f"KVCache: scales must be float32 [{P}, {H}]")
        for t in (k, v, k_scale, v_scale):
            _check(t.device == k.device and t.is_contiguous(), "KVCache: tensors must be dense and on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = P, H, S, D
        self.device = k.device
        self._desc = _lib.KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, H, S, D, 0)
        self._ref = ctypes.addressof(self._desc)
        self._index = k.get_device()

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int = 16, head_dim: int = 128, device="cuda") -> "KVCache":
        """A cache of ``pages`` free pages.  Nothing is cleared: a page's first write sets its scale."""
        codes = [torch.empty((pages, kv_heads, page_size, head_dim), dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.empty((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])


# ---------------------------------------------------------------- rotary tables

def rotary_table(rot: int, positions: int, base: float = 1e6, scaling: Optional[Dict] = None,
                 device="cuda") -> torch.Tensor:
    """fp32 [positions, rot]: rot / 2 cosines, then rot / 2 sines of each position's angles.

    Pair i turns by ``position * base ** (-2 i / rot)``.  ``scaling`` stretches the table
    for contexts longer than the model was trained on, ``{"type": ..., "factor": f, ...}``:

    - ``linear``: every angle divided by f;
    - ``ntk``: base * f ** (rot / (rot - 2)), so the slowest pair turns 1 / f as far and the fastest as before;
    - ``yarn`` (``original_positions``, ``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor``): pairs that
      turn more than beta_fast times within the original context as before, those below beta_slow divided
      by f, a linear ramp over the pair index between; cosines and sines times attention_factor
      (default 0.1 ln f + 1);
    - ``llama3`` (``original_positions``, ``low_freq_factor`` 1, ``high_freq_factor`` 4): wavelengths above
      original / low divided by f, below original / high as before, interpolated between.

    Computed in 64 bits on the host."""
    _check(rot > 0 and rot % 16 == 0, "rotary_table: rot must be a positive multiple of 16")
    _check(positions > 0, "rotary_table: positions must be positive")
    _check(base > 0, "rotary_table: base must be positive")
    half = rot // 2
    i = torch.arange(half, dtype=torch.float64)
    freq = float(base) ** (-2.0 * i / rot)
    mult = 1.0
    if scaling:
        kind, f = scaling.get("type"), float(scaling.get("factor", 1.0))
        _check(f >= 1.0, "rotary_table: scaling factor must be at least 1")
        if kind == "linear":
            freq = freq / f
        elif kind == "ntk":
            freq = (float(base) * f ** (rot / (rot - 2))) ** (-2.0 * i / rot)
        elif kind in ("yarn", "llama3"):
            orig = scaling.get("original_positions")
            _check(orig is not None and orig > 0, f"rotary_table: {kind} needs original_positions")
            if kind == "yarn":
                fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

                def pair_of(turns):          # the pair that turns this often within the original context
                    return rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

                lo = max(math.floor(pair_of(fast)), 0)
                hi = min(math.ceil(pair_of(slow)), rot - 1)
                ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)   # 0: as before, 1: divided by f
                freq = freq / f * ramp + freq * (1.0 - ramp)
                mult = float(scaling.get("attention_factor") or 0.1 * math.log(f) + 1.0)
            else:
                low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
                _check(high > low, "rotary_table: llama3 needs high_freq_factor > low_freq_factor")
                wave = 2 * math.pi / freq
                smooth = ((orig / wave - low) / (high - low)).clamp(0.0, 1.0)   # 1: as before, 0: divided by f
                freq = (1.0 - smooth) * freq / f + smooth * freq
        else:
            _check(False, f"rotary_table: unknown scaling type {kind!r}")
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return (torch.cat([ang.cos(), ang.sin()], 1) * mult).float().to(device)


# ---------------------------------------------------------------- the step's arguments

_I32, _BF16 = torch.int32, torch.bfloat16


def _batch(what: str, cache: KVCache, page_table, kv_lens, cu):
    """Checks the batch tensors; (batch, table pointer, row stride, columns).  A decode step makes many
    small calls, so the checks read each attribute once."""
    dev = cache.device
    if not (page_table.dtype is _I32 and kv_lens.dtype is _I32 and cu.dtype is _I32 and page_table.device == dev and
            kv_lens.device == dev and cu.device == dev):
        raise RuntimeError(f"{what}: page_table, kv_lens and cu must be int32 on the cache's device")
    try:
        rows, cols = page_table.shape
        B, = kv_lens.shape
        ok = rows == B and cu.shape == (B + 1,)
    except ValueError:
        ok = False
    if not ok:
        raise RuntimeError(f"{what}: page_table [batch, columns], kv_lens [batch] and cu [batch + 1] do not agree")
    if not (kv_lens.is_contiguous() and cu.is_contiguous()):
        raise RuntimeError(f"{what}: kv_lens and cu must be dense")
    if page_table.is_contiguous():
        return B, page_table.data_ptr(), cols, cols
    ld, step = page_table.stride()
    if step != 1 and cols > 1 or ld < cols and B > 1:
        raise RuntimeError(f"{what}: page_table's rows must be dense")
    return B, page_table.data_ptr(), max(ld, cols), cols


def _heads(what: str, name: str, t: torch.Tensor, cache: KVCache):
    """t as [tokens, heads, head_dim] whose heads are dense within a token and whose rows suit 16-byte
    accesses (copied if they are not); tokens, heads, row stride, pointer."""
    D = cache.head_dim
    if t.dtype is not _BF16 or t.dim() != 3 or t.shape[2] != D or t.device != cache.device:
        raise RuntimeError(f"{what}: {name} must be bfloat16 [tokens, heads, {D}] on the cache's device")
    T, H, _ = t.shape
    s0, s1, s2 = t.stride()
    ptr = t.data_ptr()
    if s2 != 1 or (s1 != D and H > 1) or s0 % 8 or s0 < H * D or ptr % 16:
        t = torch.empty((T, H, D), dtype=_BF16, device=t.device).copy_(t)
        return t, T, H, H * D, t.data_ptr()
    return t, T, H, s0, ptr


def _out_like(what: str, name: str, out: Optional[torch.Tensor], t: torch.Tensor, T: int, H: int, cache: KVCache):
    """The output of t's shape: a new dense tensor, or the caller's after the checks; its row stride and pointer."""
    if out is None:
        out = torch.empty_like(t) if t.is_contiguous() else torch.empty((T, H, cache.head_dim), dtype=_BF16, device=t.device)
        return out, H * cache.head_dim, out.data_ptr()
    if out.shape != t.shape:
        raise RuntimeError(f"{what}: {name} must have q's shape")
    dense, _, _, ld, ptr = _heads(what, name, out, cache)
    if dense is not out:
        raise RuntimeError(f"{what}: {name}'s heads must be dense and its rows 16-byte aligned")
    return out, ld, ptr


def kv_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
             cu_q: torch.Tensor, q: Optional[torch.Tensor] = None, cos_sin: Optional[torch.Tensor] = None,
             interleaved: bool = False, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the step's k, v [tokens, kv_heads, head_dim] into the cache, quantised; returns the
    rotated q [tokens, q_heads, head_dim] (into ``q_out``, which may be q) or None without q.

    With ``cos_sin`` (``rotary_table``) the first ``cos_sin.shape[1]`` elements of every q and k head
    are turned by the token's position in its sequence: first and second half pairwise, or
    neighbours with ``interleaved``.  q, k and v may be strided views of one [q | k | v] tensor."""
    N = _lib.native()
    if N is not None and q_out is None:
        got = N.kv_write(cache._ref, cache._index, page_table, kv_lens, cu_q, k, v, q, cos_sin, interleaved)
        if got is not NotImplemented:
            return got
    B, tp, ld, cols = _batch("kv_write", cache, page_table, kv_lens, cu_q)
    k, T, H, ldk, kp = _heads("kv_write", "k", k, cache)
    v, Tv, Hv, ldv, vp = _heads("kv_write", "v", v, cache)
    if H != cache.kv_heads or Hv != H or Tv != T:
        raise RuntimeError(f"kv_write: k and v must both be [tokens, {cache.kv_heads}, {cache.head_dim}]")
    qp, ldq, hq, op, ldo, out = None, 0, 0, None, 0, None
    if q is not None:
        q, Tq, hq, ldq, qp = _heads("kv_write", "q", q, cache)
        if Tq != T or hq == 0:
            raise RuntimeError("kv_write: q must have k's tokens and at least one head")
        out, ldo, op = _out_like("kv_write", "q_out", q_out, q, T, hq, cache)
    elif q_out is not None:
        raise RuntimeError("kv_write: q_out without q")
    cs, rows, rot = None, 0, 0
    if cos_sin is not None:
        if (cos_sin.dtype is not torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or
                cos_sin.device != cache.device):
            raise RuntimeError("kv_write: cos_sin must be a dense float32 [positions, rot] on the cache's device")
        rows, rot = cos_sin.shape
        if not (0 < rot <= cache.head_dim and rot % 16 == 0 and rows > 0):
            raise RuntimeError("kv_write: rot must be a multiple of 16, at most head_dim")
        cs = cos_sin.data_ptr()
    if T == 0:
        return out
    if B == 0:
        raise RuntimeError("kv_write: tokens of no sequence")
    rc = _launch(cache._index, _lib.lib().w4a8_kv_write, cache._ref, tp, ld, cols, kv_lens.data_ptr(), cu_q.data_ptr(), B,
                 T, kp, ldk, vp, ldv, qp, ldq, hq, op, ldo, cs, rows, rot, 1 if interleaved else 0, _stream_of(k))
    if rc != 0:
        _lib.check(rc, "w4a8_kv_write")
    return out


def kv_read(cache: KVCache, page_table: torch.Tensor, kv_lens: torch.Tensor, cu_out: torch.Tensor,
            tokens: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The last ``cu_out[s + 1] - cu_out[s]`` cached tokens of each sequence (``tokens`` =
    cu_out's last value, known to the caller): k, v bf16 [tokens, kv_heads, head_dim]."""
    N = _lib.native()
    if N is not None:
        got = N.kv_read(cache._ref, cache._index, page_table, kv_lens, cu_out, tokens)
        if got is not NotImplemented:
            return got
    B, tp, ld, cols = _batch("kv_read", cache, page_table, kv_lens, cu_out)
    if tokens < 0:
        raise RuntimeError("kv_read: tokens must not be negative")
    k = torch.empty((tokens, cache.kv_heads, cache.head_dim), dtype=_BF16, device=cache.device)
    v = torch.empty_like(k)
    if tokens == 0:
        return k, v
    _check(B > 0, "kv_read: tokens of no sequence")
    rc = _launch(cache._index, _lib.lib().w4a8_kv_read, cache._ref, tp, ld, cols, kv_lens.data_ptr(), cu_out.data_ptr(),
                 B, tokens, k.data_ptr(), v.data_ptr(), _stream_of(k))
    if rc != 0:
        _lib.check(rc, "w4a8_kv_read")
    return k, v


# workspace bytes per (batch, tokens, q heads, kv heads, head dim, longest query)
_WS_BYTES: Dict[Tuple[int, ...], int] = {}


def attention(q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor,
              max_q_len: int, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the step's query tokens q [tokens, q_heads, head_dim] over the cache
    (``kv_write`` comes first: ``kv_lens`` counts these tokens).  q_heads is a multiple of the
    cache's kv_heads; ``max_q_len`` is the longest cu_q[s + 1] - cu_q[s]; ``scale`` defaults to
    head_dim ** -0.5.  A row that sees no token is zero; a row that ``cu_q`` gives to no sequence is not written.

    Scratch is the device's workspace (``ops.workspace``), shared with the linears: calls on one device run
    in stream order."""
    N = _lib.native()
    if N is not None and out is None:
        # a workspace that is too small for the call is refused, and grown below
        got = N.attention(cache._ref, cache._index, page_table, kv_lens, cu_q, q, max_q_len,
                          cache.head_dim ** -0.5 if scale is None else scale, *workspace(0, cache.device))
        if got is not NotImplemented:
            return got
    B, tp, ld, cols = _batch("attention", cache, page_table, kv_lens, cu_q)
    q, T, hq, ldq, qp = _heads("attention", "q", q, cache)
    H, D = cache.kv_heads, cache.head_dim
    if hq == 0 or hq % H:
        raise RuntimeError(f"attention: q heads must be a multiple of the cache's {H}; got {hq}")
    if B > _lib.ATTENTION_MAX_BATCH:
        raise RuntimeError(f"attention: at most {_lib.ATTENTION_MAX_BATCH} sequences; got {B}")
    if max_q_len <= 0 and T > 0:
        raise RuntimeError("attention: max_q_len must be positive")
    out, ldo, op = _out_like("attention", "out", out, q, T, hq, cache)
    if T == 0:
        return out
    if B == 0:
        raise RuntimeError("attention: tokens of no sequence")
    L = _lib.lib()
    key = (B, T, hq, H, D, max_q_len)
    need = _WS_BYTES.get(key)
    if need is None:
        if len(_WS_BYTES) > 4096:
            _WS_BYTES.clear()
        need = _WS_BYTES[key] = L.w4a8_attention_workspace_size(*key)
    ws, wsb = workspace(need, cache.device)
    rc = _launch(cache._index, L.w4a8_attention, cache._ref, tp, ld, cols, kv_lens.data_ptr(), cu_q.data_ptr(), B, T, qp,
                 ldq, hq, max_q_len, D ** -0.5 if scale is None else scale, op, ldo, ws, wsb, _stream_of(q))
    if rc != 0:
        _lib.check(rc, "w4a8_attention")
    return out
