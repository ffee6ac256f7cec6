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
from typing import Dict, List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _check, _launch, _stream_of, workspace

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_I32, _BF16 = torch.int32, torch.bfloat16


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
                 device="cuda", repeat: int = 1) -> torch.Tensor:
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

    ``repeat`` > 1: the pairs are that many equal runs, each with the angles of ``rot / repeat`` elements,
    for axes (``RotaryAxes``) that each have all the frequencies, as image encoders do.

    Computed in 64 bits on the host."""
    _check(rot > 0 and rot % 16 == 0, "rotary_table: rot must be a positive multiple of 16")
    _check(repeat > 0 and rot % (2 * repeat) == 0, "rotary_table: rot must be a multiple of 2 * repeat")
    _check(positions > 0, "rotary_table: positions must be positive")
    _check(base > 0, "rotary_table: base must be positive")
    rot = rot // repeat
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
    return (torch.cat([ang.cos().repeat(1, repeat), ang.sin().repeat(1, repeat)], 1) * mult).float().to(device)


class RotaryAxes:
    """Which axis of a token's position turns which pair of a head: ``sections`` pairs of each axis (time, height,
    width, ...; up to four), one axis after another, or ``mixed``: 0 1 2 0 1 2 ..., an axis whose pairs are used
    up left out.  Twice their sum is the rotary table's width."""

    __slots__ = ("axes", "pairs", "_map", "_ref")

    def __init__(self, sections: Sequence[int], mixed: bool = False):
        left = [int(n) for n in sections]
        _check(0 < len(left) <= _lib.MAX_AXES and all(n > 0 for n in left),
               f"RotaryAxes: 1 to {_lib.MAX_AXES} sections of at least one pair")
        self.axes, self.pairs = len(left), sum(left)
        _check(2 * self.pairs <= _lib.ROTARY_MAX_DIM and self.pairs % 8 == 0,
               f"RotaryAxes: the sections must add up to a multiple of 8, at most {_lib.ROTARY_MAX_DIM // 2}")
        ids = [a for a, n in enumerate(left) for _ in range(n)]
        if mixed:
            ids = []
            while any(left):
                for a in range(len(left)):
                    if left[a]:
                        left[a] -= 1
                        ids.append(a)
        self._map = (ctypes.c_uint8 * self.pairs)(*ids)
        self._ref = ctypes.addressof(self._map)

    def axis_of_pair(self) -> List[int]:
        return list(self._map)


_ONE_AXIS = (1, None)


def _positions(what: str, positions: torch.Tensor, axes: Optional[RotaryAxes], T: int, rot: int, device):
    """Checked positions of their own: pointer, row stride, number of axes, the pairs' axes."""
    n, m = _ONE_AXIS if axes is None else (axes.axes, axes._map)
    if axes is not None and 2 * axes.pairs != rot:
        raise RuntimeError(f"{what}: the axes have {axes.pairs} pairs, cos_sin has {rot // 2}")
    if positions.dtype is not _I32 or positions.device != device:
        raise RuntimeError(f"{what}: positions must be int32 on the tensors' device")
    if positions.dim() == 1 and n == 1:
        positions = positions.view(1, -1) if positions.is_contiguous() else positions.contiguous().view(1, -1)
    if tuple(positions.shape) != (n, T):
        raise RuntimeError(f"{what}: positions must be [{n}, {T}]; got {list(positions.shape)}")
    if positions.stride(1) != 1 and T > 1 or positions.stride(0) < T and n > 1:
        positions = positions.contiguous()
    return positions, positions.data_ptr(), max(positions.stride(0), T), n, m


def _table_of(what: str, cos_sin: torch.Tensor, most: int, device):
    if (cos_sin.dtype is not torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.device != device):
        raise RuntimeError(f"{what}: cos_sin must be a dense float32 [positions, rot] on the tensors' device")
    rows, rot = cos_sin.shape
    if not (0 < rot <= most and rot % 16 == 0 and rows > 0 and cos_sin.data_ptr() % 16 == 0):
        raise RuntimeError(f"{what}: rot must be a multiple of 16, at most head_dim (and cos_sin 16-byte aligned)")
    return cos_sin.data_ptr(), rows, rot


def _plain_heads(what: str, name: str, t: torch.Tensor, D: int, device):
    """_heads without a cache: tensor, tokens, heads, row stride, pointer."""
    if t.dtype is not _BF16 or t.dim() != 3 or t.shape[2] != D or t.device != device:
        raise RuntimeError(f"{what}: {name} must be bfloat16 [tokens, heads, {D}] on one device")
    T, H, _ = t.shape
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != D and H > 1) or (T > 1 and (s0 % 8 or s0 < H * D)) or t.data_ptr() % 16:
        t = torch.empty((T, H, D), dtype=_BF16, device=device).copy_(t)
        s0 = H * D
    return t, T, H, s0 if T > 1 else H * D, t.data_ptr()


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], cos_sin: torch.Tensor, positions: torch.Tensor,
           axes: Optional[RotaryAxes] = None, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [tokens, q_heads, head_dim] and k (or None) with the first ``cos_sin.shape[1]`` elements of every head turned:
    pair i by row ``positions[a, token]`` of ``cos_sin`` (``rotary_table``), a the pair's axis (``RotaryAxes``; without,
    positions int32 [tokens] or [1, tokens]).  Pairs are those of ``kv_write``, whose arithmetic this is, without a
    cache: for encoders and other attentions.  head_dim is a multiple of 8, at most 256.

    positions int32 [axes, tokens] are read on the device; rows outside the table are its first or last one.
    ``q_out`` and ``k_out`` may be q and k."""
    nat = _lib.native()
    if nat is not None and axes is not None and q_out is None and k_out is None:
        got = nat.rotary(q, k, cos_sin, positions, axes.axes, axes.pairs, axes._ref, interleaved)
        if got is not NotImplemented:
            return got
    what = "rotary"
    if not q.is_cuda or q.dim() != 3:
        raise RuntimeError("rotary: q must be a CUDA tensor [tokens, heads, head_dim] (there is no CPU implementation)")
    dev, D = q.device, q.shape[2]
    _check(0 < D <= _lib.ROTARY_MAX_DIM and D % 8 == 0, f"rotary: head_dim must be a multiple of 8, at most {_lib.ROTARY_MAX_DIM}")
    q, T, H, ld, ptr = _plain_heads(what, "q", q, D, dev)
    args, outs = [], []
    for name, t, out in (("q", q, q_out), ("k", k, k_out)):
        if t is None:
            _check(out is None, "rotary: k_out without k")
            args += [None, 0, 0, None, 0]
            outs.append(None)
            continue
        t, Tt, H, ld, ptr = _plain_heads(what, name, t, D, dev)
        _check(Tt == T and H > 0, "rotary: q and k need the same tokens and at least one head")
        if out is None:
            out, ldo, op = torch.empty((T, H, D), dtype=_BF16, device=dev), H * D, None
            op = out.data_ptr()
        else:
            _check(out.shape == t.shape, f"rotary: {name}_out must have {name}'s shape")
            dense, _, _, ldo, op = _plain_heads(what, name + "_out", out, D, dev)
            _check(dense is out, f"rotary: {name}_out's heads must be dense and its rows 16-byte aligned")
        args += [ptr, ld, H, op, ldo]
        outs.append(out)
        if name == "k":
            k = t                                            # (a copy has to live until the launch)
    cs, rows, rot = _table_of(what, cos_sin, D, dev)
    positions, pp, ldp, n, m = _positions(what, positions, axes, T, rot, dev)
    if T > 0:
        rc = _launch(q.get_device(), _lib.lib().w4a8_rotary, *args, T, D, cs, rows, rot, 1 if interleaved else 0, pp, ldp, n, m,
                     _stream_of(q))
        _lib.check(rc, "w4a8_rotary")
    return outs[0], outs[1]


# ---------------------------------------------------------------- the step's arguments

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
             interleaved: bool = False, q_out: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
             axes: Optional[RotaryAxes] = None) -> Optional[torch.Tensor]:
    """Writes the step's k, v [tokens, kv_heads, head_dim] into the cache, quantised; returns the
    rotated q [tokens, q_heads, head_dim] (into ``q_out``, which may be q) or None without q.

    With ``cos_sin`` (``rotary_table``) the first ``cos_sin.shape[1]`` elements of every q and k head
    are turned by the token's position in its sequence: first and second half pairwise, or
    neighbours with ``interleaved``.  q, k and v may be strided views of one [q | k | v] tensor.

    ``positions`` int32 [axes, tokens] (``axes``: ``RotaryAxes``; without, [tokens]) takes the place of the tokens'
    positions in their sequences for the rotation, as ``rotary`` does; the cache is written where it was."""
    N = _lib.native()
    if N is not None and q_out is None and positions is None and axes is None:
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
    own = ()
    if positions is not None:
        if cos_sin is None:
            raise RuntimeError("kv_write: positions without cos_sin")
        positions, *own = _positions("kv_write", positions, axes, T, rot, cache.device)
    elif axes is not None:
        raise RuntimeError("kv_write: axes without positions")
    if T == 0:
        return out
    if B == 0:
        raise RuntimeError("kv_write: tokens of no sequence")
    if own:
        rc = _launch(cache._index, _lib.lib().w4a8_kv_write_axes, cache._ref, tp, ld, cols, kv_lens.data_ptr(), cu_q.data_ptr(),
                     B, T, kp, ldk, vp, ldv, qp, ldq, hq, op, ldo, cs, rows, rot, 1 if interleaved else 0, *own, _stream_of(k))
        if rc != 0:
            _lib.check(rc, "w4a8_kv_write_axes")
        return out
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


# ---------------------------------------------------------------- pages kept on the device

class PageState:
    """The pages of one cache geometry, kept on the GPU: which are free, which each sequence holds, how long it is.

    ``free`` int32 [pages] is a stack of page ids with ``free_pages`` int32 [1] of them left, its top last; ``table`` int32
    [sequences, columns] and ``lens`` int32 [sequences] say what each sequence holds.  ``pages_plan`` and
    ``pages_shrink`` change them on the device; calls on one state run in stream order.  A call that cannot
    be done changes nothing but the status word, which ``check`` reads."""

    __slots__ = ("free", "free_pages", "table", "lens", "control", "page_size", "pages", "sequences", "columns", "device",
                 "_index", "_desc", "_ref")

    def __init__(self, free: torch.Tensor, free_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, page_size: int):
        _check(free.is_cuda, "PageState: needs CUDA tensors (there is no CPU implementation)")
        _check(page_size in PAGE_SIZES, f"PageState: page_size must be one of {PAGE_SIZES}; got {page_size}")
        _check(free.dim() == 1 and tuple(free_pages.shape) == (1,) and table.dim() == 2 and tuple(lens.shape) == (table.shape[0],),
               "PageState: free [pages], free_pages [1], table [sequences, columns] and lens [sequences] do not agree")
        for t in (free, free_pages, table, lens):
            _check(t.dtype is _I32 and t.device == free.device and t.is_contiguous(),
                   "PageState: tensors must be dense int32 on one device")
        self.pages, (self.sequences, self.columns) = free.shape[0], table.shape
        _check(0 < self.pages and self.pages * page_size < 2 ** 31 and 0 < self.columns and self.columns * page_size < 2 ** 31,
               "PageState: pages * page_size and columns * page_size must be in 1..2^31 - 1")
        _check(0 < self.sequences <= _lib.PLAN_MAX_SEQUENCES, f"PageState: 1 to {_lib.PLAN_MAX_SEQUENCES} sequences")
        self.free, self.free_pages, self.table, self.lens, self.page_size = free, free_pages, table, lens, page_size
        self.device, self._index = free.device, free.get_device()
        self.control = torch.zeros(4, dtype=_I32, device=free.device)
        self._desc = _lib.PageStateDesc(free.data_ptr(), free_pages.data_ptr(), table.data_ptr(), lens.data_ptr(),
                                        self.control.data_ptr(), self.pages, self.columns, self.sequences, page_size)
        self._ref = ctypes.addressof(self._desc)

    @classmethod
    def empty(cls, pages: int, sequences: int, columns: int, page_size: int = 16, device="cuda") -> "PageState":
        """``pages`` free pages, taken from page 0 on, and empty sequences of up to ``columns`` pages."""
        i = dict(dtype=_I32, device=device)
        return cls(torch.arange(pages - 1, -1, -1, **i), torch.full((1,), pages, **i), torch.full((sequences, columns), -1, **i),
                   torch.zeros(sequences, **i), page_size)

    def status(self, reset: bool = True) -> int:
        """Why the first refused call since the last reset was refused (bits; 0: none).  Waits for the current stream."""
        v = int(self.control[0])
        if v and reset:
            self.control[0] = 0
        return v

    def check(self) -> None:
        """Raises if a call was refused since the last time."""
        v = self.status()
        if v:
            raise RuntimeError("pages: " + "; ".join(why for bit, why in _lib.PLAN_REASONS.items() if v & bit))


class StepMaps(NamedTuple):
    """One step's batch on the device, as ``kv_write``, ``attention`` and ``rotary`` take it."""
    page_table: torch.Tensor            # int32 [batch, columns], -1 past a sequence's pages
    kv_lens: torch.Tensor               # int32 [batch]
    cu: torch.Tensor                    # int32 [batch + 1]
    slots: torch.Tensor                 # int32 [tokens]: page * page_size + place in the page, -1 past the last token
    positions: torch.Tensor             # int32 [axes, tokens]


def _rows_of(what: str, state: PageState, rows: torch.Tensor, other: Optional[torch.Tensor], name: str) -> int:
    for t in (rows, other):
        if t is not None and (t.dtype is not _I32 or t.dim() != 1 or t.device != state.device or not t.is_contiguous()):
            raise RuntimeError(f"{what}: rows and {name} must be dense int32 [batch] on the state's device")
    B = rows.shape[0]
    if other is not None and other.shape[0] != B or B > _lib.PLAN_MAX_BATCH:
        raise RuntimeError(f"{what}: rows and {name} must have the same length, at most {_lib.PLAN_MAX_BATCH}")
    return B


def pages_plan(state: PageState, rows: torch.Tensor, counts: torch.Tensor, tokens: int, axes: int = 1,
               images: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> StepMaps:
    """One step: sequence ``rows[i]`` grows by ``counts[i]`` tokens (0: it rests), its new pages come off the free ones, in the
    order of ``rows``.  rows and counts int32 [batch], read on the device; ``tokens`` is the host's room for the
    step's tokens, at least their sum: past it slots are -1 and positions 0.

    ``positions`` are the tokens' places in their sequences, the same on each of ``axes``; with ``images`` =
    (seg_cu int32 [batch + 1], segs int32 [n, 4] of (start, t, h, w); axes = 3) the tokens of rows[i]'s grids
    ``segs[seg_cu[i]:seg_cu[i + 1]]``, in order and beginning at token number ``start`` of the sequence, count by time,
    height and width from the text position they begin at, and the text behind goes on at that position plus
    max(t, h, w).

    A step that cannot be done as a whole (a row twice, too few pages, ...) changes nothing, comes back without pages and
    tokens, and leaves its reason for ``state.check()``."""
    nat = _lib.native()
    if nat is not None:
        got = nat.pages_plan(state._ref, state._index, rows, counts, tokens, axes, *((None, None) if images is None else images))
        if got is not NotImplemented:
            return StepMaps(*got)
    B = _rows_of("pages_plan", state, rows, counts, "counts")
    if tokens < 0 or not 1 <= axes <= _lib.MAX_AXES:
        raise RuntimeError(f"pages_plan: tokens must not be negative, axes 1 to {_lib.MAX_AXES}")
    sc, sp, n = None, None, 0
    if images is not None:
        seg_cu, segs = images
        if not (seg_cu.dtype is _I32 and segs.dtype is _I32 and seg_cu.device == state.device and segs.device == state.device and
                tuple(seg_cu.shape) == (B + 1,) and segs.dim() == 2 and segs.shape[1] == 4 and seg_cu.is_contiguous() and
                segs.is_contiguous() and segs.data_ptr() % 16 == 0):
            raise RuntimeError("pages_plan: images must be dense int32 seg_cu [batch + 1] and segs [n, 4] on the state's device")
        if axes != 3:
            raise RuntimeError("pages_plan: images need 3 axes")
        sc, sp, n = seg_cu.data_ptr(), segs.data_ptr(), segs.shape[0]
    new = lambda *shape: torch.empty(shape, dtype=_I32, device=state.device)               # noqa: E731
    m = StepMaps(new(B, state.columns), new(B), new(B + 1), new(tokens), new(axes, tokens))
    rc = _launch(state._index, _lib.lib().w4a8_pages_plan, state._ref, rows.data_ptr(), counts.data_ptr(), B, tokens, axes, sc, sp, n,
                 m.page_table.data_ptr(), m.kv_lens.data_ptr(), m.cu.data_ptr(), m.slots.data_ptr(), m.positions.data_ptr(),
                 _stream_of(rows))
    if rc != 0:
        _lib.check(rc, "w4a8_pages_plan")
    return m


def pages_shrink(state: PageState, rows: torch.Tensor, keep: Optional[torch.Tensor] = None) -> None:
    """Sequence ``rows[i]`` keeps its first ``keep[i]`` tokens (None: none) and gives back its pages past them, from the last
    page of the last sequence to the first: what ``pages_plan`` over the same rows took, in the places it took it from.
    For sequences that ended and drafted tokens that were not accepted.  Refused as a whole like a plan."""
    nat = _lib.native()
    if nat is not None and nat.pages_shrink(state._ref, state._index, rows, keep) is not NotImplemented:
        return
    B = _rows_of("pages_shrink", state, rows, keep, "keep")
    rc = _launch(state._index, _lib.lib().w4a8_pages_shrink, state._ref, rows.data_ptr(), None if keep is None else keep.data_ptr(),
                 B, _stream_of(rows))
    if rc != 0:
        _lib.check(rc, "w4a8_pages_shrink")


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
