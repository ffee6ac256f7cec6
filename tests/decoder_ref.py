"""Plain implementations that the decoder-operator tests compare with (CPU, 64 bits
or IEEE fp32 where the operator's definition is in fp32)."""
import numpy as np
import torch


def bf16_np(t):
    """A bf16 tensor as float64 numpy."""
    return t.detach().float().cpu().numpy().astype(np.float64)


def attention64(q, codes_k, codes_v, scale_k, scale_v, table, lens, cu, scale):
    """Output and sum_j p_j |v_j| + n 2^-28 vmax of each row, in 64 bits (n visible tokens, vmax = 128
    times their largest page scale of v: see the bound in test_gpu_attention.py).  q float64 [T, Hq, D];
    codes [P, Hkv, page, D]; a page id outside the cache holds no tokens."""
    T, hq, D = q.shape
    P, hkv, page, _ = codes_k.shape
    out, mag = np.zeros((T, hq, D)), np.zeros((T, hq, D))
    for s in range(len(lens)):
        n, L = cu[s + 1] - cu[s], lens[s]
        if n == 0:
            continue
        ids = np.array([table[s][j // page] if j // page < len(table[s]) else -1 for j in range(L)], dtype=np.int64)
        there = (ids >= 0) & (ids < P)
        pos = np.arange(L)[there]
        ids = ids[there]
        for h in range(hq):
            g = h // (hq // hkv)
            k = codes_k[ids, g, pos % page].astype(np.float64) * scale_k[ids, g].astype(np.float64)[:, None]
            v = codes_v[ids, g, pos % page].astype(np.float64) * scale_v[ids, g].astype(np.float64)[:, None]
            for i in range(n):
                seen = pos <= L - n + i
                if not seen.any():
                    continue
                z = (k[seen] @ q[cu[s] + i, h]) * scale
                p = np.exp(z - z.max())
                p /= p.sum()
                out[cu[s] + i, h] = p @ v[seen]
                floor = seen.sum() * 2.0 ** -28 * 128 * scale_v[ids[seen], g].max()
                mag[cu[s] + i, h] = p @ np.abs(v[seen]) + floor
    return out, mag


def rotate32(x, pos, table, interleaved):
    """fp32 rotation with separately rounded products; x fp32 [T, H, D], pos int64 [T]."""
    half = table.shape[1] // 2
    cs = table[pos].unsqueeze(1)
    c, s = cs[..., :half], cs[..., half:]
    x = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    u, v = x[..., a].clone(), x[..., b].clone()
    x[..., a] = u * c - v * s
    x[..., b] = v * c + u * s
    return x


def write32(codes, scales, x, table, lens, cu):
    """The cache write's definition on CPU tensors in fp32: x [T, Hkv, D] rounded into codes / scales in place."""
    P, H, page, D = codes.shape
    for s in range(len(lens)):
        n = cu[s + 1] - cu[s]
        start = lens[s] - n
        for pg in range(max(start, 0) // page, -(-lens[s] // page) if lens[s] > 0 else 0):
            if n == 0 or pg >= len(table[s]) or not 0 <= table[s][pg] < P:
                continue
            at, pid = pg * page, table[s][pg]
            lo, hi = max(start - at, 0), min(lens[s] - at, page)
            first = max(lo, -at)
            if start < 0:
                first = max(first, 0)
            rows = x[cu[s] + at + first - start: cu[s] + at + hi - start]      # [m, H, D]
            if rows.shape[0] == 0:
                continue
            amax = rows.abs().amax((0, 2))
            now = amax / torch.full_like(amax, 127.0)
            if lo > 0:
                was = scales[pid].clone()
                now = torch.where((was >= now) | was.isnan(), was, now)
                ratio = was / now
                grew = (now != was)
                old = (codes[pid][:, :lo].float() * ratio[:, None, None]).round().nan_to_num(0.0).to(torch.int8)
                codes[pid][:, :lo] = torch.where(grew[:, None, None], old, codes[pid][:, :lo])
            q = (rows / now[None, :, None]).round().clamp(-127, 127).nan_to_num(0.0)
            usable = (now > 0) & torch.isfinite(now)
            q = torch.where(usable[None, :, None], q, torch.zeros(()))
            codes[pid][:, first:hi] = q.to(torch.int8).transpose(0, 1)
            scales[pid] = now


def norm64(x, res, w, eps):
    """(y, h) in 64 bits."""
    h = bf16_np(x) + (0 if res is None else bf16_np(res))
    return h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w, h
