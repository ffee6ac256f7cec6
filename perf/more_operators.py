"""Operators of a serving step on 8-bit layers, image prompts and pages planned on the GPU, as measured cases.

Three operators, each in its plain form (elementary torch operations in 32 bits,
rounded once at the end) and as a user of this package calls it:

int8    a linear in 8-bit integers: activations quantised with one scale per token,
        weights with one scale per output channel, exact integer sums, bf16 out; with a
        bias, behind a residual addition + root-mean-square norm, or on silu(gate) * up
rotary  rotary positions with several axes: each pair of a q or k head turns by the
        position of its token on its own axis (time, height, width)
pages   one step's page table, lengths, offsets, slots and positions built from the
        tokens that each sequence brings, pages taken from the free ones, and given back

Sizes are those of the repository's QwQ-32B layer (hidden 5120, ffn 27648, 40 query heads
and 8 kv heads of 128) and generic ones.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6


def _pkg():
    root = os.path.join(os.getcwd(), "vllm-ascend910_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from w4a8_b200 import kvcache, ops
    return ops, kvcache


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one token through the qkv projection: latency
        dict(name="int8_token", op="int8", m=1, n=7168, k=5120, form="plain", bias=True),
        # a small decode batch through the down projection, the activation applied on the way
        dict(name="int8_down_m16", op="int8", m=16, n=5120, k=27648, form="swiglu", bias=False),
        # a decode batch through norm and gate / up projection: the weights are read once
        dict(name="int8_gate_up_m64", op="int8", m=64, n=55296, k=5120, form="norm", bias=False),
        # a chunk of odd sizes
        dict(name="int8_ragged", op="int8", m=333, n=2056, k=1057, form="plain", bias=True),
        # a prefill chunk through norm and gate / up projection
        dict(name="int8_prefill", op="int8", m=2048, n=55296, k=5120, form="norm", bias=False),
        # one token of text on three axes
        dict(name="rotary_token", op="rotary", t=1, hq=40, hk=8, d=128, sections="16 24 24", mixed=False,
             interleaved=False, grid=False),
        # a prompt with images, the axes' pairs mixed
        dict(name="rotary_prompt", op="rotary", t=8191, hq=40, hk=8, d=128, sections="24 20 20", mixed=True,
             interleaved=False, grid=True),
        # the patches of an image encoder: two axes, heads of 80
        dict(name="rotary_patches", op="rotary", t=5041, hq=16, hk=16, d=80, sections="20 20", mixed=False,
             interleaved=True, grid=True),
        # one token of one sequence
        dict(name="pages_token", op="pages", batch=1, n_min=1, n=1, ctx_min=1000, ctx=1000, page=16, columns=512, axes=1,
             images=0, lens=1),
        # a decode batch with contexts of all lengths
        dict(name="pages_decode", op="pages", batch=256, n_min=1, n=1, ctx_min=1, ctx=8000, page=16, columns=512, axes=1,
             images=0, lens=2),
        # chunks of prompts with images
        dict(name="pages_prompts", op="pages", batch=12, n_min=300, n=4000, ctx_min=0, ctx=3000, page=32, columns=256,
             axes=3, images=5, lens=3),
        # the largest batch, drafted tokens
        dict(name="pages_draft", op="pages", batch=2048, n_min=0, n=5, ctx_min=16, ctx=16000, page=16, columns=1024,
             axes=3, images=1, lens=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("int8", "int8", "rotary", "pages"))
    if op == "int8":
        form = rng.choice(("plain", "plain", "swiglu", "norm"))
        k = _log(rng, 64, 27648)
        if rng.random() < 0.6:
            k = max(64, k // 64 * 64)
        n = _log(rng, 8, 55296)
        if rng.random() < 0.7:
            n = max(8, n // 8 * 8)
        n = min(n, 55296 * 5120 // k)
        m = _log(rng, 1, 8191)
        m = max(1, min(m, 2048 * 55296 * 5120 // (n * k), 3 * 2048 * 5120 // k, 2048 * 55296 // n))
        return dict(op="int8", m=m, n=n, k=k, form=form, bias=rng.random() < 0.5)
    if op == "rotary":
        axes, hk = rng.choice((1, 2, 3, 4)), rng.choice((1, 2, 4, 8))
        d = rng.choice((64, 80, 96, 128, 128, 256))
        rot = rng.choice((d, d, d // 32 * 16))
        cuts = sorted(rng.sample(range(1, rot // 2), axes - 1))
        sections = " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [rot // 2]))
        hq = hk * rng.choice((1, 2, 5, 8))
        t = _log(rng, 1, 7600 * 48 * 128 // ((hq + hk) * max(d, 128)))
        return dict(op="rotary", t=t, hq=hq, hk=hk, d=d, sections=sections, mixed=rng.random() < 0.5,
                    interleaved=rng.random() < 0.5, grid=rng.random() < 0.7)
    page = rng.choice((16, 16, 32, 64, 128))
    kind = rng.choice(("token", "draft", "chunk"))
    batch = _log(rng, 1, 2048) if kind != "chunk" else _log(rng, 1, 32)
    n = 1 if kind == "token" else rng.randint(2, 8) if kind == "draft" else _log(rng, 9, 4096)
    n = max(1, min(n, 16384 // batch))
    ctx = _log(rng, 1, 16000)
    axes = rng.choice((1, 3))
    return dict(op="pages", batch=batch, n_min=rng.choice((0 if batch > 8 else 1, 1, n)), n=n, ctx_min=ctx // rng.choice((1, 2, 8, 100)), ctx=ctx,
                page=page, columns=-(-(ctx + n) // page) + rng.choice((0, 1, 7)), axes=axes,
                images=rng.choice((0, 1, 4)) if axes == 3 else 0, lens=rng.randrange(1 << 20))


def _step(c):
    """(tokens brought, earlier tokens, [(start, t, h, w) of images]) of each sequence: the case's own, whatever the seed."""
    r = random.Random(c["lens"])
    out = []
    for _ in range(c["batch"]):
        n, ctx = r.randint(c["n_min"], c["n"]), r.randint(c["ctx_min"], c["ctx"])
        images, at = [], r.randint(0, 20)
        for _ in range(c["images"]):
            t, h, w = r.choice((1, 1, 1, 4, 9)), r.randint(1, 32), r.randint(1, 32)
            images.append((at, t, h, w))
            at += t * h * w + r.randint(0, 50)
        out.append((n, ctx, images))
    return out


def work(case):
    c = case
    if c["op"] == "int8":
        m, n, k = c["m"], c["n"], c["k"]
        x = {"plain": 2, "swiglu": 4, "norm": 6}[c["form"]] * m * k + (2 * k if c["form"] == "norm" else 0)
        return {"bytes": x + n * k + 4 * n * (2 if c["bias"] else 1) + 2 * m * n, "flops": 2 * m * n * k}
    if c["op"] == "rotary":
        rot, heads = 2 * sum(_sections(c)), c["hq"] + c["hk"]
        return {"bytes": c["t"] * (4 * heads * c["d"] + 4 * rot + 4 * len(_sections(c))), "flops": 3 * c["t"] * heads * rot}
    s, page = _step(c), c["page"]
    held = sum(-(-(n + x) // page) for n, x, _ in s)
    new = sum(-(-(n + x) // page) - -(-x // page) for n, x, _ in s)
    toks = sum(n for n, _, _ in s)
    # counts, rows and lengths in; lengths and offsets out; the held pages in, all columns out; new pages off the
    # free ones, into the sequences' table and back; slots and positions out; images in
    by = c["batch"] * 4 * 6 + 4 * held + 4 * c["batch"] * c["columns"] + 16 * new + 4 * toks * (1 + c["axes"])
    return {"bytes": by + 16 * c["images"] * c["batch"], "flops": 4 * toks + 4 * c["batch"]}


# ------------------------------------------------------------------ inputs

def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFFFFFF)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).to("cuda")


def _sections(c):
    return [int(n) for n in c["sections"].split()]


def _axis_of(c):
    """The axis of each pair: the sections one after another, or mixed (0 1 2 0 1 2 ..., a used-up axis left out)."""
    if not c["mixed"]:
        return [a for a, n in enumerate(_sections(c)) for _ in range(n)]
    left, out = list(_sections(c)), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def prepare(case, seed):
    c = case
    g = _gen(seed, 2)
    if c["op"] == "int8":
        m, n, k = c["m"], c["n"], c["k"]
        wide = 2 * k if c["form"] == "swiglu" else k
        x = _randn(g, m, wide)
        x[:, torch.randperm(wide, generator=g, device="cuda")[: max(1, wide // 200)]] *= 20.0
        w = torch.empty(n, k, dtype=torch.int8, device="cuda")
        for i in range(0, n, 8192):
            w[i:i + 8192] = (40.0 * _randn(g, min(8192, n - i), k)).round().clamp(-127, 127).to(torch.int8)
        s = {"case": c, "x": x.to(torch.bfloat16), "w": w, "w_scale": torch.exp(0.2 * _randn(g, n)) / (40.0 * k ** 0.5),
             "bias": 0.5 * _randn(g, n) if c["bias"] else None}
        if c["form"] == "norm":
            s["norm"] = (1.0 + 0.2 * _randn(g, k)).to(torch.bfloat16)
            s["residual"] = (3.0 * _randn(g, m, k)).to(torch.bfloat16)
        if own:   # the layer as a serving program holds it after loading
            s["layer"] = _pkg()[0].prepare_int8(w, s["w_scale"], s["bias"])
        return s
    if c["op"] == "rotary":
        t, d, rot, axes = c["t"], c["d"], 2 * sum(_sections(c)), len(_sections(c))
        rows = t + 40
        # one row [q | k | v] for each token, as the linear before hands it over
        qkv = _randn(g, t, (c["hq"] + 2 * c["hk"]) * d).to(torch.bfloat16)
        pos = torch.arange(t, device="cuda").repeat(axes, 1) + int(torch.randint(0, 32, (1,), generator=g, device="cuda"))
        if c["grid"]:   # each axis its own coordinate of a grid about as wide as high
            side = max(1, math.isqrt(t))
            for a in range(axes):
                pos[a] = (torch.arange(t, device="cuda") // side ** (axes - 1 - a)) % max(side, 2) + a
        freq = 1e6 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
        ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
        s = {"case": c, "q": qkv[:, :c["hq"] * d].view(t, c["hq"], d),
             "k": qkv[:, c["hq"] * d:(c["hq"] + c["hk"]) * d].view(t, c["hk"], d),
             "table": torch.cat([ang.cos(), ang.sin()], 1).float(), "positions": pos.to(torch.int32),
             "axis_of": torch.tensor(_axis_of(c), device="cuda")}
        if own:   # which pair goes with which axis: the model's own
            s["axes"] = _pkg()[1].RotaryAxes(_sections(c), mixed=c["mixed"])
        return s
    step, page, cols, batch = _step(c), c["page"], c["columns"], c["batch"]
    held = [-(-x // page) for _, x, _ in step]
    new = sum(-(-(n + x) // page) - h for (n, x, _), h in zip(step, held))
    spare, sequences = 5, batch + 3
    total = sum(held) + new + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    rows = torch.randperm(sequences, generator=g, device="cuda")[:batch]
    h = torch.tensor(held, device="cuda")
    table = torch.full((sequences, cols), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(cols, device="cuda")
    src = (h.cumsum(0) - h)[:, None] + at
    table[rows] = torch.where(at < h[:, None], order[src.clamp(max=total - 1)], table[rows])
    lens = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    lens[rows] = _i32([x for _, x, _ in step])
    seg_cu, segs = [0], []
    for _, _, images in step:
        segs += images
        seg_cu.append(len(segs))
    s = {"case": c, "rows": rows.to(torch.int32), "counts": _i32([n for n, _, _ in step]),
         "keep": _i32([x for _, x, _ in step]), "tokens": sum(n for n, _, _ in step), "table": table, "lens": lens,
         "free": order.roll(-sum(held)).contiguous(), "free_pages": torch.tensor([total - sum(held)], dtype=torch.int32,
                                                                                  device="cuda"),
         "images": (_i32(seg_cu), _i32(segs).view(-1, 4)) if c["images"] else None}
    if own:
        s["state"] = _pkg()[1].PageState(s["free"], s["free_pages"], table, lens, page)
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"int8": _int8_own, "rotary": _rotary_own, "pages": _pages_own}[op](state)
    return {"int8": _int8_plain, "rotary": _rotary_plain, "pages": _pages_plain}[op](state)


def _int8_own(s):
    ops, _ = _pkg()
    form = s["case"]["form"]
    if form == "norm":
        return list(ops.linear_int8_rms_norm(s["x"], s["norm"], s["layer"], EPS, residual=s["residual"]))
    return ops.linear_int8(s["x"], s["layer"], act="swiglu" if form == "swiglu" else None)


def _int8_plain(s):
    c, res = s["case"], None
    h = s["x"].float()
    if c["form"] == "swiglu":
        gate, up = h.chunk(2, 1)
        h = (gate / (1.0 + torch.exp(-gate)) * up).to(torch.bfloat16).float()   # the activation is a bf16 tensor
    elif c["form"] == "norm":
        h = h + s["residual"].float()
        res = h.to(torch.bfloat16)
        h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["norm"].float()
    amax = h.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    q = torch.where(scale == 0, torch.zeros((), device="cuda"), (h / scale).round().clamp(-127, 127))
    total = torch.zeros(c["m"], c["n"], dtype=torch.int32, device="cuda")
    for i in range(0, c["k"], 1024):          # sums of 1024 products are exact in 32 bits
        total += (q[:, i:i + 1024] @ s["w"][:, i:i + 1024].float().T).to(torch.int32)
    y = total.float().mul_(scale).mul_(s["w_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y.to(torch.bfloat16)
    return [y, res] if res is not None else y


def _rotary_own(s):
    _, kvcache = _pkg()
    return list(kvcache.rotary(s["q"], s["k"], s["table"], s["positions"], s["axes"], interleaved=s["case"]["interleaved"]))


def _rotary_plain(s):
    half = s["axis_of"].shape[0]
    row = s["positions"].long()[s["axis_of"]]                  # [pairs, tokens]
    i = torch.arange(half, device="cuda")[:, None]
    cos, sin = s["table"][row, i].T.unsqueeze(1), s["table"][row, i + half].T.unsqueeze(1)
    out = []
    for x in (s["q"], s["k"]):
        x = x.float()
        rot, rest = x[..., :2 * half], x[..., 2 * half:]
        if s["case"]["interleaved"]:
            a, b = rot[..., 0::2], rot[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = rot[..., :half], rot[..., half:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([turned, rest], -1).to(torch.bfloat16))
    return out


def _pages_own(s):
    # a step's tokens, all of them drafted ones that the step then rejects: the pages come and go
    _, kvcache = _pkg()
    m = kvcache.pages_plan(s["state"], s["rows"], s["counts"], s["tokens"], axes=s["case"]["axes"], images=s["images"])
    kvcache.pages_shrink(s["state"], s["rows"], s["keep"])
    return [m.page_table, m.kv_lens, m.cu, m.slots, m.positions, s["table"], s["lens"], s["free"], s["free_pages"]]


def _pages_plain(s):
    c, dev = s["case"], "cuda"
    page, cols, tokens, batch = c["page"], c["columns"], s["tokens"], c["batch"]
    rows, n = s["rows"].long(), s["counts"].long()
    was = s["lens"][rows].long()
    now = was + n
    before = torch.div(was + page - 1, page, rounding_mode="floor")
    after = torch.div(now + page - 1, page, rounding_mode="floor")
    need = after - before
    taken = need.cumsum(0) - need
    # the j-th new page of the step is the j-th from the top of the free ones
    at = torch.arange(cols, device=dev)
    nth = taken[:, None] + at - before[:, None]
    fresh = (at >= before[:, None]) & (at < after[:, None])
    pick = (s["free_pages"].long() - 1 - nth).clamp(0, s["free"].shape[0] - 1)
    page_table = torch.where(fresh, s["free"][pick], s["table"][rows])
    cu = torch.zeros(batch + 1, dtype=torch.int64, device=dev)
    cu[1:] = n.cumsum(0)
    seq = torch.repeat_interleave(torch.arange(batch, device=dev), n, output_size=tokens)
    pos = torch.arange(tokens, device=dev) - cu[seq] + was[seq]
    slots = page_table[seq, torch.div(pos, page, rounding_mode="floor")].long() * page + pos % page
    places = pos.repeat(c["axes"], 1)
    if s["images"] is not None:
        seg_cu, segs = s["images"][0].long(), s["images"][1].long()
        size = segs[:, 1] * segs[:, 2] * segs[:, 3]
        step = segs[:, 1:].amax(1) - size                     # how far positions fall behind past a grid
        run_ = step.cumsum(0)
        owner = torch.repeat_interleave(torch.arange(batch, device=dev), seg_cu[1:] - seg_cu[:-1], output_size=segs.shape[0])
        first = torch.where(seg_cu[:-1] > 0, run_[(seg_cu[:-1] - 1).clamp(min=0)], torch.zeros((), dtype=torch.int64, device=dev))
        behind = run_ - first[owner]                          # of the sequence's grids up to this one
        last = torch.searchsorted(owner * (1 << 32) + segs[:, 0], seq * (1 << 32) + pos, right=True) - 1
        there = last >= seg_cu[seq]                           # a grid begins at or before the token
        last = last.clamp(min=0)
        r = pos - segs[last, 0]
        inside = there & (r < size[last])
        base = segs[last, 0] + behind[last] - step[last]
        _, h, w = segs[last, 1], segs[last, 2], segs[last, 3]
        grid = torch.stack([base + torch.div(r, h * w, rounding_mode="floor"),
                            base + torch.div(r, w, rounding_mode="floor") % h, base + r % w])
        text = pos + torch.where(there, behind[last], torch.zeros((), dtype=torch.int64, device=dev))
        places = torch.where(inside, grid, text.expand(3, -1))
    # the rejected tokens' pages go back where they came from: what the sequences hold is as before
    s["lens"][rows] = (now - n).to(torch.int32)
    put = lambda v: v.to(torch.int32)                                                       # noqa: E731
    return [page_table, put(now), put(cu), put(slots), put(places), s["table"], s["lens"], s["free"], s["free_pages"]]


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"int8": _int8_exact, "rotary": _rotary_exact, "pages": _pages_exact}[case["op"]](case, s)


def _int8_exact(c, s):
    if 2 * c["m"] * c["n"] * c["k"] > 3e14:       # (about 10 seconds of 64-bit products)
        return None
    x, res = s["x"].double(), None
    if c["form"] == "swiglu":
        x = (x[:, :c["k"]] * torch.sigmoid(x[:, :c["k"]]) * x[:, c["k"]:]).to(torch.bfloat16).double()
    elif c["form"] == "norm":
        res = x + s["residual"].double()
        x = res / torch.sqrt(res.square().sum(1, keepdim=True) / c["k"] + EPS) * s["norm"].double()
    scale = (x.abs().max(1, keepdim=True).values / 127).float().double()     # (held in 32 bits)
    q = torch.round(x / torch.where(scale == 0, torch.ones_like(scale), scale)).clamp(-127, 127)
    y = torch.empty(c["m"], c["n"], dtype=torch.float64, device="cuda")
    for i in range(0, c["n"], 8192):
        y[:, i:i + 8192] = torch.mm(q, s["w"][i:i + 8192].double().t()) * scale * s["w_scale"][i:i + 8192].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    return [y, res] if res is not None else y


def _rotary_exact(c, s):
    half = sum(_sections(c))
    t, out = s["table"].double(), []
    z = torch.empty(c["t"], half, dtype=torch.complex128, device="cuda")
    for i, a in enumerate(_axis_of(c)):
        rows = t.index_select(0, s["positions"][a].long())
        z[:, i] = torch.complex(rows[:, i], rows[:, half + i])
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        u, v = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["interleaved"] else (slice(0, half), slice(half, 2 * half))
        w = torch.complex(y[..., u].contiguous(), y[..., v].contiguous()) * z[:, None]
        y[..., u], y[..., v] = w.real, w.imag
        out.append(y)
    return out


def _pages_exact(c, s):
    page, step = c["page"], _step(c)
    free = s["free"].tolist()[:int(s["free_pages"])]
    rows, table = s["rows"].tolist(), s["table"].tolist()
    out, lens, cu, slots, places = [], [], [0], [], []
    for row, (n, ctx, images) in zip(rows, step):
        held = table[row][: -(-ctx // page)]
        while len(held) * page < ctx + n:
            held.append(free.pop())
        out.append(held + [-1] * (c["columns"] - len(held)))
        lens.append(ctx + n)
        cu.append(cu[-1] + n)
        slots += [held[p // page] * page + p % page for p in range(ctx, ctx + n)]
        # the sequence's places from its first token on
        grids, at, p = list(images), 0, 0
        while p < ctx + n:
            if grids and grids[0][0] == p:
                _, t, h, w = grids.pop(0)
                places += [(at + r // (h * w), at + r // w % h, at + r % w)
                           for r in range(max(0, ctx - p), min(t * h * w, ctx + n - p))]
                p, at = p + t * h * w, at + max(t, h, w)
            else:
                stop = min(grids[0][0] if grids else ctx + n, ctx + n)
                places += [(at + i - p,) * 3 for i in range(max(p, ctx), stop)]
                p, at = stop, at + stop - p
    put = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")                       # noqa: E731
    return [put(out).view(c["batch"], c["columns"]), put(lens), put(cu), put(slots),
            put(places).view(-1, 3).T[:c["axes"]].contiguous(), s["table"], s["lens"], s["free"], s["free_pages"]]
