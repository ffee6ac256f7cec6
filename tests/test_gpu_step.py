"""Serving steps whose pages are planned on the GPU, with images' positions on three axes and 8-bit linears among the
4-bit ones, as a program runs them together.

Bound of the step's output against a plain 64-bit model on the dequantised weights, as in test_gpu_decoder.py: int8 codes
with one scale a token round by at most half a step of amax / 127, amax / 127 / sqrt(12) on average; amax of 512 to
768 normal values is 3.2 deviations, 0.73 % (qkv, o, gate_up), and of as many products silu(g) u about 8, 1.8 % (down);
cache 0.9 % twice, ten bf16 roundings of 0.2 %.  sqrt(2 (3 0.73^2 + 1.8^2 + 2 0.9^2 + 10 0.2^2)) % = 3.7 %, doubled as
there: 7.4 %."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_decoder import Plain  # noqa: E402
from test_gpu_pages import places  # noqa: E402

BOUND = 0.074


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _cfg(sections=None, mixed=False):
    from w4a8_b200 import decoder
    return decoder.Config(hidden=512, q_heads=8, kv_heads=2, head_dim=64, ffn=768, group_size=64, page_size=16, positions=256,
                          rope_base=1e4, rope_sections=sections, rope_mixed=mixed)


class PlainAxes(Plain):
    """``Plain`` with the tokens' own positions on several axes: whole sequences at once, causal."""

    def __init__(self, *a, axis_of):
        super().__init__(*a)
        self.axis_of = axis_of

    def run_at(self, x, places):
        c, T, D, half = self.c, x.shape[0], self.c.head_dim, self.c.head_dim // 2
        n, kv = c.q_heads * D, c.kv_heads * D
        freq = c.rope_base ** (-torch.arange(half, dtype=torch.float64) / half)
        ang = torch.tensor(places, dtype=torch.float64)[:, self.axis_of] * freq
        cos, sin = ang.cos()[:, None], ang.sin()[:, None]
        hidden = torch.ones(T, T, dtype=torch.bool).triu(1)
        for w, (n1, n2) in zip(self.w, self.n):
            q, k, v = (t.reshape(T, -1, D) for t in (self.norm(x, n1) @ w["qkv"].T).split((n, kv, kv), 1))
            q, k = (torch.cat([a * cos - b * sin, b * cos + a * sin], -1) for a, b in (q.chunk(2, -1), k.chunk(2, -1)))
            k, v = (t.repeat_interleave(c.q_heads // c.kv_heads, 1) for t in (k, v))
            s = (torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5).masked_fill(hidden, float("-inf"))
            x = x + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(T, n) @ w["o"].T
            gate, up = (self.norm(x, n2) @ w["gate_up"].T).chunk(2, 1)
            x = x + (gate * torch.sigmoid(gate) * up) @ w["down"].T
        return self.norm(x, self.final)


def _build(dev, pages, int8=(), sections=None, mixed=False):
    from w4a8_b200 import decoder, kvcache, ops, vendor
    cfg = _cfg(sections, mixed)
    g = torch.Generator().manual_seed(11)
    layers, weights, norms = [], [], []
    for i in range(2):
        prep, full = {}, {}
        for name, (N, K) in cfg.projections().items():
            if name in int8:
                codes = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
                scale = torch.exp(torch.randn(N, generator=g) * 0.2) / (73.6 * K ** 0.5)
                ckpt = {f"{i}.{name}.weight": codes, f"{i}.{name}.weight_scale": scale[:, None],
                        f"{i}.{name}.weight_offset": torch.zeros(N, 1)}
                prep[name] = vendor.prepare_int8(vendor.load_int8(ckpt.__getitem__, [f"{i}.{name}"]), dev)
                full[name] = codes.double() * scale.double()[:, None]
                continue
            codes = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8)
            scale = torch.exp(torch.randn(K // 64, N, generator=g) * 0.2) / (4.6 * K ** 0.5)
            full[name] = codes.double() * scale.double().T.repeat_interleave(64, 1)
            prep[name] = ops.prepare_weights(ops.pack_int4_grouped(codes, 64).to(dev), scale.to(dev), None, K, 64)
        w = (torch.rand(2, cfg.hidden, generator=g) + 0.5).bfloat16()
        norms.append((w[0].double(), w[1].double()))
        weights.append(full)
        layers.append(decoder.Layer(norm1=w[0].to(dev), norm2=w[1].to(dev), **prep))
    final = (torch.rand(cfg.hidden, generator=g) + 0.5).bfloat16()
    ids = [0] * 32 if sections is None else kvcache.RotaryAxes(sections, mixed).axis_of_pair()
    return decoder.Decoder(cfg, layers, final.to(dev), pages, dev), PlainAxes(cfg, weights, norms, final.double(), axis_of=ids)


@pytest.mark.gpu
@pytest.mark.parametrize("int8,sections,mixed", [((), None, False), (("o", "down"), (8, 12, 12), False),
                                                 (("qkv", "o", "gate_up", "down"), (12, 10, 10), True)])
def test_prompts_images_and_captured_steps(int8, sections, mixed):
    from w4a8_b200 import ops
    dev = _dev()
    dec, plain = _build(dev, 40, int8, sections, mixed)
    for cache in dec.caches:
        cache.k.fill_(127), cache.v.fill_(-127), cache.k_scale.fill_(float("nan")), cache.v_scale.fill_(1e30)
    pages = dec.device_pages(4)
    g = torch.Generator().manual_seed(4)
    grids = {0: [(3, 1, 4, 5), (30, 2, 3, 3)], 2: [(0, 1, 6, 6)], 3: []} if sections else {0: [], 2: [], 3: []}
    xs, seen = {s: [] for s in grids}, {s: [] for s in grids}

    def images(rows):
        if not sections:
            return None
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + len(grids[r]))
        return (torch.tensor(cu, dtype=torch.int32, device=dev),
                torch.tensor([s for r in rows for s in grids[r]], dtype=torch.int32, device=dev).view(-1, 4))

    def step(rows, counts, run=None):
        new = [torch.randn(n, dec.cfg.hidden, generator=g).bfloat16() for n in counts]
        h = torch.cat(new).to(dev)
        y = run(h) if run else dec.step(h, pages.plan(rows, counts, sum(counts), max(counts), images(rows)))
        for s, x, part in zip(rows, new, y.cpu().double().split(list(counts))):
            xs[s].append(x)
            seen[s].append(part)

    step([0, 2], [60, 41])                                      # prompts with images, and one that goes on in chunks
    step([2, 3, 0], [20, 1, 1])
    run = dec.capture_steps(pages, [3, 0, 2], images=images([3, 0, 2]))
    for _ in range(18):                                         # every sequence passes a page's end
        step([3, 0, 2], [1, 1, 1], run)
    step([2, 0], [3, 2])                                        # drafted tokens, some of them not accepted
    pages.shrink([2, 0], [sum(map(len, xs[2])) - 2, sum(map(len, xs[0])) - 1])
    for s, n in ((2, 1), (0, 1)):
        xs[s][-1], seen[s][-1] = xs[s][-1][:n], seen[s][-1][:n]
    step([3, 0, 2], [1, 1, 1], run)
    pages.check()
    for s in grids:
        x, y = torch.cat(xs[s]).double(), torch.cat(seen[s])
        at = places(x.shape[0], grids[s])
        want = plain.run_at(x, at)
        err = ((y - want).norm() / want.norm()).item()
        assert err < BOUND, (s, err)
        if sections and grids[s]:                               # positions on one axis are another model
            assert ((y - plain.run_at(x, [(p,) * 3 for p in range(len(at))])).norm() / want.norm()).item() > BOUND
    pages.release([0, 2, 3])
    pages.check()
    assert pages.state.free_pages.item() == 40 and not pages.state.lens.any()
    assert ops.workspace_status(dev) == 0


@pytest.mark.gpu
def test_pages_on_the_gpu_give_the_same_bits():
    """The same steps on pages kept by the host and on the GPU, eager and captured."""
    dev = _dev()
    outs = []
    for kind in ("host", "gpu", "captured"):
        dec, _ = _build(dev, 24, ("o",))
        for c in dec.caches:
            for t in (c.k, c.v, c.k_scale, c.v_scale):
                t.zero_()
        g = torch.Generator().manual_seed(5)
        seqs = [dec.pages.add() for _ in range(3)] if kind == "host" else [0, 1, 2]
        pages = None if kind == "host" else dec.device_pages(3)
        plan = (lambda n: dec.pages.plan(seqs, n, dev)) if kind == "host" else (lambda n: pages.plan(seqs, n, sum(n), max(n)))
        got = [dec.step(torch.randn(60, 512, generator=g).bfloat16().to(dev), plan([15, 30, 15]))]
        run = dec.capture_steps(pages, seqs) if kind == "captured" else None
        for _ in range(4):
            h = torch.randn(3, 512, generator=g).bfloat16().to(dev)
            got.append((run(h) if run else dec.step(h, plan([1, 1, 1]))).clone())
        outs.append(got + [t for c in dec.caches for t in (c.k, c.v, c.k_scale, c.v_scale)])
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))


@pytest.mark.gpu
def test_sequences_that_rest_and_steps_that_cannot_be():
    dev = _dev()
    dec, _ = _build(dev, 6)
    pages = dec.device_pages(3)
    g = torch.Generator().manual_seed(6)
    h = torch.randn(9, 512, generator=g).bfloat16().to(dev)
    dec.step(h[:8], pages.plan([0, 1], [4, 4], 8, 4))
    run = dec.capture_steps(pages, [0, 1, 2], [1, 0, 2], tokens=3, max_q_len=2)
    run(h[:3])
    assert run.plan.kv_lens.tolist() == [5, 4, 2] and run.plan.cu.tolist() == [0, 1, 1, 3]
    run.counts.copy_(torch.tensor([0, 1, 0]))
    alone = run(h[:3])[:1].clone()
    assert run.plan.kv_lens.tolist() == [5, 5, 2]
    pages.shrink([1], [4])
    assert torch.equal(dec.step(h[:1], pages.plan([1], [1], 1, 1)), alone)
    caches = [t.clone() for c in dec.caches for t in (c.k, c.v, c.k_scale, c.v_scale)]
    run.counts.copy_(torch.tensor([1, 1, 90]))                  # more than the step has rows for
    run(h[:3])
    with pytest.raises(RuntimeError, match="more tokens"):
        pages.check()
    pages.plan([0], [95], 95, 95)                               # more than there are pages
    with pytest.raises(RuntimeError, match="too few free pages|past its columns"):
        pages.check()
    pages.check()
    assert pages.state.lens.tolist() == [5, 5, 2]
    assert all(torch.equal(a, b) for a, b in zip(caches, [t for c in dec.caches for t in (c.k, c.v, c.k_scale, c.v_scale)]))


@pytest.mark.gpu
def test_counts_past_the_longest_that_was_named():
    """A captured step whose counts grow past its max_q_len runs another kernel than the plan of their length would, and
    is as near the plain model."""
    dev = _dev()
    dec, plain = _build(dev, 24)
    for c in dec.caches:
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            t.zero_()
    pages = dec.device_pages(2)
    g = torch.Generator().manual_seed(9)
    xs = [torch.randn(n, 512, generator=g).bfloat16() for n in (20, 17, 30, 2)]
    dec.step(torch.cat(xs[:2]).to(dev), pages.plan([0, 1], [20, 17], 37, 20))
    run = dec.capture_steps(pages, [0, 1], [1, 1], tokens=32, max_q_len=1)
    run.counts.copy_(torch.tensor([30, 2]))
    y = run(torch.cat(xs[2:]).to(dev)).cpu().double()
    pages.check()
    for before, new, got in ((xs[0], xs[2], y[:30]), (xs[1], xs[3], y[30:])):
        x = torch.cat([before, new]).double()
        want = plain.run_at(x, places(x.shape[0], []))[len(before):]
        assert ((got - want).norm() / want.norm()).item() < BOUND


@pytest.mark.gpu
def test_refusals():
    from w4a8_b200 import decoder
    dev = _dev()
    dec, _ = _build(dev, 6, sections=(8, 12, 12))
    pages = dec.device_pages(2)
    h = torch.zeros(2, 512, dtype=torch.bfloat16, device=dev)
    plain = decoder.Pages(6, 16)
    with pytest.raises(RuntimeError, match="rope_sections"):
        dec.step(h, plain.plan([plain.add()], [2], dev))
    run = dec.capture_steps(pages, [0, 1])
    for bad in (h[:1], h.float(), h[:, :256]):
        with pytest.raises(RuntimeError):
            run(bad)
    with pytest.raises(RuntimeError, match="room"):
        dec.capture_steps(pages, [0, 1], [2, 1])
    with pytest.raises(RuntimeError, match="tokens"):
        dec.capture_steps(pages, [])
    for rows, counts in (([0, 1], [1]), (torch.zeros(2, device=dev), [1, 1])):
        with pytest.raises(RuntimeError):
            dec.capture_steps(pages, rows, counts, tokens=2)
    with pytest.raises(RuntimeError, match="images"):
        dec.capture_steps(pages, [0, 1], images=(torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(0, 4, dtype=torch.int32, device=dev)))
    assert pages.state.status() == 0
    a, b = pages.plan([0], [2], 2, 2), pages.plan([0, 1], [1, 1], 2, 2)
    with pytest.raises(RuntimeError):
        a.copy_(b)
    import dataclasses
    with pytest.raises(RuntimeError, match="rotary positions"):
        a.copy_(dataclasses.replace(a, positions=None))
    with pytest.raises(RuntimeError, match="add up"):
        decoder.Decoder(_cfg((8, 8)), dec.layers, dec.final_norm, 4, dev)
    with pytest.raises(RuntimeError):
        decoder.DevicePages(4, 16, 2, 15, dev)


@pytest.mark.gpu
def test_the_command(capsys):
    from w4a8_b200 import decoder
    _dev()
    args = ["--layers", "1", "--batch", "2", "--prompt", "20", "--steps", "2"]
    assert decoder.main(args + ["--gpu-pages", "--int8", "o,down"]) == 0 and decoder.main(args) == 0
    assert "2 sequences" in capsys.readouterr().out
    with pytest.raises(RuntimeError, match="names"):
        decoder.main(args + ["--int8", "embed"])


def test_loading_8_bit_projections():
    from w4a8_b200 import vendor
    g = torch.Generator().manual_seed(1)
    t = {}
    for name, n in (("q", 6), ("k", 3)):
        t[f"{name}.weight"] = torch.randint(-128, 128, (n, 10), generator=g, dtype=torch.int8)
        t[f"{name}.weight_scale"] = torch.rand(n, 1, generator=g)
    t["q.weight_offset"] = torch.zeros(6, 1)
    t["k.bias"] = torch.randn(3, generator=g)
    c = vendor.load_int8(t.__getitem__, ["q", "k"])
    assert torch.equal(c["w"], torch.cat([t["q.weight"], t["k.weight"]]))
    assert torch.equal(c["w_scale"], torch.cat([t["q.weight_scale"], t["k.weight_scale"]])[:, 0])
    assert torch.equal(c["bias"], torch.cat([torch.zeros(6), t["k.bias"]]))
    assert vendor.load_int8(t.__getitem__, ["q"])["bias"] is None
    for name, bad in (("q.weight_offset", torch.ones(6, 1)), ("q.weight", t["q.weight"].float()), ("q.weight_scale", torch.rand(6, 2)),
                      ("k.weight", t["k.weight"][:, :9]), ("k.bias", torch.zeros(2)), ("k.weight", t["k.weight"][0])):
        with pytest.raises(ValueError):
            vendor.load_int8({**t, name: bad}.__getitem__, ["q", "k"])


@pytest.mark.gpu
@pytest.mark.parametrize("mixed", [False, True])
def test_one_section_is_the_ordinary_rotation(mixed):
    """A configuration with a single axis on pages of the GPU, eager and captured: its positions are the tokens' places, so
    the stack gives the bits of one without sections."""
    from w4a8_b200 import ops
    dev = _dev()
    outs = []
    for sections in (None, (32,)):
        dec, _ = _build(dev, 24, ("o",), sections, mixed)
        for c in dec.caches:
            for t in (c.k, c.v, c.k_scale, c.v_scale):
                t.zero_()
        g = torch.Generator().manual_seed(12)
        pages = dec.device_pages(3)
        plan = pages.plan([2, 0, 1], [15, 30, 15], 60, 30)
        assert (plan.positions is None) == (sections is None)
        got = [dec.step(torch.randn(60, 512, generator=g).bfloat16().to(dev), plan)]
        run = dec.capture_steps(pages, [0, 1, 2])
        for _ in range(3):
            got.append(run(torch.randn(3, 512, generator=g).bfloat16().to(dev)).clone())
        pages.check()
        outs.append(got + [t for c in dec.caches for t in (c.k, c.v, c.k_scale, c.v_scale)])
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and ops.workspace_status(dev) == 0


@pytest.mark.gpu
def test_captures_are_made_on_the_decoders_device(monkeypatch):
    """A capture's stream is one of the decoder's GPU, which is made current for it, whichever was: on another's stream
    nothing of the step would be captured.  (One GPU here: what the capture is told is looked at.)"""
    dev = _dev()
    dec, _ = _build(dev, 8)
    inside, seen, real_graph = [], [], torch.cuda.graph

    class Device(torch.cuda.device):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *a):
            inside.pop()
            return super().__exit__(*a)

    def graph(g, *a, stream=None, **k):
        seen.append((stream is not None and stream.device == dev, 0 in inside))
        return real_graph(g, *a, stream=stream, **k)

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    dec.capture(dec.pages.plan([dec.pages.add()], [1], dev))
    dec.capture_steps(dec.device_pages(2), [0, 1])
    assert seen == [(True, True)] * 2
