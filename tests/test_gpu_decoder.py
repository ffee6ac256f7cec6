"""The decoder stack on the package's kernels against a plain 64-bit model on the same
(dequantised) weights, without activation or cache quantisation.

Bound on the relative error of a step's output in the Frobenius norm.  Sources, each
relative to its own tensor: int8 activation codes per 64-element group, a rounding of
at most half a step of amax / 127, on average (uniform) amax / 127 / sqrt(12); amax of 64
normal values is 2.4 deviations, so 0.6 % (four linears a layer); cache codes the same
over a page's tile, amax up to 4 deviations, 0.9 % for v, and for k 0.9 % of a score of
deviation about 1 (weights off by 0.9 %); bf16 roundings of 0.2 % at ten places.  Added in
quadrature over two layers, each source passed on at its size at most (residual sums
and norms only shrink it): sqrt(2 (4 0.6^2 + 2 0.9^2 + 10 0.2^2)) % = 2.6 %.  SwiGLU's product and
the growth of an error through later layers are covered by a factor of 2: 5.2 %.  A row in
the wrong place, a missed residual or a position off by one moves the output by tens of percent.
"""
import pytest

torch = pytest.importorskip("torch")

BOUND = 0.052


def _cfg():
    from w4a8_b200 import decoder
    return decoder.Config(hidden=512, q_heads=8, kv_heads=2, head_dim=64, ffn=768, group_size=64, page_size=16,
                          positions=256, rope_base=1e4)


def test_pages():
    from w4a8_b200 import decoder
    p = decoder.Pages(6, 16)
    a, b = p.add(), p.add()
    plan = p.plan([a, b], [17, 3], "cpu", columns=4)
    assert plan.page_table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]]
    assert plan.kv_lens.tolist() == [17, 3] and plan.cu.tolist() == [0, 17, 20]
    assert (plan.tokens, plan.max_q_len, p.free_pages) == (20, 17, 3)
    with pytest.raises(RuntimeError, match="5 pages needed, 3 free"):
        p.plan([a, b], [1, 78], "cpu")
    assert p.length(a) == 17 and p.length(b) == 3 and p.free_pages == 3     # as before the refusal
    p.release(a)
    nxt = p.plan([b], [14], "cpu")
    assert nxt.page_table.tolist() == [[2, 0]] and nxt.kv_lens.tolist() == [17]
    for seqs, counts in (([], []), ([b, b], [1, 1]), ([b], [0]), ([b], [1, 1])):
        with pytest.raises(RuntimeError):
            p.plan(seqs, counts, "cpu")
    with pytest.raises(RuntimeError, match="another shape"):
        plan.copy_(nxt)
    one = p.plan([b], [1], "cpu")
    wide = p.plan([b], [1], "cpu", columns=4)
    wide.copy_(one)
    assert wide.page_table.tolist() == [[2, 0, -1, -1]] and wide.kv_lens.tolist() == [18]
    with pytest.raises(RuntimeError, match="room"):
        one.copy_(wide)


class Plain:
    """The same layers in 64 bits: whole sequences at once, causal."""

    def __init__(self, cfg, weights, norms, final):
        self.c, self.w, self.n, self.final = cfg, weights, norms, final

    def norm(self, x, w):
        return x / (x.square().mean(-1, keepdim=True) + self.c.eps).sqrt() * w

    def run(self, x):
        c, T = self.c, x.shape[0]
        D, half, n = c.head_dim, c.head_dim // 2, c.q_heads * c.head_dim
        ang = torch.arange(T, dtype=torch.float64)[:, None] * c.rope_base ** (-torch.arange(half, dtype=torch.float64) / half)
        cos, sin = ang.cos()[:, None], ang.sin()[:, None]

        def turn(t):
            a, b = t[..., :half], t[..., half:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        r = x
        for w, (n1, n2) in zip(self.w, self.n):
            qkv = self.norm(r, n1) @ w["qkv"].T
            q, k, v = (t.reshape(T, -1, D) for t in qkv.split((n, c.kv_heads * D, c.kv_heads * D), 1))
            q, k = turn(q), turn(k)
            k, v = (t.repeat_interleave(c.q_heads // c.kv_heads, 1) for t in (k, v))
            s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5
            s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), float("-inf"))
            r = r + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(T, n) @ w["o"].T
            g, u = (self.norm(r, n2) @ w["gate_up"].T).chunk(2, 1)
            r = r + (g * torch.sigmoid(g) * u) @ w["down"].T
        return self.norm(r, self.final)


def _build(dev, pages):
    from w4a8_b200 import decoder, ops
    cfg = _cfg()
    g = torch.Generator().manual_seed(3)
    layers, weights, norms = [], [], []
    for _ in range(2):
        prep, full = {}, {}
        for name, (N, K) in cfg.projections().items():
            codes = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8)
            scale = torch.exp(torch.randn(K // 64, N, generator=g) * 0.2) / (4.6 * K ** 0.5)
            full[name] = codes.double() * scale.double().T.repeat_interleave(64, 1)
            prep[name] = ops.prepare_weights(ops.pack_int4_grouped(codes, 64).to(dev), scale.to(dev), None, K, 64)
        w = (torch.rand(2, cfg.hidden, generator=g) + 0.5).bfloat16()
        norms.append((w[0].double(), w[1].double()))
        weights.append(full)
        layers.append(decoder.Layer(norm1=w[0].to(dev), norm2=w[1].to(dev), **prep))
    final = (torch.rand(cfg.hidden, generator=g) + 0.5).bfloat16()
    return decoder.Decoder(cfg, layers, final.to(dev), pages, dev), Plain(cfg, weights, norms, final.double())


@pytest.mark.gpu
def test_prompts_and_steps_against_plain():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from w4a8_b200 import ops
    dev = torch.device("cuda", 0)
    dec, plain = _build(dev, 24)
    for cache in dec.caches:                        # a new page's old contents must not matter
        cache.k.fill_(127), cache.v.fill_(-127), cache.k_scale.fill_(float("nan")), cache.v_scale.fill_(1e30)
    g = torch.Generator().manual_seed(4)
    xs, seen = {}, {}

    def step(seqs, counts):
        new = [torch.randn(n, dec.cfg.hidden, generator=g).bfloat16() for n in counts]
        plan = dec.pages.plan(seqs, counts, dev)
        h = torch.cat(new).to(dev)
        y = dec.step(h, plan).cpu().double()
        for s, x, part in zip(seqs, new, y.split(list(counts))):
            xs.setdefault(s, []).append(x)
            seen.setdefault(s, []).append(part)

    a, b, c = (dec.pages.add() for _ in range(3))
    step([a, b], [70, 1])                           # a prompt, and one of a single token
    step([a, b, c], [1, 1, 37])                     # another joins while two decode
    step([b, a], [5, 3])                            # several tokens at once, other order
    for _ in range(3):
        step([c, a, b], [1, 1, 1])
    for s in (a, b, c):
        x, y = torch.cat(xs[s]).double(), torch.cat(seen[s])
        want = plain.run(x)
        err = ((y - want).norm() / want.norm()).item()
        assert err < BOUND, (s, err)
    dec.pages.release(a)
    d = dec.pages.add()
    step([d], [33])                                 # on released pages
    want = plain.run(torch.cat(xs[d]).double())
    assert ((torch.cat(seen[d]) - want).norm() / want.norm()).item() < BOUND
    assert ops.workspace_status(dev) == 0


@pytest.mark.gpu
def test_captured_steps_equal_eager_ones():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda", 0)
    outs = []
    for captured in (False, True):
        dec, _ = _build(dev, 24)
        g = torch.Generator().manual_seed(5)
        for cache in dec.caches:
            for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
                t.zero_()
        seqs = [dec.pages.add() for _ in range(3)]
        dec.step(torch.randn(60, dec.cfg.hidden, generator=g).bfloat16().to(dev), dec.pages.plan(seqs, [15, 30, 15], dev))
        got, run = [], None
        for _ in range(4):                          # two sequences cross into a new page
            h = torch.randn(3, dec.cfg.hidden, generator=g).bfloat16().to(dev)
            plan = dec.pages.plan(seqs, [1, 1, 1], dev, 4)
            if captured and run is None:
                run = dec.capture(plan)
            got.append((run(h, plan) if captured else dec.step(h, plan)).clone())
        outs.append(got + [t for c in dec.caches for t in (c.k, c.v, c.k_scale, c.v_scale)])
    for x, y in zip(*outs):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_step_keeps_its_decoder():
    """The graph reads weights, caches and rotary table by address: they live as long as it does.  (Nothing is
    replayed here.)"""
    import gc
    import weakref
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda", 0)
    dec, _ = _build(dev, 24)
    s = dec.pages.add()
    run = dec.capture(dec.pages.plan([s], [1], dev))
    held = [weakref.ref(dec)] + [weakref.ref(t) for L in dec.layers for t in (L.qkv.buf, L.norm1, L.down.buf)]
    held += [weakref.ref(t) for c in dec.caches for t in (c.k, c.v_scale)] + [weakref.ref(dec.cos_sin), weakref.ref(dec.final_norm)]
    dec.layers = []                                # as a caller that goes on to other layers leaves it
    del dec
    gc.collect()
    assert all(r() is not None for r in held)
    del run
    gc.collect()
    assert all(r() is None for r in held)


def test_pages_refuse_lengths_past_the_positions():
    from w4a8_b200 import decoder
    p = decoder.Pages(100, 16, positions=40)
    a, b = p.add(), p.add()
    p.plan([a, b], [39, 40], "cpu")
    free = p.free_pages
    with pytest.raises(RuntimeError, match="41 tokens.*40 positions"):
        p.plan([a, b], [1, 1], "cpu")
    assert (p.length(a), p.length(b), p.free_pages) == (39, 40, free)      # as before the refusal
    assert p.plan([a], [1], "cpu").kv_lens.tolist() == [40]
    c = p.add()
    with pytest.raises(RuntimeError, match="positions"):
        p.plan([c], [41], "cpu")
    unbounded = decoder.Pages(9, 16)
    assert unbounded.plan([unbounded.add()], [100], "cpu").tokens == 100


@pytest.mark.gpu
def test_decoder_refuses_positions_past_its_table():
    """A token without a row in the rotary table is refused, not turned by the last row's angles."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda", 0)
    dec, _ = _build(dev, 40)
    s = dec.pages.add()
    dec.pages.plan([s], [dec.cfg.positions], dev)
    with pytest.raises(RuntimeError, match="positions"):
        dec.pages.plan([s], [1], dev)


@pytest.mark.gpu
def test_captured_step_refuses_what_the_step_refuses():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda", 0)
    dec, _ = _build(dev, 24)
    seqs = [dec.pages.add() for _ in range(3)]
    plan = dec.pages.plan(seqs, [1, 1, 1], dev)
    run = dec.capture(plan)
    for bad in (torch.zeros(1, 512, dtype=torch.bfloat16, device=dev), torch.zeros(512, dtype=torch.bfloat16, device=dev),
                torch.zeros(3, 512, device=dev)):
        for f in (run, dec.step):
            with pytest.raises(RuntimeError):
                f(bad, plan)
