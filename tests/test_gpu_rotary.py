"""Rotary positions with several axes: the definition's arithmetic in IEEE fp32 (products rounded one by one), the
same bits, alone and on the way into the cache."""
import pytest

torch = pytest.importorskip("torch")

from decoder_ref import write32  # noqa: E402

BF = torch.bfloat16


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def turn32(x, positions, axis_of, table, interleaved):
    """x [T, H, D] fp32, positions [axes, T], the pairs' axes."""
    half = len(axis_of)
    rows = positions.long().clamp(0, table.shape[0] - 1)[torch.tensor(axis_of)]      # [pairs, T]
    i = torch.arange(half)[:, None]
    c, s = table[rows, i].T[:, None], table[rows, half + i].T[:, None]
    x = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    u, v = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = u * c - v * s, v * c + u * s
    return x


def test_axes_of_pairs():
    from w4a8_b200 import kvcache
    assert kvcache.RotaryAxes([2, 3, 3]).axis_of_pair() == [0, 0, 1, 1, 1, 2, 2, 2]
    assert kvcache.RotaryAxes([4, 2, 2], mixed=True).axis_of_pair() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert kvcache.RotaryAxes([8]).axis_of_pair() == [0] * 8
    m = kvcache.RotaryAxes([24, 20, 20], mixed=True).axis_of_pair()
    assert m[:6] == [0, 1, 2, 0, 1, 2] and m[60:] == [0] * 4 and len(m) == 64
    for bad in ([], [8, 0], [1, 2, 3], [2] * 5, [200], [4, -4, 8]):
        with pytest.raises(RuntimeError):
            kvcache.RotaryAxes(bad)


def test_tables_that_begin_again():
    from w4a8_b200 import kvcache
    one = kvcache.rotary_table(48, 9, base=1e4, device="cpu")
    two = kvcache.rotary_table(96, 9, base=1e4, device="cpu", repeat=2)
    assert torch.equal(two, torch.cat([one[:, :24], one[:, :24], one[:, 24:], one[:, 24:]], 1))
    assert kvcache.rotary_table(80, 4, device="cpu", repeat=2).shape == (4, 80)
    for k in ({"repeat": 0}, {"repeat": 3}, {"repeat": -1}):
        with pytest.raises(RuntimeError):
            kvcache.rotary_table(80, 4, device="cpu", **k)


CASES = [
    # tokens, q heads, k heads, head_dim, sections, mixed, interleaved
    (1, 40, 8, 128, [16, 24, 24], False, False),
    (5, 5, 1, 128, [24, 20, 20], True, False),
    (37, 3, 3, 80, [20, 20], False, True),
    (3, 2, 1, 72, [11, 13, 8], True, False),          # 8 elements past the rotated ones
    (600, 2, 2, 64, [8, 12, 12], False, False),
    (70, 7, 2, 256, [40, 40, 40, 8], True, True),
    (9, 1, 1, 8 + 16, [8], False, False),
    (2, 1, 4, 96, [5, 3, 4, 4], False, True),
    (4099, 4, 1, 128, [1, 62, 1], False, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hk,d,sections,mixed,inter", CASES)
def test_rotary(T, hq, hk, d, sections, mixed, inter):
    from w4a8_b200 import kvcache
    dev = _dev()
    g = torch.Generator().manual_seed(T + d)
    axes = kvcache.RotaryAxes(sections, mixed=mixed)
    table = kvcache.rotary_table(2 * axes.pairs, 50, base=1e4, device="cpu")
    q, k = (torch.randn(T, h, d, generator=g).to(BF) for h in (hq, hk))
    pos = torch.randint(-3, 60, (axes.axes, T), generator=g, dtype=torch.int32)      # past both ends of the table
    want = [turn32(x.float(), pos, axes.axis_of_pair(), table, inter).to(BF) for x in (q, k)]
    td, pd = table.to(dev), pos.to(dev)
    got = kvcache.rotary(q.to(dev), k.to(dev), td, pd, axes, interleaved=inter)
    assert all(torch.equal(x.cpu(), w) for x, w in zip(got, want))
    # views of one row, positions with longer rows; in place
    wide = torch.randn(T, (hq + hk) * d + 8, generator=g).to(BF).to(dev)
    qv, kv = wide[:, :hq * d].unflatten(1, (hq, d)), wide[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    qv.copy_(q), kv.copy_(k)
    before = wide[:, (hq + hk) * d:].clone()
    long = torch.zeros(axes.axes, T + 7, dtype=torch.int32, device=dev)
    long[:, 2:T + 2] = pd
    got = kvcache.rotary(qv, kv, td, long[:, 2:T + 2], axes, interleaved=inter, q_out=qv, k_out=kv)
    assert got[0].data_ptr() == qv.data_ptr() and got[1].data_ptr() == kv.data_ptr()
    assert torch.equal(qv.cpu(), want[0]) and torch.equal(kv.cpu(), want[1]) and torch.equal(wide[:, (hq + hk) * d:], before)
    # rows that begin at odd addresses, and q alone
    odd = torch.zeros(T, hq * d + 3, dtype=BF, device=dev)
    odd[:, 1:hq * d + 1] = q.flatten(1).to(dev)
    got = kvcache.rotary(odd[:, 1:hq * d + 1].unflatten(1, (hq, d)), None, td, pd, axes, interleaved=inter)
    assert got[1] is None and torch.equal(got[0].cpu(), want[0])


@pytest.mark.gpu
def test_one_axis_is_the_ordinary_rotation():
    from w4a8_b200 import kvcache
    dev = _dev()
    q = torch.randn(20, 4, 128, device=dev).to(BF)
    table = kvcache.rotary_table(128, 64)
    pos = torch.arange(20, dtype=torch.int32, device=dev)
    a, _ = kvcache.rotary(q, None, table, pos)
    b, _ = kvcache.rotary(q, None, table, pos.view(1, -1), kvcache.RotaryAxes([64]))
    c, _ = kvcache.rotary(q, None, table, pos.repeat(3, 1), kvcache.RotaryAxes([24, 20, 20], mixed=True))
    cache = kvcache.KVCache.empty(2, 1, 16, 128, dev)
    i = dict(dtype=torch.int32, device=dev)
    kv = torch.zeros(20, 1, 128, dtype=BF, device=dev)
    want = kvcache.kv_write(cache, kv, kv, torch.tensor([[0, 1]], **i), torch.tensor([20], **i), torch.tensor([0, 20], **i), q=q,
                            cos_sin=table)
    assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(c, want)


WRITES = [
    # hkv, hq, d, page, query tokens, lengths after, sections, mixed, interleaved
    (1, 5, 128, 16, [1], [1], [16, 24, 24], False, False),
    (8, 40, 128, 16, [1, 1, 1], [17, 32, 100], [24, 20, 20], True, False),
    (2, 4, 128, 32, [50, 3, 33], [50, 40, 65], [10, 22], False, True),
    (3, 6, 64, 64, [200], [200], [8, 12, 12], True, False),
    (2, 2, 128, 128, [129, 1], [300, 257], [16, 16, 16], False, False),
    (2, 3, 64, 128, [40, 0, 9], [47, 3, 9], [8], False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,hq,d,page,qs,lens,sections,mixed,inter", WRITES)
def test_cache_write_at_positions_of_their_own(hkv, hq, d, page, qs, lens, sections, mixed, inter):
    from w4a8_b200 import kvcache
    dev = _dev()
    g = torch.Generator().manual_seed(hkv + d + page)
    axes = kvcache.RotaryAxes(sections, mixed=mixed)
    table = kvcache.rotary_table(2 * axes.pairs, 70, base=1e4, device="cpu")
    npages = [-(-n // page) for n in lens]
    P, at, pages = sum(npages) + 2, 0, []
    for n in npages:
        pages.append(list(range(at, at + n)) + [-1] * (max(npages) - n))
        at += n
    codes = [torch.randint(-127, 128, (P, hkv, page, d), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(P, hkv, generator=g) * 0.02 for _ in range(2)]
    cache = kvcache.KVCache(*[x.to(dev) for x in codes + scales])
    T = sum(qs)
    q, k, v = (torch.randn(T, h, d, generator=g).to(BF) for h in (hq, hkv, hkv))
    pos = torch.randint(-2, 80, (axes.axes, T), generator=g, dtype=torch.int32)
    cu = [0]
    for n in qs:
        cu.append(cu[-1] + n)
    i = dict(dtype=torch.int32, device=dev)
    got = kvcache.kv_write(cache, k.to(dev), v.to(dev), torch.tensor(pages, **i), torch.tensor(lens, **i), torch.tensor(cu, **i),
                           q=q.to(dev), cos_sin=table.to(dev), interleaved=inter, positions=pos.to(dev), axes=axes)
    ids = axes.axis_of_pair()
    assert torch.equal(got.cpu(), turn32(q.float(), pos, ids, table, inter).to(BF))
    write32(codes[0], scales[0], turn32(k.float(), pos, ids, table, inter), pages, lens, cu)
    write32(codes[1], scales[1], v.float(), pages, lens, cu)
    for mine, plain in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), codes + scales):
        assert torch.equal(mine.cpu(), plain)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A q of more than 2^31 elements: its last tokens."""
    from w4a8_b200 import kvcache
    dev = _dev()
    T, H, D = (1 << 31) // (64 * 256) + 5, 64, 256
    q = torch.zeros(T, H, D, dtype=BF, device=dev)
    q[-5:] = torch.randn(5, H, D, device=dev).to(BF)
    table, axes = kvcache.rotary_table(256, 40), kvcache.RotaryAxes([60, 68])
    pos = torch.zeros(2, T, dtype=torch.int32, device=dev)
    pos[:, -5:] = torch.tensor([[1, 2, 3, 4, 5], [9, 8, 7, 39, 50]], dtype=torch.int32, device=dev)
    tail = q[-5:].float().cpu()
    kvcache.rotary(q, None, table, pos, axes, q_out=q)
    assert torch.equal(q[-5:].cpu(), turn32(tail, pos[:, -5:].cpu(), axes.axis_of_pair(), table.cpu(), False).to(BF))
    assert not q[:-5].any()


@pytest.mark.gpu
def test_captured_positions_and_refusals():
    from w4a8_b200 import kvcache
    dev = _dev()
    axes, table = kvcache.RotaryAxes([24, 20, 20]), kvcache.rotary_table(128, 30)
    q, k = torch.randn(6, 4, 128, device=dev).to(BF), torch.randn(6, 2, 128, device=dev).to(BF)
    pos = torch.zeros(3, 6, dtype=torch.int32, device=dev)
    kvcache.rotary(q, k, table, pos, axes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kvcache.rotary(q, k, table, pos, axes)
    pos.copy_(torch.randint(0, 30, (3, 6)))
    graph.replay()
    want = kvcache.rotary(q, k, table, pos, axes)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    cache = kvcache.KVCache.empty(2, 2, 16, 128, dev)
    i = dict(dtype=torch.int32, device=dev)
    batch = (torch.tensor([[0]], **i), torch.tensor([6], **i), torch.tensor([0, 6], **i))
    bad = [
        lambda: kvcache.rotary(q.float(), k, table, pos, axes), lambda: kvcache.rotary(q, k[:5], table, pos, axes),
        lambda: kvcache.rotary(q, k[..., :64], table, pos, axes), lambda: kvcache.rotary(q, k, table, pos[:2], axes),
        lambda: kvcache.rotary(q, k, table, pos.long(), axes), lambda: kvcache.rotary(q, k, table, pos[:, :5], axes),
        lambda: kvcache.rotary(q, k, table, pos.cpu(), axes), lambda: kvcache.rotary(q, k, table.double(), pos, axes),
        lambda: kvcache.rotary(q, k, table, pos), lambda: kvcache.rotary(q, k, table, pos, kvcache.RotaryAxes([8, 8, 8])),
        lambda: kvcache.rotary(q, k, table[:0], pos, axes), lambda: kvcache.rotary(q, None, table, pos, axes, k_out=k),
        lambda: kvcache.rotary(q, k, table, pos, axes, q_out=k), lambda: kvcache.rotary(q.cpu(), k, table, pos, axes),
        lambda: kvcache.rotary(q[..., :64].contiguous(), None, table, pos, axes), lambda: kvcache.rotary(q[:, 0], None, table, pos, axes),
        lambda: kvcache.rotary(q, k, table, pos, axes, q_out=torch.zeros(6, 4 * 128 + 1, dtype=BF, device=dev)[:, 1:].unflatten(1, (4, 128))),
        lambda: kvcache.kv_write(cache, k, k, *batch, q=q, positions=pos, axes=axes),
        lambda: kvcache.kv_write(cache, k, k, *batch, q=q, cos_sin=table, axes=axes),
        lambda: kvcache.kv_write(cache, k, k, *batch, q=q, cos_sin=table, positions=pos[:, :5], axes=axes),
        lambda: kvcache.kv_write(cache, k, k, *batch, q=q, cos_sin=table, positions=pos),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    assert kvcache.rotary(q[:0], k[:0], table, pos[:, :0], axes)[1].shape == (0, 2, 128)


MANY = [
    # tokens, q heads, k heads, head_dim, sections, mixed, interleaved: four, eight or sixteen tokens a block, the last block partly full
    (661, 16, 16, 80, [20, 20], False, True),
    (602, 5, 4, 128, [24, 20, 20], True, True),
    (601, 3, 2, 128, [16, 24, 24], False, False),
    (607, 2, 3, 128, [16, 24, 24], True, True),
    (611, 1, 1, 96, [5, 3, 4, 4], False, True),
    (650, 1, 0, 64, [8, 12, 12], True, False),
    # elements behind the turned ones, copied or left alone
    (599, 7, 2, 72, [11, 13, 8], True, False),
    (605, 4, 3, 72, [32], False, True),
    (613, 2, 1, 72, [10, 22], False, False),
    (597, 9, 1, 256, [4, 4], True, True),
    (1191, 1, 2, 40, [8, 8], False, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hk,d,sections,mixed,inter", MANY)
def test_rotary_of_many_tokens(T, hq, hk, d, sections, mixed, inter):
    if hk:
        test_rotary(T, hq, hk, d, sections, mixed, inter)
    from w4a8_b200 import kvcache
    dev = _dev()
    g = torch.Generator().manual_seed(T)
    axes = kvcache.RotaryAxes(sections, mixed=mixed)
    table = kvcache.rotary_table(2 * axes.pairs, 33, base=1e4, device="cpu")
    pos = torch.randint(-3, 40, (axes.axes, T), generator=g, dtype=torch.int32)
    # in rows longer than the heads, into others: what lies beside both stays
    x = torch.randn(T, hq * d + 8, generator=g).to(BF).to(dev)
    out = torch.full((T + 2, hq * d + 24), 7.0, dtype=BF, device=dev)
    q = x[:, 8:].unflatten(1, (hq, d))
    want = turn32(q.float().cpu(), pos, axes.axis_of_pair(), table, inter).to(BF)
    view = out[1:T + 1, 8:hq * d + 8].unflatten(1, (hq, d))
    kvcache.rotary(q, None, table.to(dev), pos.to(dev), axes, interleaved=inter, q_out=view)
    assert torch.equal(view.cpu(), want)
    assert (out[[0, -1]] == 7).all() and (out[:, :8] == 7).all() and (out[:, hq * d + 8:] == 7).all()
    before = x[:, :8].clone()
    kvcache.rotary(q, None, table.to(dev), pos.to(dev), axes, interleaved=inter, q_out=q)
    assert torch.equal(q.cpu(), want) and torch.equal(x[:, :8], before)
