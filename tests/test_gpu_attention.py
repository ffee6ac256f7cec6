"""Attention over the paged 8-bit cache against a 64-bit plain implementation.

Bound, element by element: the output is rounded once to bf16 (at most 2^-8 of
it), weights are rounded to fp16 (at most 2^-11 each, so 2^-11 of sum p |v|),
and as much again covers the fp32 arithmetic before it:

    |o - ref| <= 2^-8 |ref| + 2^-10 (sum_j p_j |v_j| + n 2^-28 vmax)

The last term is fp16's range: a weight enters as p vs / vr 2^14 with vr < 2 max vs,
so one below fp16's normal numbers is off by up to 2^-25, which is 2^-38 max vs
for each of the n visible tokens (vmax = 128 max vs).  It shows only where every
heavier token's code is 0.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from decoder_ref import attention64, bf16_np  # noqa: E402

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


class Case:
    """A batch with random codes in shuffled pages."""

    def __init__(self, hq, hkv, d, page, qs, lens, seed=0, spread=1.0, spare=2):
        dev = _dev()
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.page, self.qs, self.lens = hq, hkv, d, page, list(qs), list(lens)
        npages = [-(-n // page) for n in lens]
        self.P = sum(npages) + spare
        order = torch.randperm(self.P, generator=g).tolist()
        wide = max(npages + [1])
        self.table, at = [], 0
        for n in npages:
            self.table.append(order[at:at + n] + [-1] * (wide - n))
            at += n
        self.codes = [torch.randint(-127, 128, (self.P, hkv, page, d), generator=g, dtype=torch.int8) for _ in range(2)]
        self.scales = [(torch.randn(self.P, hkv, generator=g) * 0.7 * sp).exp() * m / 127
                       for sp, m in ((1.0, 2.6), (spread, 2.0))]
        self.cu = [0]
        for n in qs:
            self.cu.append(self.cu[-1] + n)
        self.T = self.cu[-1]
        self.q = torch.randn(self.T, hq, d, generator=g).to(torch.bfloat16)
        self.dev = dev

    def cache(self):
        from w4a8_b200 import kvcache
        t = [x.to(self.dev) for x in self.codes + self.scales]
        return kvcache.KVCache(*t)

    def batch(self):
        i = dict(dtype=torch.int32, device=self.dev)
        return (torch.tensor(self.table, **i), torch.tensor(self.lens, **i), torch.tensor(self.cu, **i))

    def run(self, cache=None, **kw):
        from w4a8_b200 import kvcache, ops
        o = kvcache.attention(self.q.to(self.dev), cache or self.cache(), *self.batch(), max(self.qs + [1]), **kw)
        assert ops.workspace_status(self.dev) == 0
        return o

    def ref(self, scale=None):
        return attention64(bf16_np(self.q), self.codes[0].numpy(), self.codes[1].numpy(), self.scales[0].numpy(),
                           self.scales[1].numpy(), self.table, self.lens, self.cu, scale or self.d ** -0.5)

    def check(self, out, scale=None):
        ref, mag = self.ref(scale)
        got = bf16_np(out)
        assert np.isfinite(got).all()
        over = np.abs(got - ref) - (2.0 ** -8 * np.abs(ref) + 2.0 ** -10 * mag)
        assert over.max() <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))


CASES = [
    # hq, hkv, d, page, query tokens, lengths
    (40, 8, 128, 16, [1], [1]),
    (40, 8, 128, 16, [1, 1, 1, 1], [15, 16, 17, 33]),
    (40, 8, 128, 16, [1], [1500]),
    (5, 1, 128, 32, [1, 1, 1], [700, 31, 65]),
    (8, 8, 64, 16, [1, 1], [100, 257]),                 # one query head per kv head
    (16, 2, 64, 64, [1, 1, 1], [5, 64, 129]),
    (7, 1, 128, 128, [1, 1], [300, 128]),
    (40, 1, 128, 16, [1, 1], [90, 400]),                # 40 heads on one kv head
    (5, 1, 128, 32, [5, 2, 3], [200, 77, 300]),         # drafted tokens
    (14, 7, 64, 16, [7], [50]),
    (4, 2, 128, 16, [9, 1, 20], [9, 80, 47]),           # a whole prompt, a token, a chunk
    (10, 2, 128, 16, [70], [70]),
    (10, 2, 128, 16, [33, 129], [300, 129]),
    (5, 1, 128, 64, [257], [511]),
    (8, 1, 64, 32, [300], [300]),
    (3, 3, 64, 16, [200, 1, 131], [333, 40, 131]),
    (6, 1, 128, 16, [64, 300, 1], [64, 1000, 17]),
    (5, 1, 128, 16, [1] * 30 + [40, 2, 0, 60], [100] * 30 + [90, 300, 5, 61]),   # single tokens beside two chunks
    (16, 2, 64, 32, [2, 1, 1, 50, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1],
     [33, 70, 64, 120] + [50] * 24),
]


@pytest.mark.parametrize("hq,hkv,d,page,qs,lens", CASES)
def test_against_64_bits(hq, hkv, d, page, qs, lens):
    c = Case(hq, hkv, d, page, qs, lens, seed=hq + page)
    c.check(c.run())


@pytest.mark.parametrize("qs,lens", [([1, 1, 1], [0, 40, 0]), ([0, 2, 0, 1], [10, 20, 0, 3]), ([5], [3]),
                                     ([80, 0], [50, 9]), ([1], [0])])
def test_rows_that_see_nothing_are_zero(qs, lens):
    """Length zero, sequences without tokens in the call, more query tokens than cached ones."""
    c = Case(10, 2, 128, 16, qs, lens, seed=3)
    out = c.run()
    c.check(out)
    for s, (n, L) in enumerate(zip(qs, lens)):
        for i in range(n):
            if L - n + i < 0:
                assert (out[c.cu[s] + i] == 0).all()


@pytest.mark.parametrize("qs", [[1], [40]])
def test_pages_that_are_not_there(qs):
    """Page ids outside the cache hold no tokens; what their memory would hold does not matter."""
    c = Case(8, 2, 128, 16, qs, [200], seed=4)
    c.table[0][3], c.table[0][7], c.table[0][12] = -1, c.P, 1 << 30
    c.check(c.run())


@pytest.mark.parametrize("qs", [[1], [3], [100]])
def test_masked_places_may_hold_anything(qs):
    """Infinite and NaN scales of pages behind the length and of pages that a row cannot see yet, codes of
    -128 past the length: rows that do not see them are not touched."""
    c = Case(5, 1, 128, 16, qs, [164], seed=5, spare=4)
    used = set(c.table[0][:11])
    free = [p for p in range(c.P) if p not in used]
    c.table[0] += [free[0], free[1]]                     # pages wholly behind the length
    for p, bad in ((free[0], float("nan")), (free[1], float("inf"))):
        c.scales[0][p], c.scales[1][p] = bad, bad
    last = c.table[0][10]
    for x in c.codes:
        x[last][:, 4:] = -128                            # rows past the length in the last page
    c.check(c.run())
    if qs == [100]:
        # the last page (tokens 160..163) becomes NaN: rows before token 160 stay as they were
        want, mag = c.ref()
        c.scales[0][last] = float("nan")
        c.scales[1][last] = float("nan")
        got = bf16_np(c.run())
        upto = 100 - 4
        assert np.isnan(got[upto:]).all()
        assert (np.abs(got[:upto] - want[:upto]) <= 2.0 ** -8 * np.abs(want[:upto]) + 2.0 ** -10 * mag[:upto]).all()


@pytest.mark.parametrize("qs,big", [([1], 1e4), ([50], 1e4), ([1], 1e-4), ([50], 1e-4), ([1], 1e30), ([50], 1e-30)])
def test_magnitudes(qs, big):
    """Queries far from 1 with the softmax scale that brings scores back, and values likewise."""
    c = Case(4, 1, 128, 16, qs, [150], seed=6)
    c.q = (c.q.float() * big).to(torch.bfloat16)
    c.scales[1] *= min(max(big, 1e-20), 1e20)
    scale = 128 ** -0.5 / big
    c.check(c.run(scale=scale), scale)


@pytest.mark.parametrize("qs", [[1], [60]])
def test_zero_pages_and_uneven_scales(qs):
    """Pages of zeros (scale 0), and value scales over six decades."""
    c = Case(4, 1, 128, 16, qs, [333], seed=7, spread=3.0)
    for x in c.scales:
        x[c.table[0][2]] = 0.0
    c.check(c.run())


@pytest.mark.parametrize("qs", [[1, 1], [30, 45]])
def test_one_score_outweighs_all(qs):
    """Scores that rise and fall by hundreds: the running maximum moves often."""
    c = Case(4, 1, 64, 16, qs, [300, 200], seed=8)
    c.q = (c.q.float() * 30).to(torch.bfloat16)
    ref, mag = c.ref()
    got = bf16_np(c.run())
    # scores up to about 400: fp32 sums of 64 products leave 64 * 2^-24 * 400 in the exponent
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -10 + 4e-3) * mag).all()


@pytest.mark.parametrize("qs,lens", [([1] * 5, [100, 900, 33, 1, 16]), ([120, 3], [400, 64])])
def test_strided_views_and_out(qs, lens):
    """q as a view of [q | k | v] rows, out as a view of wider rows: the same bits as dense tensors."""
    from w4a8_b200 import kvcache
    c = Case(10, 2, 128, 16, qs, lens, seed=9)
    cache, batch, mq = c.cache(), c.batch(), max(qs)
    dense = kvcache.attention(c.q.to(c.dev), cache, *batch, mq)
    wide = torch.full((c.T, 14 * 128 + 8), float("nan"), dtype=torch.bfloat16, device=c.dev)
    wide[:, :1280] = c.q.to(c.dev).view(c.T, 1280)
    o = torch.full((c.T, 12 * 128), float("nan"), dtype=torch.bfloat16, device=c.dev)
    ret = kvcache.attention(wide[:, :1280].unflatten(1, (10, 128)), cache, *batch, mq,
                            out=o[:, :1280].unflatten(1, (10, 128)))
    assert torch.equal(ret, dense)
    assert torch.isnan(o[:, 1280:]).all()
    # misaligned rows are copied, not refused
    odd = torch.empty(c.T * 1280 + 3, dtype=torch.bfloat16, device=c.dev)[3:].view(c.T, 10, 128)
    odd.copy_(c.q)
    assert torch.equal(kvcache.attention(odd, cache, *batch, mq), dense)


@pytest.mark.parametrize("qs,lens", [([1] * 7, [1000, 3, 500, 16, 77, 2000, 15]), ([5, 4], [700, 900]), ([200], [500])])
def test_repeats_streams_and_graphs(qs, lens):
    """The same bits on every run, on another stream, and from a captured graph after its lengths changed."""
    from w4a8_b200 import kvcache
    c = Case(5, 1, 128, 16, qs, lens, seed=10)
    cache, (table, kl, cu) = c.cache(), c.batch()
    q, mq = c.q.to(c.dev), max(qs)
    first = kvcache.attention(q, cache, table, kl, cu, mq)
    for _ in range(5):
        assert torch.equal(kvcache.attention(q, cache, table, kl, cu, mq), first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = kvcache.attention(q, cache, table, kl, cu, mq)
    side.synchronize()
    assert torch.equal(other, first)
    out = torch.empty_like(first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kvcache.attention(q, cache, table, kl, cu, mq, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    shorter = [max(n, L // 2) for n, L in zip(qs, lens)]
    kl.copy_(torch.tensor(shorter, dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    c.lens = shorter
    c.check(out)
    del g


@pytest.mark.parametrize("qs", [[1, 2], [90, 1]])
def test_cache_past_32_bits(qs):
    """Pages whose byte offset does not fit 32 bits."""
    from w4a8_b200 import kvcache
    dev = _dev()
    P, H, page, D = (1 << 31) // (8 * 16 * 128) + 40, 8, 16, 128
    cache = kvcache.KVCache.empty(P, H, page, D, dev)
    small = Case(40, 8, 128, 16, qs, [100, 250], seed=11)
    shift = P - small.P
    for dst, src in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), small.codes + small.scales):
        dst[shift:].copy_(src)
    table, kl, cu = small.batch()
    out = kvcache.attention(small.q.to(dev), cache, table + shift, kl, cu, max(qs))
    small.check(out)
    assert shift * H * page * D > 1 << 31


def test_many_sequences():
    """The largest batch, most of it short, some of it empty."""
    g = np.random.default_rng(0)
    lens = g.integers(0, 40, 2048).tolist()
    c = Case(2, 1, 64, 16, [1] * 2048, lens, seed=12)
    c.check(c.run())


def test_refusals():
    from w4a8_b200 import kvcache
    c = Case(4, 2, 64, 16, [1], [20], seed=13)
    cache, (table, kl, cu), q = c.cache(), c.batch(), c.q.to(c.dev)
    bad = [
        lambda: kvcache.attention(q.float(), cache, table, kl, cu, 1),
        lambda: kvcache.attention(q[:, :3], cache, table, kl, cu, 1),                  # 3 heads on 2 kv heads
        lambda: kvcache.attention(q.repeat(1, 1, 2), cache, table, kl, cu, 1),         # head_dim 128 on a cache of 64
        lambda: kvcache.attention(q, cache, table.long(), kl, cu, 1),
        lambda: kvcache.attention(q, cache, table, kl, cu[:1], 1),
        lambda: kvcache.attention(q, cache, table, kl.cpu(), cu, 1),
        lambda: kvcache.attention(q, cache, table, kl, cu, 0),
        lambda: kvcache.attention(q, cache, table, kl, cu, 1, out=torch.empty(1, 4, 128, device=c.dev)),
        lambda: kvcache.attention(q, cache, table, kl, cu, 1, scale=float("nan")),
        lambda: kvcache.attention(q, cache, table.repeat(2049, 1), kl.repeat(2049), cu[:1].repeat(2050), 1),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    assert kvcache.attention(q[:0], cache, table, kl, cu, 1).shape == (0, 4, 64)


@pytest.mark.parametrize("qs,over", [([1], 1), ([3], 2), ([20], 5), ([100], 40), ([2], 900)])
def test_lengths_past_the_table(qs, over):
    """Tokens past the table's last column are not there; the others stay at their positions."""
    c = Case(5, 1, 128, 16, qs, [160], seed=14)
    c.lens = [160 + over]
    c.check(c.run())
    if over >= qs[0]:                                    # every row sees all that is there, wherever it is itself
        first = c.run()
        c.lens = [2 ** 31 - 1]
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("qs,lens", [([1], [4000]), ([3, 2], [700, 900]), ([1] * 30 + [40, 2, 0, 60], [100] * 30 + [90, 300, 5, 61])])
def test_counters_left_by_a_spoiled_call(qs, lens):
    """Calls that overlapped on one workspace, against its rule, may leave counts of parts behind.  The calls
    after them are right: counts are kept in the byte of the call's number modulo 4, and each call clears the
    other bytes."""
    from w4a8_b200 import ops
    c = Case(5, 1, 128, 16, qs, lens, seed=17)
    cache = c.cache()
    first = c.run(cache)
    c.check(first)
    torch.cuda.synchronize()
    sms = torch.cuda.get_device_properties(c.dev).multi_processor_count
    buf = ops._WS[0]
    off = (ops.workspace(0, c.dev)[0] - buf.data_ptr()) // 4
    words = buf.view(torch.int32)[off:off + 256]
    for left in (0x01, 0x03, 0x90):
        calls = int(words[8].item())
        assert calls % sms == 0 and calls < 4 * sms
        lane = calls // sms                              # the next call's; the two before it hold what was left
        stale = sum((left << (8 * ((lane - k) % 4))) for k in (1, 2))
        stale = stale - (1 << 32) if stale >= 1 << 31 else stale
        words[16:16 + sms] = stale
        for _ in range(6):
            assert torch.equal(c.run(cache), first)


# one kv head and a long context: parts of tens of CTAs, shares of one unit and of several
LONG = [
    # hq, d, page, query tokens, lengths
    (5, 128, 16, [1], [4000]),
    (5, 128, 16, [1], [16000]),
    (8, 64, 32, [1], [16000]),
    (1, 64, 16, [1], [5003]),
    (5, 128, 32, [3], [4000]),
    (5, 128, 16, [3], [16000]),
    (5, 128, 64, [5, 2], [9000, 16000]),
    (4, 64, 16, [4], [12001]),
    (5, 128, 16, [1] * 7, [1000, 3, 500, 16, 77, 2000, 15]),
    (5, 128, 16, [5, 4], [700, 900]),
]


@pytest.mark.parametrize("hq,d,page,qs,lens", LONG)
def test_long_contexts_against_64_bits(hq, d, page, qs, lens):
    """Segments that many CTAs share: their join against 64 bits."""
    c = Case(hq, 1, d, page, qs, lens, seed=15 + d)
    c.check(c.run())


@pytest.mark.parametrize("hq,d,page,qs,lens", LONG[:8] + [(5, 128, 16, [40], [6000])])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_grow_along_the_context(hq, d, page, qs, lens, falling):
    """Scores whose deviation grows (or falls) twentyfold along the context: parts joined later outweigh earlier ones.

    Deviations up to about 15: the products of one score have magnitudes that sum to about 0.64 sqrt(D) 15 = 110, so
    their fp32 sum is off by D 2^-24 110 = 8.4e-4 at most, in numerator and denominator: 2e-3 of sum p |v| beside
    the bound above."""
    c = Case(hq, 1, d, page, qs, lens, seed=16 + d)
    for s, n in enumerate(lens):
        pages = -(-n // page)
        ramp = torch.linspace(0.5, 10.0, pages)
        c.scales[0][c.table[s][:pages], 0] = (ramp.flip(0) if falling else ramp) * 2.6 / 127
    ref, mag = c.ref()
    got = bf16_np(c.run())
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -10 + 2e-3) * mag).all()
