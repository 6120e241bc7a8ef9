"""The paged 8-bit cache on the GPU against tests/kv8_oracle.py: what enters it bit for bit, attention against 64 bits."""
import math
import random

import pytest
import torch

from tests import kv8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def K():
    from spec_mcts_amd import kernels
    return kernels


class World:
    """A cache on the GPU and the same sequences in the oracle"""

    def __init__(self, B, H, Hkv, max_len, seed, spare=3, places=None, scale=1.0):
        self.g = torch.Generator().manual_seed(seed)
        self.B, self.H, self.Hkv = B, H, Hkv
        self.cols = (max_len + 63) // 64
        n = B * self.cols + spare
        self.cache = K().kv8_cache(B, max_len, Hkv, DEV, n_pages=n)
        order = torch.randperm(n, generator=self.g)[:B * self.cols].view(B, self.cols).to(torch.int32)
        self.cache.pages.copy_(order)
        self.cache.open_k.fill_(math.nan)                       # what no row was written to may hold anything
        self.cache.open_v.fill_(math.nan)
        self.cache.scales.fill_(math.nan)
        self.cos, self.sin = O.tables(places or max_len + 64)
        self.cos_d, self.sin_d = self.cos.to(DEV), self.sin.to(DEV)
        self.seqs = [O.Sequence(Hkv) for _ in range(B)]
        self.lens = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.scale = scale

    def old(self):
        return [s.k.shape[0] for s in self.seqs]

    def rows(self, T):
        r = lambda h, s: (torch.randn((T, h, 128), generator=self.g) * s).half()
        return r(self.H, 1.5), r(self.Hkv, 1.5 * self.scale), r(self.Hkv, self.scale)

    def step(self, new, qkv=None, behind=0, advance=True, max_new=None, single=False, packed=False):
        """`new` rows for each sequence; (q rotated on the GPU, q rotated by the oracle, cu)"""
        T = sum(new) + behind
        q, k, v = qkv or self.rows(T)
        cu = None if single else torch.tensor([sum(new[:b]) for b in range(self.B + 1)], dtype=torch.int32, device=DEV)
        if packed:
            p = torch.cat([x.reshape(T, -1) for x in (q, k, v)], 1).to(DEV)
            a, b = self.H * 128, (self.H + self.Hkv) * 128
            args = p[:, :a].view(T, self.H, 128), p[:, a:b].view(T, self.Hkv, 128), p[:, b:].view(T, self.Hkv, 128)
        else:
            args = q.to(DEV), k.to(DEV), v.to(DEV)
        out = torch.full((T, self.H, 128), 7.0, dtype=torch.float16, device=DEV)
        got = K().kv8_append(*args, self.cos_d, self.sin_d, self.cache, self.lens, cu=cu, max_new=1 if single else max_new or max(max(new), 1), out=out)
        assert got is out
        want = torch.full((T, self.H, 128), 7.0, dtype=torch.float16)
        at = 0
        for s, n in zip(self.seqs, new):
            place = torch.arange(s.k.shape[0], s.k.shape[0] + n).clamp(max=self.cos.shape[0] - 1)
            want[at:at + n] = O.rotate(q[at:at + n], self.cos, self.sin, place)
            s.add(O.rotate(k[at:at + n], self.cos, self.sin, place), v[at:at + n])
            at += n
        self.before = self.lens.clone()
        if advance:
            self.lens += torch.tensor(new, dtype=torch.int32, device=DEV)
        return got, want, cu

    def check_cache(self):
        """codes and scales of whole blocks and the rows of open ones, bit for bit"""
        c = [t.cpu() for t in self.cache]
        for b, s in enumerate(self.seqs):
            n = s.k.shape[0]
            for j in range(min(n // 64, self.cols)):
                page = int(c[5][b, j])
                codes, scales = s.block(j)
                assert torch.equal(c[0][page], codes[0]), (b, j)
                assert torch.equal(c[1][page], codes[1].transpose(1, 2)[..., torch.argsort(torch.tensor(O.PLACE))]), (b, j)
                assert torch.equal(c[2][page], torch.stack(scales, -1)), (b, j)
            left = n % 64
            assert torch.equal(c[3][b, :, :left], s.k[n - left:].transpose(0, 1)), b
            assert torch.equal(c[4][b][..., O.PLACE[:left]], s.v[n - left:].permute(1, 2, 0)), b

    def check_attn(self, q, new, cu, **kw):
        """q: as kv8_append returned it, behind the step that brought `new`"""
        window, sinks = kw.get("window", 0), kw.get("sinks", 0)
        out = torch.full(q.shape, 9.0, dtype=torch.float16, device=DEV)
        got = K().kv8_attn(q, self.cache, self.before, cu=cu, max_new=max(max(new), 1), out=out, **kw)
        assert got is out
        got, q = got.cpu().double(), q.cpu()
        at = 0
        for b, (s, n) in enumerate(zip(self.seqs, new)):
            k, v = s.held()
            old = k.shape[0] - n
            o, mean = O.attention(q[at:at + n], k, v, old, window, sinks)
            bound = O.attention_bound(o, mean, k.shape[0], float(v.abs().max()) if v.numel() else 0.0)
            off = (got[at:at + n] - o).abs()
            assert bool((off <= bound).all()), (b, old, n, float((off / bound).max()))
            at += n
        assert bool((got[at:] == 9.0).all())                    # rows behind the last sequence


# ---- what enters the cache -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,H,Hkv", [(1, 1, 1), (3, 4, 4), (2, 8, 1), (5, 12, 4), (2, 40, 2)])
def test_single_tokens_across_blocks(B, H, Hkv):
    """one row at a time from an empty cache past two borders of a block"""
    w = World(B, H, Hkv, 200, seed=B * 100 + H)
    for i in range(131):
        got, want, _ = w.step([1] * B, single=i % 2 == 0, packed=i % 3 == 0)
        assert torch.equal(got.cpu(), want), i
        if i in (0, 62, 63, 64, 130):
            w.check_cache()


@pytest.mark.parametrize("steps", [[[1, 2, 3]], [[63, 64, 65], [1, 1, 1]], [[63, 1, 62], [2, 0, 5], [0, 0, 0], [130, 64, 1]], [[200, 7, 0], [57, 121, 300], [1, 1, 1], [63, 64, 65]],
                                   [[127, 128, 129], [129, 128, 127], [65, 64, 63]], [[1, 0, 500]]], ids=str)
def test_ragged_packs(steps):
    w = World(3, 6, 2, 700, seed=len(steps))
    for i, new in enumerate(steps):
        got, want, _ = w.step(new, behind=i, packed=i % 2 == 1)
        assert torch.equal(got.cpu(), want), i                  # (the rows behind the last sequence among them)
        w.check_cache()


def test_what_it_holds_does_not_depend_on_the_calls():
    """the same 300 rows in one call, in chunks and row by row: the same bytes"""
    rng = random.Random(3)
    seen = []
    for way in ("one", "chunks", "rows"):
        w = World(2, 4, 2, 320, seed=11)
        q, k, v = w.rows(600)
        at = 0
        while at < 300:
            n = 300 if way == "one" else 1 if way == "rows" else min(rng.randint(1, 140), 300 - at)
            pick = torch.cat((torch.arange(at, at + n), torch.arange(300 + at, 300 + at + n)))
            w.step([n, n], qkv=(q[pick], k[pick], v[pick]))
            at += n
        w.check_cache()
        seen.append([t[w.cache.pages.long()].cpu()[:, :4] for t in w.cache[:3]])
    assert all(torch.equal(a, b) for other in seen[1:] for a, b in zip(seen[0], other))


def test_bad_pages_and_lengths_write_nothing():
    """a block without a page, past the table or past the capacity is not written, and nothing else is touched"""
    w = World(4, 2, 2, 128, seed=5)
    n_pages = w.cache.codes_k.shape[0]
    w.cache.pages[0, 0] = -1
    w.cache.pages[1, 0] = n_pages
    w.cache.pages[1, 1] = 2 ** 31 - 1
    before = [t.clone() for t in w.cache]
    lens = torch.tensor([0, 0, 128, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    T = 4 * 130
    q, k, v = (x.to(DEV) for x in w.rows(T))
    cu = torch.arange(0, T + 1, 130, dtype=torch.int32, device=DEV)
    K().kv8_append(q, k, v, w.cos_d, w.sin_d, w.cache, lens, cu=cu, max_new=130)
    kept = {int(w.cache.pages[0, 1])}                           # the one block that has a page and a place
    for t, old in zip(w.cache[:3], before[:3]):
        changed = {p for p in range(n_pages) if not torch.equal(t[p].cpu().view(torch.uint8), old[p].cpu().view(torch.uint8))}
        assert changed <= kept
    assert int((w.cache.scales[list(kept)] > 0).sum()) == 4
    for t, old in zip(w.cache[3:5], before[3:5]):
        assert torch.equal(t[2:].view(torch.int16), old[2:].view(torch.int16))      # sequences whose rows end past the capacity


def test_numbers_past_the_tensors_are_cut():
    """cu past the pack or going down, negative lengths, max_new below what cu says"""
    w = World(3, 2, 1, 64, seed=6)
    q, k, v = (x.to(DEV) for x in w.rows(10))
    for cu, lens in (([0, 4, 99, 100], [0, 0, 0]), ([0, 8, 3, 10], [0, -5, 0]), ([-7, 2, 4, 9], [-1, 0, 3])):
        out = torch.full_like(q, 7.0)
        K().kv8_append(q, k, v, w.cos_d, w.sin_d, w.cache, torch.tensor(lens, dtype=torch.int32, device=DEV), cu=torch.tensor(cu, dtype=torch.int32, device=DEV), max_new=3, out=out)
        o = K().kv8_attn(out, w.cache, torch.tensor(lens, dtype=torch.int32, device=DEV), cu=torch.tensor(cu, dtype=torch.int32, device=DEV), max_new=3)
        a = min(max(cu[0], 0), 10)
        assert torch.equal(out[a:a + 2].cpu(), O.rotate(q[a:a + 2].cpu(), w.cos, w.sin, torch.arange(2) + max(lens[0], 0)))
        assert torch.isfinite(o[a:a + 2]).all()


def test_places_past_the_tables_take_the_last_row():
    w = World(2, 2, 2, 256, seed=7, places=70)
    got, want, _ = w.step([100, 69])
    assert torch.equal(got.cpu(), want)
    got, want, _ = w.step([1, 1], single=True)
    assert torch.equal(got.cpu(), want)
    w.check_cache()


def test_zeros_and_extremes():
    """blocks of zeros have a scale of 0; the largest and the least fp16 values keep their block's codes in 1 .. 255"""
    w = World(2, 2, 2, 128, seed=8)
    q, k, v = w.rows(256)
    k[:64], v[:64] = 0, 0
    v[64:128] = 65504.0
    k[128:192] = 2.0 ** -24
    v[128:192] *= 2.0 ** -20
    w.step([128, 128], qkv=(q, k, v))
    w.check_cache()
    assert int(w.cache.codes_k[w.cache.pages.long()].min()) >= 1
    rows = K().kv8_rows(w.cache, w.lens, torch.zeros_like(w.lens), 128)
    assert bool((rows[0][0, :64] == 0).all()) and bool((rows[1][0, 64:128] == 65504.0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_stays_in_its_block_and_head(bad):
    w = World(1, 2, 2, 256, seed=9)
    q, k, v = w.rows(200)
    v[70, 0, 5] = bad
    k2 = k.clone()
    w.step([200], qkv=(q, k2, v), advance=True)
    rows_k, rows_v = K().kv8_rows(w.cache, w.lens, torch.zeros_like(w.lens), 200)
    assert bool(torch.isfinite(rows_k).all())
    fine = torch.ones((200, 2), dtype=torch.bool)
    fine[64:128, 0] = False
    assert torch.equal(torch.isfinite(rows_v[0]).all(-1).cpu(), fine) and bool(torch.isnan(rows_v[0, 64:128, 0]).all())
    # attention: head 1 and the queries in front of the block are as they were
    cu = torch.tensor([0, 200], dtype=torch.int32, device=DEV)
    o = K().kv8_attn(q.to(DEV), w.cache, w.before, cu=cu, max_new=200)[:, :, :].cpu()
    assert bool(torch.isfinite(o[:, 1]).all()) and bool(torch.isfinite(o[:64, 0]).all()) and bool(torch.isnan(o[64:, 0]).all())


@pytest.mark.parametrize("first,count", [([0, 0, 0], 1), ([0, 63, 64], 66), ([5, 130, 199], 130), ([0, 0, 0], 300), ([1000, -4, 150], 64), ([0, 1, 2], 0)], ids=str)
def test_rows_come_back(first, count):
    w = World(3, 2, 2, 256, seed=10)
    w.step([200, 131, 64])
    f = torch.tensor(first, dtype=torch.int32, device=DEV)
    k, v = K().kv8_rows(w.cache, w.lens, f, count)
    assert k.shape == v.shape == (3, count, 2, 128)
    for b, s in enumerate(w.seqs):
        for got, x in zip((k, v), s.held()):
            want = torch.zeros((count, 2, 128), dtype=torch.float64)
            a = max(first[b], 0)
            part = x[a:a + count]
            want[:part.shape[0]] = part
            assert torch.equal(got[b].cpu(), want.float().half()), b      # (a code times its scale: fp32 rounds once before fp16)


# ---- attention -------------------------------------------------------------------------------------------------------------------
SIGHTS = [(0, 0), (1, 0), (5, 3), (64, 0), (64, 64), (100, 4), (200, 130), (4096, 4), (37, 4096)]


@pytest.mark.parametrize("window,sinks", SIGHTS, ids=str)
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (8, 1), (6, 2), (32, 2)])
def test_one_query(H, Hkv, window, sinks):
    """one token for sequences of length 0 to 1000, no two alike"""
    old = [0, 1, 62, 63, 64, 65, 127, 300, 511, 999]
    w = World(len(old), H, Hkv, 1024, seed=H * 1000 + window + sinks)
    w.step(old)
    q, _, cu = w.step([1] * len(old), single=True)
    w.check_attn(q, [1] * len(old), cu, window=window, sinks=sinks)
    w.check_attn(q, [1] * len(old), cu, window=window, sinks=sinks, max_len=1000)


@pytest.mark.parametrize("window,sinks", SIGHTS, ids=str)
@pytest.mark.parametrize("H,Hkv,new", [(4, 4, [3, 0, 7, 5]), (8, 1, [2, 1, 2, 0]), (8, 1, [4, 3, 4, 1]), (8, 1, [6, 5, 0, 6]), (8, 1, [8, 8, 1, 3]), (6, 2, [17, 21, 2, 9])])
def test_a_few_queries(H, Hkv, new, window, sinks):
    """all tile counts of the kernel for up to 64 queries a head"""
    w = World(4, H, Hkv, 1024, seed=H + sum(new) + window)
    w.step([500, 61, 0, 190])
    q, _, cu = w.step(new, behind=2)
    w.check_attn(q, new, cu, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", SIGHTS, ids=str)
@pytest.mark.parametrize("H,Hkv,old,new", [(2, 2, [0, 0], [130, 65]), (8, 1, [64, 333], [40, 9]), (6, 2, [700, 5], [100, 250]), (4, 4, [1, 0], [0, 300]), (16, 1, [100, 640], [64, 63])])
def test_many_queries(H, Hkv, old, new, window, sinks):
    w = World(2, H, Hkv, 1024, seed=H + sum(new) + window)
    w.step(old)
    q, _, cu = w.step(new, behind=3)
    w.check_attn(q, new, cu, window=window, sinks=sinks)
    w.check_attn(q, new, cu, window=window, sinks=sinks, max_len=sum(new) + max(old))


@pytest.mark.parametrize("max_len", [1, 64, 5000, 10 ** 6])
@pytest.mark.parametrize("new", [[1], [30], [200]])
def test_every_split_of_a_long_sequence(max_len, new):
    """max_len decides the split alone: also one that is too small gives the same attention"""
    w = World(1, 2, 1, 5000, seed=len(new) + max_len)
    w.step([4700])
    q, _, cu = w.step(new)
    w.check_attn(q, new, cu, max_len=max_len)
    w.check_attn(q, new, cu, max_len=max_len, window=1500, sinks=70)


@pytest.mark.parametrize("scale", [2.0 ** -12, 2.0 ** -6, 64.0])
def test_small_and_large_values(scale):
    """V of all sizes next to an open block: scales meet in fp32"""
    w = World(2, 4, 2, 512, seed=21, scale=scale)
    if scale > 1:
        q, k, v = w.rows(400)
        w.step([200, 200], qkv=(q, k / 64, v))                 # (scores stay below 64)
        q, k, v = w.rows(2)
        q, _, cu = w.step([1, 1], qkv=(q, k / 64, v))
    else:
        w.step([200, 200])
        q, _, cu = w.step([1, 1])
    w.check_attn(q, [1, 1], cu)


def test_steep_scores():
    """a maximum that grows block by block, and one that stands in the first row"""
    for order in (1, -1):
        w = World(1, 2, 1, 1024, seed=22)
        q, k, v = w.rows(701)
        q[:] = 0
        q[..., 0] = 1.0
        k[:] = 0
        k[:, :, 0] = (200 + order * torch.linspace(-200, 200, 701))[:, None].half()
        w.cos_d.fill_(1), w.sin_d.fill_(0)
        w.cos.fill_(1), w.sin.fill_(0)
        w.step([700], qkv=(q[:700], k[:700], v[:700]))
        got, _, cu = w.step([1], qkv=(q[700:], k[700:], v[700:]))
        w.check_attn(got, [1], cu)


def test_pages_out_of_range_are_read_as_the_nearest():
    w = World(2, 2, 2, 256, seed=23)
    w.step([256, 256])
    w.cache.scales.nan_to_num_(0.01)
    w.cache.pages[0, 1] = -9
    w.cache.pages[1, 2] = 10 ** 6
    q, _, _ = w.rows(2)
    w.before = w.lens - 1
    ref = w.cache.pages.clamp(0, w.cache.codes_k.shape[0] - 1)
    got = K().kv8_attn(q.to(DEV), w.cache, w.before, max_len=256)
    assert torch.equal(got, K().kv8_attn(q.to(DEV), w.cache._replace(pages=ref), w.before, max_len=256))


def test_tables_wider_than_the_batch_and_strided_queries():
    """a slice of a wider page table, a smaller batch than the cache's, queries out of a packed product"""
    w = World(4, 4, 2, 512, seed=24)
    w.step([300, 10, 64, 200])
    wide = torch.full((4, w.cols + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + w.cols] = w.cache.pages
    q, _, cu = w.step([1, 1, 1, 1], packed=True)
    packed = torch.randn((4, 8, 128), device=DEV).half()
    packed[:, 4:] = q
    one = K().kv8_attn(q, w.cache, w.before)
    part = K().kv8_attn(packed[:2, 4:], w.cache._replace(pages=wide[:, 2:2 + w.cols]), w.before[:2])
    assert torch.equal(part, one[:2])
    assert K().kv8_attn(q[:0], w.cache, w.before[:0]).shape == (0, 4, 128)
    w.check_attn(q, [1] * 4, cu)


def test_outputs_over_the_queries():
    """q rotated and the attention in place of the queries"""
    for new, max_len in (([1, 1], 512), ([1, 1], 64), ([9, 3], 512), ([150, 40], 512)):
        w = World(2, 8, 2, 512, seed=29)
        w.step([200, 77])
        q, k, v = w.rows(sum(new))
        ref, _, cu = w.step(new, qkv=(q, k, v), advance=False)
        mine = q.to(DEV)
        K().kv8_append(mine, k.to(DEV), v.to(DEV), w.cos_d, w.sin_d, w.cache, w.before, cu=cu, max_new=max(new), out=mine)
        assert torch.equal(mine, ref)
        want = K().kv8_attn(ref, w.cache, w.before, cu=cu, max_new=max(new), max_len=max_len)
        assert torch.equal(K().kv8_attn(mine, w.cache, w.before, cu=cu, max_new=max(new), max_len=max_len, out=mine), want)


def test_a_nan_query_has_a_nan_output():
    w = World(1, 2, 1, 4096, seed=25)
    w.step([3000])
    q, _, cu = w.step([1])
    q[0, 1] = math.nan
    for max_len in (64, 4096):
        o = K().kv8_attn(q, w.cache, w.before, max_len=max_len).cpu()
        assert bool(torch.isnan(o[0, 1]).all()) and bool(torch.isfinite(o[0, 0]).all())


def test_captured_steps():
    """one graph of append, attention and the step of the lengths, replayed over a border of a block with eager work between, against eager steps"""
    worlds = [World(3, 4, 2, 512, seed=26) for _ in range(2)]
    for w in worlds:
        w.step([60, 126, 300])
    rows = [worlds[0].rows(3) for _ in range(6)]
    eager, graphed = worlds
    want = []
    for r in rows:
        q, _, cu = eager.step([1, 1, 1], qkv=r, single=True)
        want.append(K().kv8_attn(q, eager.cache, eager.before, max_len=512).clone())
    q, k, v = (x.to(DEV) for x in rows[0])
    lens, one = graphed.lens, torch.ones(3, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                               # warm up
        K().kv8_attn(K().kv8_append(q, k, v, graphed.cos_d, graphed.sin_d, graphed.cache, lens), graphed.cache, lens, max_len=512)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotated = K().kv8_append(q, k, v, graphed.cos_d, graphed.sin_d, graphed.cache, lens)
        out = K().kv8_attn(rotated, graphed.cache, lens, max_len=512)
        lens += one
    for r, o in zip(rows, want):
        for t, x in zip((q, k, v), r):
            t.copy_(x)
        graph.replay()
        assert torch.equal(out, o)
        torch.randn((64, 64), device=DEV).sum()
        torch.cuda.synchronize()
    for a, b in zip(eager.cache[:3], graphed.cache[:3]):
        assert torch.equal(a[eager.cache.pages[:, 0].long()], b[graphed.cache.pages[:, 0].long()])


def test_two_streams_at_once():
    """attention over one cache from two streams, split and merged: each call has its own workspace"""
    w = World(1, 2, 1, 8192, seed=27)
    w.step([8000])
    q, _, cu = w.step([1])
    other = q.flip(1).contiguous()
    want = [K().kv8_attn(x, w.cache, w.before, max_len=8192) for x in (q, other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, x in enumerate((q, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(K().kv8_attn(x, w.cache, w.before, max_len=8192))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_offsets_past_32_bits():
    """pages whose codes lie more than 4 GiB into the pool"""
    Hkv, n_pages = 8, 70000                                     # 70000 x 8 x 8 KiB = 4.6 GB a side
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    c = K().kv8_cache(1, 256, Hkv, DEV, n_pages=n_pages)
    w = World(1, 8, Hkv, 256, seed=28)
    w.cache = c
    c.pages.copy_(torch.tensor([[69999, 3, 69000, 65536]], dtype=torch.int32))
    w.step([250])
    q, _, cu = w.step([1])
    w.check_cache()
    w.check_attn(q, [1], cu)
    k, _ = K().kv8_rows(c, w.lens, torch.zeros_like(w.lens), 251)
    assert torch.equal(k[0].cpu(), w.seqs[0].held()[0].float().half())


# ---- past the capacity -----------------------------------------------------------------------------------------------------------
PAST = [(0, 192), (0, 255), (70, 193), (127, 192), (128, 200), (128, 255), (150, 192), (188, 193), (190, 254), (191, 192), (191, 255), (195, 230), (0, 256), (70, 300), (140, 256), (191, 400), (300, 310)]


@pytest.mark.parametrize("old,total", PAST, ids=str)
def test_a_call_past_the_capacity_keeps_the_rows_in_front_of_it(old, total):
    """a cache of 128 + 63 rows, from `old` rows to `total` in one call and row by row: the same rows, and the attention of the call over them; from 256 on they are those of the table's
    blocks"""
    cap = 191 if total < 256 else 128
    ways = []
    for one in (True, False):
        w = World(1, 4, 2, 128, seed=51)
        w.cos, w.sin = O.tables(512)
        w.cos_d, w.sin_d = w.cos.to(DEV), w.sin.to(DEV)
        q, k, v = w.rows(total)
        qkv = lambda a, b: (q[a:b], k[a:b], v[a:b])             # noqa: E731
        for i in range(old):
            w.step([1], qkv=qkv(i, i + 1), single=True)
        if one:
            rotated, _, cu = w.step([total - old], qkv=qkv(old, total))
            out = K().kv8_attn(rotated, w.cache, w.before, cu=cu, max_new=total - old)
        else:
            for i in range(old, total):
                w.step([1], qkv=qkv(i, i + 1), single=True)
        ways.append((w, K().kv8_rows(w.cache, w.lens, torch.zeros_like(w.lens), total + 70)))
    w, rows = ways[0]
    assert all(torch.equal(a, b) for a, b in zip(rows, ways[1][1]))
    s = w.seqs[0]
    s.k, s.v = s.k[:cap], s.v[:cap]
    held = s.held()
    for got, x in zip(rows, held):
        assert torch.equal(got[0, :min(cap, total)].cpu(), x.float().half()) and bool((got[0, cap:] == 0).all())
    for a, b in zip(w.cache[:3], ways[1][0].cache[:3]):
        assert torch.equal(a[w.cache.pages.long()], b[w.cache.pages.long()])
    o, mean = O.attention(rotated.cpu(), *held, old)
    bound = O.attention_bound(o, mean, cap, float(held[1].abs().max()))
    assert bool(((out.cpu().double() - o).abs() <= bound).all())


def test_drafted_tokens_at_the_end():
    """five drafted tokens of which three have room and are accepted: the next step sees them"""
    w = World(2, 8, 2, 128, seed=52, places=300)
    w.step([188, 40])
    q, k, v = w.rows(10)
    w.step([5, 5], qkv=(q, k, v), advance=False)
    w.lens += 3
    for s in w.seqs:
        s.k, s.v = s.k[:-2], s.v[:-2]
    rows = K().kv8_rows(w.cache, w.lens, torch.zeros_like(w.lens), 191)
    for b, s in enumerate(w.seqs):
        for got, x in zip(rows, s.held()):
            assert torch.equal(got[b, :x.shape[0]].cpu(), x.float().half())


@pytest.mark.parametrize("window,sinks,sees", [(62, 0, False), (63, 0, False), (64, 0, True), (63, 128, False), (63, 129, True)])
def test_a_query_past_the_capacity_sees_what_its_window_shows(window, sinks, sees):
    """rows 128 .. 190 of a cache of 191, the last of them not finite, and a query at place 253: a window of 63 ends behind them"""
    w = World(1, 2, 1, 128, seed=53, places=300)
    q, k, v = w.rows(254)
    v[190] = math.nan
    w.step([253], qkv=(q[:253], k[:253], v[:253]))
    rotated, _, _ = w.step([1], qkv=(q[253:], k[253:], v[253:]), single=True)
    o = K().kv8_attn(rotated, w.cache, w.before, window=window, sinks=sinks).cpu()
    assert bool(torch.isnan(o).all()) if sees else bool(torch.isfinite(o).all())
    if sinks == 0 and not sees:
        assert bool((o == 0).all())                             # nothing in sight


# ---- blocks whose V differs in size ----------------------------------------------------------------------------------------------
def scale_world(order, low, rows, H, Hkv, seed):
    """`rows` rows whose blocks hold V of about 1000 or of 2^low, with one strong row in the first of the large blocks: all others have 2^-11 of its weight, and about as
    much together.  The tables do not rotate, the scores are the first value's"""
    w = World(1, H, Hkv, rows + 512, seed=seed)
    w.cos_d.fill_(1), w.sin_d.fill_(0)
    w.cos.fill_(1), w.sin.fill_(0)
    blocks = (rows + 63) // 64
    large = {"first": [0], "last": [rows // 64 - 1], "middle": [blocks // 2], "turns": range(0, blocks, 2), "zeros": [1]}[order]
    q, k, v = w.rows(rows)
    q[:], k[:] = 0, 0
    q[..., 0] = 1.0
    k[64 * large[0] + 7, :, 0] = 86.25                          # 86.25 / sqrt(128) = 11 ln 2
    v = (v.float().abs() * 0.25 + 0.5).half()                   # (one sign: a lost row moves the mean)
    for j in range(blocks):
        at = slice(j * 64, j * 64 + 64)
        v[at] = v[at] * 1000 if j in large else (v[at].float() * 2.0 ** low).half()
        if order == "zeros" and j % 3 == 2:
            v[at] = 0
    w.step([rows], qkv=(q, k, v))
    return w


def check_by_scales(w, q, new, cu, **kw):
    """As check_attn, with the rounding of the weights counted in the sum that they are divided by too: sum p d (v - o) with |v - o| <= |v| + |o| and |o| below the mean of |v|"""
    got = K().kv8_attn(q, w.cache, w.before, cu=cu, max_new=max(max(new), 1), **kw).cpu().double()
    at = 0
    for b, (s, n) in enumerate(zip(w.seqs, new)):
        k, v = s.held()
        o, mean = O.attention(q[at:at + n].cpu(), k, v, k.shape[0] - n, kw.get("window", 0), kw.get("sinks", 0))
        bound = O.attention_bound(o, mean, k.shape[0], float(v.abs().max())) + 2.0 ** -11 * mean
        off = (got[at:at + n] - o).abs()
        assert bool((off <= bound).all()), (b, k.shape[0], kw, float((off / bound).max()))
        at += n


@pytest.mark.parametrize("order", ["first", "last", "middle", "turns", "zeros"])
@pytest.mark.parametrize("low", [4, -2, -8, -14, -20, -24])
@pytest.mark.parametrize("new", [1, 9, 150])
def test_a_block_s_v_does_not_change_what_its_rows_weigh(order, low, new):
    """large and small V block by block, for few and many queries, in one part and in several"""
    w = scale_world(order, low, 2500, 4, 2, seed=40 + new)
    q, k, v = w.rows(new)
    q[:], k[:] = 0, 0
    q[..., 0] = 1.0
    q, _, cu = w.step([new], qkv=(q, k, (v.float() * 2.0 ** low).half()))
    for kw in (dict(max_len=64), dict(max_len=10 ** 6), dict(window=2000, sinks=100), dict(window=2300, max_len=64)):
        check_by_scales(w, q, [new], cu, **kw)


@pytest.mark.parametrize("new", [[1, 1], [12, 3], [200, 90]], ids=str)
def test_v_of_any_size_from_block_to_block(new):
    """random scores over blocks whose V goes from 2^-20 to 2^6, between heads and sequences too"""
    w = World(2, 6, 2, 2400, seed=43)
    q, k, v = w.rows(1900 + 801)
    size = 2.0 ** torch.randint(-20, 7, ((1900 + 801) // 64 + 1, 2), generator=w.g).repeat_interleave(64, 0)[:1900 + 801]
    w.step([1900, 801], qkv=(q, k, (v.float() * size[..., None]).half()))
    q, _, cu = w.step(new)
    for kw in (dict(max_len=64), dict(), dict(max_len=10 ** 6, window=700, sinks=64), dict(max_len=64, window=64)):
        check_by_scales(w, q, new, cu, **kw)


def test_rows_that_are_not_seen_do_not_set_the_unit():
    """small values in the window behind large ones that it has passed, and in front of large ones that are yet to come"""
    w = scale_world("middle", -20, 2500, 8, 1, seed=44)
    q, k, v = w.rows(130)
    q[:], k[:] = 0, 0
    q[..., 0] = 1.0
    v = v.float() * 2.0 ** -20
    v[70:] *= 2.0 ** 28
    q, _, cu = w.step([130], qkv=(q, k, v.half()))
    for max_len in (64, 10 ** 6):
        check_by_scales(w, q, [130], cu, max_len=max_len, window=300)
