"""beam_select and beam_reorder on the GPU against 64 bits and indexing."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EOS = 2


def K():
    from spec_mcts_amd import kernels
    return kernels


def oracle(logits, scores, W, n, ended=None, eos=EOS):
    """On the CPU: scores in 64 bits, the n best of each group by (score down, beam, token)"""
    x, s = logits.double(), scores.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    x = x.clamp(max=65536.0)                                                 # (an infinite logit counts as that)
    s = torch.where(torch.isnan(s), torch.full_like(s, -math.inf), s)
    m = x.amax(1, keepdim=True)
    d = torch.where(x == m, torch.zeros_like(x), x - m)                      # (also where both are infinite)
    total = s[:, None] + d - torch.log(torch.exp(d).sum(1, keepdim=True))
    total[(x == -math.inf) | (s == -math.inf)[:, None]] = -math.inf
    if ended is not None:
        stay = torch.full_like(total, -math.inf)
        stay[:, eos] = s
        total = torch.where(ended.bool()[:, None], stay, total)
    G, V = logits.shape[0] // W, logits.shape[1]
    best, at = torch.sort(total.view(G, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    parent, token = at // V, at % V
    done = token == eos
    if ended is not None:
        done |= ended.view(G, W).bool().gather(1, parent)
    return best, parent, token, done


def check(logits, scores, W, n, ended=None, eos=EOS):
    """Whole numbers equal; scores to 2^-22 of the largest term (sums of fp32 exponentials: 2^-23 of the sum each, the result rounded once, 2^-24)"""
    got = K().beam_select(logits.to(DEV) if not logits.is_cuda else logits, scores.to(DEV), W, n, ended=None if ended is None else ended.to(DEV), eos=eos)
    best, parent, token, done = oracle(logits.cpu(), scores, W, n, ended, eos)
    assert torch.equal(got[1].cpu().long(), parent) and torch.equal(got[2].cpu(), token)
    assert torch.equal(got[3].cpu().bool(), done)
    s = got[0].cpu().double()
    fine = torch.isfinite(best)
    assert torch.equal(s[~fine], best[~fine])
    assert bool(((s - best)[fine].abs() <= 2.0 ** -22 * (1 + best[fine].abs())).all())


def logits_of(rows, vocab, seed, spread=2.0):
    return (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(seed)) * spread).half()


@pytest.mark.parametrize("G,W,n,vocab", [(1, 1, 1, 1), (1, 1, 3, 3), (2, 3, 5, 7), (3, 1, 4, 100), (1, 4, 4, 2047), (2, 4, 8, 2048), (1, 5, 5, 2049), (1, 4, 8, 32016), (2, 64, 128, 300), (3, 6, 18, 3), (2, 40, 80, 2),
                                         (1, 64, 64, 32016), (70, 8, 16, 2500), (600, 1, 2, 130), (9, 60, 7, 8193), (1, 2, 128, 129280), (130, 4, 4, 8191)])
@pytest.mark.parametrize("ended", [False, True])
def test_sizes(G, W, n, vocab, ended):
    g = torch.Generator().manual_seed(G + W)
    scores = -torch.rand(G * W, generator=g) * 9
    done = (torch.rand(G * W, generator=g) < 0.3).to(torch.uint8) if ended else None
    check(logits_of(G * W, vocab, vocab), scores, W, n, done, eos=min(EOS, vocab - 1))


def rearranged(rows, vocab, seed):
    """a row and the same values in other orders"""
    g = torch.Generator().manual_seed(seed)
    x = logits_of(1, vocab, seed)[0]
    return torch.stack([x] + [x[torch.randperm(vocab, generator=g)] for _ in range(rows - 1)])


@pytest.mark.parametrize("groups", [1, 80])
@pytest.mark.parametrize("vocab", [8000, 32016, 129280])
def test_beams_of_the_same_values_in_another_order(groups, vocab):
    """rows whose true sums are equal: with scores 2^-16 apart, twice the distance from which an order is kept, candidates are in it"""
    W = 7
    x = rearranged(W, vocab, vocab).repeat(groups, 1)
    check(x, (-torch.arange(W) * 2.0 ** -16).repeat(groups), W, 64)
    check(x, (torch.arange(W) * 2.0 ** -16 - 1).repeat(groups), W, 64)


@pytest.mark.parametrize("vocab", [3000, 8192, 32016])
def test_equal_beams_of_the_same_values(vocab):
    """at equal scores too the values are in their order, each beam's candidates in that of their tokens, and scores are as close as is said; beams of one slice are in order"""
    W, n = 6, 60
    x = rearranged(W, vocab, vocab + 1)
    s, parents, tokens, _ = (t.cpu() for t in K().beam_select(x.to(DEV), torch.zeros(W, device=DEV), W, n))
    value = x[parents[0].long(), tokens[0]].float()
    assert bool((value.diff() <= 0).all())
    exact = torch.log_softmax(x[:1].double(), 1)[0].max()
    assert bool((s[0].double() - (exact + (value.double() - value[0].double()))).abs().max() <= 2.0 ** -18 + 2.0 ** -24 * 16)
    for a, b in zip(range(n - 1), range(1, n)):
        if value[a] == value[b] and (parents[0, a] == parents[0, b] or vocab <= 8192):
            assert (parents[0, a], tokens[0, a]) < (parents[0, b], tokens[0, b])
    top = x[0].float().sort(descending=True).values.repeat_interleave(W)[:n]
    assert torch.equal(value, top)


def test_more_rows_than_a_grid_has():
    check(logits_of(70000, 9, 3), -torch.rand(70000, generator=torch.Generator().manual_seed(3)), 1, 3)
    check(logits_of(70000, 9, 4), -torch.rand(70000, generator=torch.Generator().manual_seed(4)), 10, 12)


@pytest.mark.parametrize("W,n,vocab", [(4, 64, 32016), (8, 32, 32016), (8, 33, 32016), (32, 64, 32016), (33, 64, 32016), (64, 128, 8192), (64, 128, 8193), (64, 128, 32768), (64, 128, 32769)])
def test_every_way_to_pick(W, n, vocab):
    """candidates for one wave, four, sixteen, and more of them than that; equal ones among them"""
    x = logits_of(W, vocab, W + n)
    check(x, -torch.rand(W, generator=torch.Generator().manual_seed(n)), W, n)
    check((x * 2).round() / 2, torch.zeros(W), W, n)
    check(x[:1].expand(W, -1).contiguous(), torch.zeros(W), W, n)


def test_first_step():
    """all beams are the same prompt and only the first counts; then none does but one"""
    row = logits_of(1, 32016, 1)
    scores = torch.full((4,), -math.inf)
    scores[0] = 0
    check(row.expand(4, -1).contiguous(), scores, 4, 8)
    scores[0], scores[2] = -math.inf, math.nan
    check(row.expand(4, -1).contiguous(), scores, 4, 8)
    check(row.expand(4, -1).contiguous(), torch.zeros(4), 4, 128)            # equal candidates of all beams


@pytest.mark.parametrize("vocab", [50, 2048, 10000])
@pytest.mark.parametrize("n", [1, 7, 128])
def test_ties_and_orders(vocab, n):
    """rows that are all equal, go up, go down, take two values, have their best values next to one another; zeros of both signs"""
    n = min(n, vocab)
    i = torch.arange(vocab)
    rows = [torch.zeros(vocab), i / 16.0, -i / 16.0, (i % 2).float(), torch.where((i >= vocab // 2) & (i < vocab // 2 + 40), 5.0 + i % 3, -i / 999.0), torch.where(i % 2 == 0, 0.0, -0.0),
            (i % 8 == 7).float() * 3]
    x = torch.stack(rows).half()
    for W in (1, 7):
        check(x, torch.zeros(7), W, n)
        check(x.flip(0).contiguous(), -torch.arange(7.0), W, n)


def test_many_candidates_in_one_thread():
    """the n largest values stand in as few threads as they can: every slice finds the most keys that it may"""
    for vocab, threads in ((8192, 128), (2048, 128), (40000, 100)):
        x = torch.full((1, vocab), -5.0)
        for t in range(threads):
            for c in range(vocab // 2048):
                x[0, c * 2048 + t * 8: c * 2048 + t * 8 + 8] = torch.arange(8) / 8 + t / 4 + c / 64
        x = x.half()
        check(x, torch.zeros(1), 1, 128)
        check(x.expand(600, -1).contiguous()[:, :], torch.zeros(600), 1, 128)        # (in slices of the wide kind)


def test_what_is_not_finite():
    x = logits_of(6, 3000, 5)
    x[0, :] = -math.inf                                                       # a row that forbids everything
    x[1, ::2] = math.nan
    x[2, 100:] = -math.inf
    x[3, 77] = math.inf
    x[4, [5, 2500]] = math.inf
    scores = torch.tensor([0.0, -1.0, -2.0, -0.5, -3.0, -0.25])
    for W in (1, 2, 3, 6):
        check(x, scores, W, 20)
        check(x, scores, W, 20, torch.tensor([0, 1, 0, 0, 0, 1], dtype=torch.uint8))
    check(torch.full((2, 70), -math.inf).half(), torch.zeros(2), 2, 100 if 100 <= 70 else 70)
    check(torch.full((2, 70), -math.inf).half(), torch.zeros(2), 2, 70, torch.ones(2, dtype=torch.uint8), eos=69)
    check(torch.full((2, 70), -math.inf).half(), torch.full((2,), -math.inf), 2, 70, torch.ones(2, dtype=torch.uint8), eos=0)


@pytest.mark.parametrize("infinite", [False, True])
def test_every_pattern_of_a_logit(infinite):
    """All values that 16 bits have, quiet and signalling NaN of either sign among them, which count as -infinity"""
    x = torch.arange(65536, dtype=torch.int32)
    x = torch.stack([x[torch.randperm(65536, generator=torch.Generator().manual_seed(s))] for s in (1, 2)]).to(torch.int16).view(torch.float16)
    if not infinite:
        x = torch.where(x == math.inf, torch.zeros_like(x), x)
    check(x, torch.tensor([0.0, -0.5]), 2, 128)
    check(x, torch.tensor([0.0, -0.5]), 1, 128)


def test_wide_range_of_scores():
    """sums of scores as long outputs have them, and logits of large magnitude"""
    check(logits_of(8, 32016, 6, 30.0), -torch.rand(8, generator=torch.Generator().manual_seed(6)) * 4000, 4, 8)


def test_strides_and_offsets():
    """rows further apart than the vocabulary, beginning at any value"""
    base = logits_of(6, 5003, 7).to(DEV)
    for a, b in ((0, 5003), (1, 5000), (3, 4100), (8, 2056)):
        check(base[:, a:b], torch.linspace(-1, 0, 6), 3, 6)
    check(base.view(-1)[5:5 + 2 * 5003].view(2, 5003), torch.zeros(2), 2, 4)


def test_defaults_and_empty():
    x, s = logits_of(6, 100, 8).to(DEV), torch.zeros(6, device=DEV)
    a, b = K().beam_select(x, s, 3), K().beam_select(x, s, 3, 3, ended=torch.zeros(6, dtype=torch.bool, device=DEV))
    assert all(torch.equal(p, q) and p.shape == (2, 3) for p, q in zip(a, b))
    assert K().beam_select(x[:0], s[:0], 3)[2].shape == (0, 3)


@pytest.mark.parametrize("kw,why", [(dict(beams=65), "beams"), (dict(n=129), "n="), (dict(n=10 ** 9), "n="), (dict(eos=100), "eos"), (dict(eos=-1), "eos")], ids=str)
def test_sizes_that_are_refused(kw, why):
    from spec_mcts_amd._lib import SmhError
    x, s = logits_of(65, 100, 8).to(DEV), torch.zeros(65, device=DEV)
    with pytest.raises(SmhError, match=why):
        K().beam_select(x, s, **{**dict(beams=13, n=5), **kw})


def test_captured_and_on_two_streams():
    x, s = logits_of(8, 32016, 9).to(DEV), torch.linspace(-2, 0, 8, device=DEV)
    want = [K().beam_select(x.roll(i, 0).contiguous(), s, 4) for i in range(4)]
    side = torch.cuda.Stream()
    buf = x.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K().beam_select(buf, s, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K().beam_select(buf, s, 4)
    for i in range(4):
        buf.copy_(x.roll(i, 0))
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = K().beam_select(x, s, 4)
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))


# ---- reordering -----------------------------------------------------------------------------------------------------------------
def moved(x, parents, cols=None):
    G, W = parents.shape
    row = (torch.arange(G, device=x.device)[:, None] * W + parents.to(x.device).clamp(0, W - 1)).view(-1)
    y = x.clone()
    if cols is None:
        y[:] = x[row]
    else:
        y[:, :cols] = x[row][:, :cols]
    return y


@pytest.mark.parametrize("G,W", [(1, 1), (1, 2), (3, 4), (2, 64), (17, 5), (4, 8), (2, 9), (2, 16), (1, 17), (1, 33)])
@pytest.mark.parametrize("upto", [0, 1, 33, 1000, 2 ** 31 - 1, -5])
def test_states_follow(G, W, upto):
    g = torch.Generator(device=DEV).manual_seed(G * W)
    R = G * W
    cols = [torch.randint(0, 1 << 30, (R, 133), device=DEV, generator=g).int(), torch.randint(0, 1 << 60, (R, 50), device=DEV, generator=g)]
    rows = [torch.randn((R, 2, 64, 128), device=DEV, generator=g).half(), torch.randn(R, device=DEV, generator=g), torch.randn((R, 7, 3), device=DEV, generator=g),
            torch.randint(0, 255, (R, 64), device=DEV, generator=g).to(torch.uint8)]
    for parents in (torch.arange(W).repeat(G, 1), torch.arange(W).roll(1).repeat(G, 1), torch.zeros((G, W)), torch.randint(0, W, (G, W), generator=torch.Generator().manual_seed(W)),
                    torch.randint(-3, W + 3, (G, W), generator=torch.Generator().manual_seed(W))):
        parents = parents.to(torch.int32).to(DEV)
        want = [moved(x, parents) for x in rows] + [moved(x, parents, min(max(upto, 0), x.shape[1])) for x in cols]
        K().beam_reorder(parents, rows=rows, columns=cols, upto=torch.tensor([upto], dtype=torch.int32, device=DEV))
        assert all(torch.equal(a, b) for a, b in zip(rows + cols, want))


def test_strided_and_odd_states():
    """rows of a wider tensor (what lies between them stays), widths that are no multiple of 16 bytes, empty ones, none at all"""
    wide = torch.arange(12 * 100, device=DEV, dtype=torch.int32).view(12, 100).clone()
    parents = torch.tensor([[3, 0, 0, 1], [1, 1, 2, 0], [0, 1, 2, 3]], dtype=torch.int32, device=DEV)
    want = wide.clone()
    want[:, 10:47] = moved(wide[:, 10:47], parents)
    K().beam_reorder(parents, rows=[wide[:, 10:47], torch.empty((12, 0), device=DEV)])
    assert torch.equal(wide, want)
    want[:, 1:90] = moved(wide[:, 1:90], parents, 60)
    K().beam_reorder(parents, columns=[wide[:, 1:90]], upto=torch.tensor([60], dtype=torch.int32, device=DEV))
    assert torch.equal(wide, want)
    K().beam_reorder(parents)
    K().beam_reorder(parents[:0], rows=[wide[:0]])


def test_captured_reorder():
    x = torch.randn((8, 4, 64, 128), device=DEV).half()
    t = torch.arange(8 * 40, device=DEV, dtype=torch.int32).view(8, 40).clone()
    parents, n = torch.zeros((2, 4), dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    K().beam_reorder(parents + torch.arange(4, dtype=torch.int32, device=DEV), rows=[x], columns=[t], upto=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K().beam_reorder(parents, rows=[x], columns=[t], upto=n)
    for i, p in enumerate(([[1, 0, 3, 2], [0, 0, 0, 0]], [[3, 3, 1, 0], [2, 1, 0, 3]], [[0, 1, 2, 3], [1, 2, 3, 0]])):
        parents.copy_(torch.tensor(p, dtype=torch.int32))
        n.fill_(10 * i + 5)
        want = moved(x, parents), moved(t, parents, 10 * i + 5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(t, want[1])
