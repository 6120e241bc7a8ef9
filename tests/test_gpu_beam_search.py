"""Beam search through the model, and beams over the 8-bit cache, against searches that keep every beam's tokens and start over."""
import math

import pytest
import torch

from oracle import q40_oracle as OR
from tests import kv8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def small_model(max_batch=8, max_seq=24, heads=2, kv_heads=None, seed=1, vocab=320):
    from spec_mcts_amd import ModelArgs
    from spec_mcts_amd.load_q40 import load_q40
    cfg = dict(dim=heads * 128, n_layers=2, n_heads=heads, n_kv_heads=kv_heads, vocab_size=vocab, multiple_of=128, max_batch_size=max_batch, max_seq_len=max_seq, max_prompt_seq_len=16)
    return load_q40(OR.random_q40_state_dict(OR.OracleArgs(**cfg), seed=seed, std=0.05), ModelArgs(**cfg), device=DEV)


def pick(logits, scores, ended, eos):
    """The W best continuations in 64 bits"""
    x = logits.double().cpu()
    total = scores[:, None] + torch.log_softmax(x, 1)
    stay = torch.full_like(total, -math.inf)
    stay[:, eos] = scores
    total = torch.where(ended[:, None], stay, total)
    best, at = torch.sort(total.view(-1), descending=True, stable=True)
    W, V = logits.shape
    best, at = best[:W], at[:W]
    return best, at // V, at % V


@torch.inference_mode()
def by_starting_over(m, prompt, W, steps, eos):
    """Every step runs the prompt and all tokens of the W beams again, each beam in a row of its own"""
    tokens = torch.zeros((W, 0), dtype=torch.int64)
    scores = torch.full((W,), -math.inf, dtype=torch.float64)
    scores[0] = 0
    ended, lengths = torch.zeros(W, dtype=torch.bool), torch.zeros(W, dtype=torch.int64)
    for t in range(steps):
        m.resetSeq()
        logits = m(prompt, 0)[:, -1].expand(W, -1)
        m._table(logits.device)
        m._forked = True                           # rows are read through the (identity) table, by the kernels that the search uses
        for j in range(t):
            logits = m(tokens[:, j:j + 1].to(DEV).contiguous(), prompt.shape[1] + j)[:, -1]
        scores, parent, token = pick(logits, scores, ended, eos)
        scores = scores.float().double()
        tokens, ended, lengths = torch.cat((tokens[parent], token[:, None]), 1), ended[parent] | (token == eos), lengths[parent]
        lengths += ~ended
        if bool(ended.all()):
            break
    return tokens, lengths, scores


@pytest.mark.parametrize("W,heads,kv_heads", [(1, 2, None), (3, 2, None), (4, 2, None), (5, 4, 2), (8, 2, None)])
@pytest.mark.parametrize("use_graph", [True, False])
def test_the_model_s_beams(W, heads, kv_heads, use_graph):
    from spec_mcts_amd.beam import BeamSearch
    m = small_model(heads=heads, kv_heads=kv_heads, seed=W)
    for seed, P in ((0, 9), (1, 16), (0, 9)):
        prompt = torch.randint(0, 320, (1, P), generator=torch.Generator().manual_seed(seed)).to(DEV)
        want, lengths, scores = by_starting_over(m, prompt, W, 12, 2)
        search = BeamSearch(m, W, 12, use_graph=use_graph)
        for _ in range(2):                         # (the second one replays what the first recorded)
            tokens, n, s = search.search(prompt)
            assert torch.equal(tokens.cpu(), want) and torch.equal(n.cpu().long(), lengths)
            assert bool(((s.cpu().double() - scores).abs() <= 1e-4).all())


def test_beams_end_and_are_ranked():
    """an end token that is often likely: beams end at different steps, the search with them; length penalties only reorder"""
    from spec_mcts_amd.beam import BeamSearch
    m = small_model(seed=3)
    prompt = torch.randint(0, 320, (1, 9), generator=torch.Generator().manual_seed(5)).to(DEV)
    free, _, _ = BeamSearch(m, 4, 12, eos=319).search(prompt)
    values, counts = torch.unique(free[:, 1:8], return_counts=True)
    eos = int(values[counts.argmax()])
    want, lengths, scores = by_starting_over(m, prompt, 4, 12, eos)
    tokens, n, s = BeamSearch(m, 4, 12, eos=eos).search(prompt)
    steps = want.shape[1]
    assert torch.equal(tokens.cpu()[:, :steps], want) and torch.equal(n.cpu().long(), lengths) and bool((tokens[:, steps:] == eos).all())
    other, n2, s2 = BeamSearch(m, 4, 12, length_penalty=1.0, eos=eos).search(prompt)
    assert bool((s2 / n2.clamp(min=1)).diff().le(0).all()) and sorted(s2.tolist()) == sorted(s.tolist())


def test_limits():
    from spec_mcts_amd.beam import BeamSearch
    m = small_model(max_batch=4, max_seq=5)
    for bad in (dict(beams=5), dict(beams=0), dict(max_new=0), dict(eos=320)):
        with pytest.raises(AssertionError):
            BeamSearch(**{**dict(model=m, beams=2, max_new=4), **bad})
    tokens, n, _ = BeamSearch(m, 4, 100).search(torch.zeros((1, 3), dtype=torch.int64, device=DEV))
    assert tokens.shape == (4, 5) and int(n.max()) <= 5
    with pytest.raises(AssertionError):
        BeamSearch(m, 2, 4).search(torch.zeros((1, 17), dtype=torch.int64, device=DEV))


def test_one_search_object_for_everything():
    """prompts of several lengths, other numbers of beams, and the sampler on the same model in between, by one object"""
    from spec_mcts_amd.beam import BeamSearch
    from spec_mcts_amd.mcts import mcts
    m = small_model(seed=4)
    search = BeamSearch(m, 4, 10)
    for W, P in ((4, 9), (4, 16), (6, 9), (3, 9), (4, 9)):
        prompt = torch.randint(0, 320, (1, P), generator=torch.Generator().manual_seed(P)).to(DEV)
        want, lengths, scores = by_starting_over(m, prompt, W, 10, 2)
        search.beams = W
        for _ in range(2):
            tokens, n, s = search.search(prompt)
            assert torch.equal(tokens.cpu()[:, :want.shape[1]], want) and torch.equal(n.cpu().long(), lengths)
            assert bool(((s.cpu().double() - scores).abs() <= 1e-4).all())
            mcts(m, 8, top_k=8, temp=1.0).search(prompt, 8)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_beams_over_the_8_bit_cache(window, sinks):
    """Append, attend, project, select, reorder - one layer over random weights, two prompts of different lengths with three beams each - for 70 steps, past a
    border of a block: at every step the cache holds, for each beam, the rows of its own history, and the attention is that of 64 bits over them"""
    from spec_mcts_amd import kernels as K
    g = torch.Generator().manual_seed(31)
    G, W, H, Hkv, V, steps = 2, 3, 4, 2, 250, 70
    R = G * W
    emb = torch.randn((V, (H + 2 * Hkv) * 128), generator=g).half()
    head = (torch.randn((V, H * 128), generator=g) * 0.2).half().to(DEV)
    emb_d = emb.to(DEV)
    cos, sin = O.tables(400)
    cos_d, sin_d = cos.to(DEV), sin.to(DEV)
    prompts = [torch.randint(0, V, (n,), generator=g) for n in (100, 37)]
    history = [prompts[r // W].tolist() for r in range(R)]
    split = lambda x: (x[:, :H * 128].view(-1, H, 128), x[:, H * 128:(H + Hkv) * 128].view(-1, Hkv, 128), x[:, (H + Hkv) * 128:].view(-1, Hkv, 128))      # noqa: E731
    cache = K.kv8_cache(R, 256, Hkv, DEV)
    lens = torch.zeros(R, dtype=torch.int32, device=DEV)
    new = [len(h) for h in history]
    cu = torch.tensor([sum(new[:r]) for r in range(R + 1)], dtype=torch.int32, device=DEV)
    q, k, v = split(emb_d[torch.tensor(sum(history, []), device=DEV)])
    q = K.kv8_append(q, k, v, cos_d, sin_d, cache, lens, cu=cu, max_new=max(new))
    o = K.kv8_attn(q, cache, lens, cu=cu, max_new=max(new), window=window, sinks=sinks)[cu[1:].long() - 1]
    lens += cu.diff()
    scores = torch.full((R,), -math.inf, device=DEV)
    scores[::W] = 0
    for step in range(steps):
        logits = K.f16_linear(o.reshape(R, H * 128).contiguous(), head)
        best, parents, tokens, _ = K.beam_select(logits, scores, W, eos=V - 1)
        want = torch.sort((scores[:, None].double() + torch.log_softmax(logits.double(), 1)).view(G, -1), dim=1, descending=True, stable=True).indices[:, :W]
        assert torch.equal(parents.long() * V + tokens, want)
        scores = best.view(-1)
        # both prompts' blocks: what beams of a group have in common is the number of blocks, so each group reorders by its own
        for i in range(G):
            mine = slice(i * W, i * W + W)
            K.beam_reorder(parents[i:i + 1], rows=[cache.open_k[mine], cache.open_v[mine]], columns=[cache.pages[mine]], upto=lens[i * W:i * W + 1] // 64)
        p = parents.cpu()
        history = [history[r // W * W + int(p[r // W, r % W])] + [int(tokens.view(-1)[r])] for r in range(R)]
        q, k, v = split(emb_d[tokens.view(-1)])
        q = K.kv8_append(q, k, v, cos_d, sin_d, cache, lens)
        o = K.kv8_attn(q, cache, lens, max_len=256, window=window, sinks=sinks)
        lens += 1
        if step in (0, 1, 26, 27, 28, 69):
            for r, h in enumerate(history):
                s = O.Sequence(Hkv)
                hq, hk, hv = split(emb[torch.tensor(h)])
                place = torch.arange(len(h))
                s.add(O.rotate(hk, cos, sin, place), hv)
                hk, hv = s.held()
                got = K.kv8_rows(cache, lens, torch.zeros_like(lens), len(h))
                assert torch.equal(got[0][r].cpu(), hk.float().half()) and torch.equal(got[1][r].cpu(), hv.float().half()), (step, r)
                want_o, mean = O.attention(O.rotate(hq[-1:], cos, sin, place[-1:]), hk, hv, len(h) - 1, window, sinks)
                bound = O.attention_bound(want_o, mean, len(h), float(hv.abs().max()))
                assert bool(((o[r:r + 1].cpu().double() - want_o).abs() <= bound).all()), (step, r)
