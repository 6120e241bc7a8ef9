"""Beam search next to the tree sampler: the `beams` most likely continuations of one prompt instead of drawn ones (the reference has only the sampler,
mcts.py:67-182).

The beams are branches that share the prompt's K/V, as in the sampler.  A step is the forward of all beams, kernels.beam_select (which beams go on with which
token) and kernels.beam_reorder (the page table's ids of the suffix rows written so far and the tokens so far follow their beams: no K or V row moves, because a
beam appends to its own slot of the step and earlier slots are never written again).  With the fused forward a step is one replay of a captured HIP graph
(decode.BucketedForward); the host reads one number a step, a step late, to see whether all beams have ended.
"""
from __future__ import annotations

import torch

from . import kernels as K
from .decode import BucketedForward
from .mcts import EOS


class BeamSearch:
    def __init__(self, model, beams: int, max_new: int, length_penalty: float = 0.0, eos: int = EOS, use_graph: bool = True):
        """length_penalty a: hypotheses are returned in the order of score / max(length, 1) ** a; the search itself keeps the largest scores."""
        assert 1 <= beams <= min(64, model.params.max_batch_size) and max_new >= 1 and 0 <= eos < model.params.vocab_size
        self.model, self.beams, self.max_new, self.length_penalty, self.eos, self.use_graph = model, beams, max_new, float(length_penalty), eos, use_graph
        self._fwd = None
        self.last_steps = 0                        # decode steps of the last search

    def _buffers(self, dev, steps: int) -> None:
        W = self.beams
        self._fwd = BucketedForward(self.model, W, use_graph=self.use_graph)
        self._key = (W, steps, self.eos, self.use_graph, dev)
        self.results = torch.zeros((W, steps), dtype=torch.int64, device=dev)
        self.scores = torch.zeros(W, dtype=torch.float32, device=dev)
        self.ended = torch.zeros(W, dtype=torch.uint8, device=dev)
        self.lengths = torch.zeros(W, dtype=torch.int32, device=dev)
        self.left = torch.zeros(1, dtype=torch.int64, device=dev)
        self._host = torch.zeros((2, 1), dtype=torch.int64).pin_memory()
        self._events = [torch.cuda.Event(), torch.cuda.Event()]

    def _expand(self, logits: torch.Tensor) -> None:
        """Selection and reordering on logits [beams, vocab]; state[1] rows and tokens exist.  All tensors live at fixed addresses."""
        W, written = self.beams, self._fwd.state[1:2]
        scores, parents, tokens, ended = K.beam_select(logits, self.scores, W, W, ended=self.ended, eos=self.eos)
        K.beam_reorder(parents, rows=[self.lengths], columns=[self.model._table(logits.device)[:W], self.results], upto=written)
        self.results.scatter_(1, written.long().expand(W, 1), tokens.view(W, 1))
        self.scores.copy_(scores.view(-1))
        self.ended.copy_(ended.view(-1))
        self.lengths.add_(1 - self.ended)
        self._fwd.tokens.view(-1).copy_(tokens.view(-1))
        torch.sum(1 - self.ended, 0, keepdim=True, out=self.left)

    @torch.inference_mode()
    def search(self, prompt: torch.Tensor):
        """prompt int64 [1, P] -> (tokens int64 [beams, steps], lengths int32 [beams], scores float32 [beams]), best first: a hypothesis is its first
        `length` tokens (the end token not among them), its score the sum of their log probabilities (and the end token's)."""
        m, W = self.model, self.beams
        assert m.fused and m.paged_kv and not m.per_branch_kv, "beams share suffix rows through the page table"
        dev = m.norm.weight.device
        assert prompt.shape[1] <= m.params.max_prompt_seq_len
        steps = min(self.max_new, m.params.max_seq_len)
        if self._fwd is None or self._key != (W, steps, self.eos, self.use_graph, dev) or self._fwd.model is not m:
            self._buffers(dev, steps)
        fwd = self._fwd
        m.resetSeq()
        self.results.fill_(self.eos)
        self.scores.fill_(-float("inf"))
        self.scores[0] = 0.0                       # all beams are the prompt: the first counts
        self.ended.zero_()
        self.lengths.zero_()
        fwd.post = lambda logits: self._expand(logits[:, -1, :])
        logits = m(prompt[:1].to(dev), 0)
        fwd.begin()
        self._expand(logits[:, -1, :].expand(W, -1).contiguous())
        done = 1
        for t in range(1, steps):
            self._host[t & 1].copy_(self.left, non_blocking=True)      # how many go on behind token t - 1
            self._events[t & 1].record()
            if t > 1:
                self._events[(t - 1) & 1].synchronize()
                if int(self._host[(t - 1) & 1]) == 0:                  # all had ended a step ago: the last one added nothing
                    break
            fwd.step(None, W)
            done = t + 1
        torch.cuda.synchronize()
        self.last_steps = done - 1
        rank = self.scores / self.lengths.clamp(min=1).float() ** self.length_penalty
        order = torch.sort(rank, descending=True, stable=True).indices
        return self.results[order, :done], self.lengths[order], self.scores[order]
