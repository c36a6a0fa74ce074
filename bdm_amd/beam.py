"""Beam search over the language model.

The reference's inference decodes one continuation a prompt
(reproduction/experiments/perf_inference_case.py:140-160).  Here a prompt's
``beams`` continuations are decoded side by side: one model step for all of them,
``ops.beam_select`` over beams and vocabulary, and the caches put in the order of
the chosen parents.  Dense caches are reordered in place
(``ops.reorder_states``); a paged cache (``BankPages``) forks, which moves no
state: beams share the pages of every bank that they have not written since
they parted.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import ops
from .pages import BankPages


class BeamResult(NamedTuple):
    tokens: Tensor   # [B, beams, length] int64, best first; eos behind the end
    scores: Tensor   # [B, beams] FP32 summed log-probabilities
    lengths: Tensor  # [B, beams] int32 tokens up to and with eos


class _Search:
    """The beams of a batch of prompts: what one step reads and leaves."""

    def __init__(self, model, prompt: Tensor, beams: int, eos, length_penalty: float, paged: bool, length: int) -> None:
        self.model, self.beams, self.eos, self.penalty = model, beams, eos, length_penalty
        batch = prompt.shape[0]
        rows = batch * beams
        self.pages = self.caches = None
        firsts = range(0, rows, beams)
        if paged:
            memory, layers = model.config.memory, len(model.layers)
            # enough whatever the routes: the initial state, the banks that each prompt and each beam's own tokens
            # can write, and the pages that a step takes before those that it abandons are free
            banks, selected = memory.bank_count, memory.selected_banks
            prompts, own = (min(banks, selected * n) for n in (prompt.shape[1], length))
            need = layers * min(banks + batch * prompts + rows * own, (rows + 1) * banks) + rows * selected
            self.pages = model.create_pages(rows + 1, need)
            model.load_initial(self.pages, rows)
            logits = model.prefill_pages(prompt, self.pages, firsts, base=rows)
            self.pages.fork(torch.arange(rows, device=prompt.device) // beams * beams)
        else:
            logits, caches = model.prefill(prompt)
            self.caches = [c.repeat_interleave(beams, 0) if beams > 1 else c for c in caches]
        chosen = self._choose(logits.view(batch, 1, -1), torch.zeros(batch, 1, device=prompt.device), None,
                              torch.zeros(batch, 1, dtype=torch.int32, device=prompt.device))
        self.tokens, self.scores, self.lengths = chosen.tokens, chosen.scores, chosen.lengths
        self.finished, self.parents = chosen.finished, torch.zeros_like(chosen.tokens)

    def _choose(self, logits, scores, finished, lengths):
        return ops.beam_select(logits, scores, width=self.beams, finished=finished, eos=self.eos, lengths=lengths,
                               length_penalty=self.penalty)

    def step(self) -> None:
        """One token: the static tensors are read and written in place."""
        batch, beams = self.tokens.shape
        tokens = self.tokens.view(-1, 1)
        if self.pages is not None:
            logits = self.model.step_pages(tokens, self.pages)
        else:
            logits, _ = self.model.step(tokens, self.caches)
        chosen = self._choose(logits.view(batch, beams, -1), self.scores, self.finished, self.lengths)
        if self.pages is not None:
            self.pages.fork(chosen.parents)
        else:
            ops.reorder_states(self.caches, chosen.parents, beams=beams)
        self.tokens.copy_(chosen.tokens)
        self.scores.copy_(chosen.scores)
        self.parents.copy_(chosen.parents)
        self.lengths.copy_(chosen.lengths)
        if self.finished is not None:
            self.finished.copy_(chosen.finished)


@torch.no_grad()
def beam_search(model, prompt: Tensor, *, beams: int, length: int, eos: int | None = None,
                length_penalty: float = 0.0, paged: bool = False, graph: bool = False) -> BeamResult:
    """The ``beams`` best continuations of up to ``length`` tokens of each prompt.

    model: a ``BDMLanguageModel`` on a ROCm device; prompt [B, T] int64.  A
    continuation that takes ``eos`` is ended and keeps its score; with
    ``length_penalty`` a, continuations compare by score / length**a.  ``paged``
    keeps the beams in a ``BankPages`` cache instead of one dense cache a beam
    (the same search; its decode step rounds once where the dense step rounds
    every product and sum, so near ties can fall the other way).  Its pool holds
    what the search can need whatever the routes are, which for long prompts is
    as much as the dense caches; a loop over ``create_pages`` with a pool of the
    caller's own size saves memory where banks stay shared.  ``graph`` replays the
    steps behind the third token from one HIP graph, captured in each call.  Every
    16 tokens the host looks whether all continuations have ended."""
    if prompt.ndim != 2 or prompt.dtype != torch.int64 or 0 in prompt.shape:
        raise ValueError('prompt must be int64 [batch, positive time]')
    if not prompt.is_cuda:
        raise ValueError('the HIP path requires tensors on a ROCm device')
    if not 1 <= beams <= min(ops.BEAM_MAX, model.config.vocab_size) or length < 1:
        raise ValueError(f'beam_search needs 1 to {min(ops.BEAM_MAX, model.config.vocab_size)} beams and a length')
    device, batch = prompt.device, prompt.shape[0]
    tokens = torch.empty(length, batch, beams, dtype=torch.int64, device=device)
    parents = torch.empty_like(tokens)
    stream = torch.cuda.Stream(device) if graph else torch.cuda.current_stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    captured = None
    try:
        with torch.cuda.stream(stream):
            search = _Search(model, prompt, beams, eos, length_penalty, paged, length)
            done = length
            for t in range(length):
                if t == 0:
                    pass  # chosen from the prompt's logits
                elif not graph or t < 3:
                    search.step()
                else:
                    if captured is None:
                        captured = torch.cuda.CUDAGraph()
                        torch.cuda.synchronize(device)
                        with torch.cuda.graph(captured, stream=stream):
                            search.step()
                    captured.replay()
                tokens[t].copy_(search.tokens)
                parents[t].copy_(search.parents)
                if eos is not None and t % 16 == 15 and bool(search.finished.all()):
                    done = t + 1
                    break
            # each continuation from its last token back to its first
            out = torch.full((batch, beams, length), 0 if eos is None else eos, dtype=torch.int64, device=device)
            beam = torch.arange(beams, device=device).expand(batch, beams)
            for t in range(done - 1, -1, -1):
                out[:, :, t] = tokens[t].gather(1, beam)
                beam = parents[t].gather(1, beam) % beams
            result = BeamResult(out, search.scores, search.lengths)
    finally:  # also where a step fails: what the stream still reads and writes is not given back before it is done
        torch.cuda.current_stream(device).wait_stream(stream)
        if captured is not None:
            stream.synchronize()  # the last replay, before the graph and its memory go
    if graph:
        for t in result:
            t.record_stream(torch.cuda.current_stream(device))
    return result
