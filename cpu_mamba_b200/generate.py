"""Autoregressive generation on the GPU around forward_step.

The reference's README (README.md:75-86) sketches the loop: prefill the prompt
once with forward_with_final_state, then forward_step token by token -- "sample,
append, repeat" -- with the sampling left to the caller.  Here the whole loop
stays on the device: a sampler maps each step's output y (B, d_model) to the
next step's input and a token id in device ops only, so ``steps_per_graph``
consecutive steps (model step + sampling) are captured as ONE CUDA graph and
replayed; the host neither waits for nor reads a token until the end.

Any model with ``forward_with_final_state`` / ``forward_step`` works: a
CPUMamba, a MambaStack, or a ChannelShardedMamba (whose graph then holds its
all-reduces).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import ops


class LogitRules:
    """What a sampler or a beam search applies to the logits of its rows
    (ops.adjust_logits): penalties for tokens already seen, biases, a grammar's bit
    mask.  Holds the rows' histories, ``tokens`` (rows, capacity) with ``lengths`` and
    ``prompt_lengths`` (rows,), int64, on the device; the loops append each chosen token,
    inside their graphs, and a full history takes no more.

    ``prompt_tokens`` (rows, n) int64 with optional ``prompt_lengths`` (rows,) starts the
    histories (they count for the repetition penalty only).  The penalties are numbers or
    float32 (rows,); bias_tokens and bias (rows, n) and mask (rows, ceil(vocab / 32)) are
    as in ops.adjust_logits, and may be changed in place between steps; a number is part
    of a loop's graph and stays what it was.  Histories go on from call to call: a new
    prompt takes new rules (or ``tokens``, ``lengths`` and ``prompt_lengths`` set anew).

    In a beam search of B requests the rows are its B x beams beams, beam j of request b
    in row b x beams + j.  A request's beams start alike, with one prompt and one set of
    penalties and biases; their histories follow them, and their masks where rows have
    masks of their own."""

    def __init__(self, rows: int, capacity: int, device="cuda",
                 prompt_tokens: Optional[torch.Tensor] = None,
                 prompt_lengths: Optional[torch.Tensor] = None, repetition_penalty=1.0,
                 frequency_penalty=0.0, presence_penalty=0.0,
                 bias_tokens: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                 mask: Optional[torch.Tensor] = None):
        if rows < 1 or capacity < 1:
            raise ValueError("rows and capacity must be >= 1")
        self.tokens = torch.full((rows, capacity), -1, dtype=torch.long, device=device)
        self.prompt_lengths = torch.zeros(rows, dtype=torch.long, device=device)
        if prompt_tokens is not None:
            n = prompt_tokens.shape[-1]
            if prompt_tokens.shape != (rows, n) or n > capacity:
                raise ValueError(f"prompt_tokens must be ({rows}, up to {capacity}), got "
                                 f"{tuple(prompt_tokens.shape)}")
            self.tokens[:, :n] = prompt_tokens
            self.prompt_lengths.fill_(n)
            if prompt_lengths is not None:
                self.prompt_lengths.copy_(prompt_lengths.clamp(0, n))
        elif prompt_lengths is not None:
            raise ValueError("prompt_lengths need prompt_tokens")
        self.lengths = self.prompt_lengths.clone()
        self.penalties = (repetition_penalty, frequency_penalty, presence_penalty)
        self.bias_tokens, self.bias, self.mask = bias_tokens, bias, mask

    def adjust(self, logits: torch.Tensor, temperature=1.0, rows: slice = slice(None)
               ) -> torch.Tensor:
        """The logits of (a slice of) the rows, adjusted in place where they are a new
        tensor's; returns them."""
        def part(t):
            return t[rows] if isinstance(t, torch.Tensor) else t

        rep, freq, pres = (part(v) for v in self.penalties)
        return ops.adjust_logits(logits, part(self.tokens), part(self.lengths),
                                 part(self.prompt_lengths), rep, freq, pres,
                                 part(self.bias_tokens), part(self.bias), part(self.mask),
                                 temperature, out=logits)

    def append(self, tokens: torch.Tensor) -> None:
        """Each row's newest token (rows,)."""
        capacity = self.tokens.shape[1]
        at = self.lengths.clamp(max=capacity - 1)[:, None]
        kept = self.tokens.gather(1, at)
        self.tokens.scatter_(1, at, torch.where((self.lengths < capacity)[:, None],
                                                tokens[:, None], kept))
        self.lengths.add_(1).clamp_(max=capacity)

    def _own_mask(self) -> list:
        """The mask where each row has its own (not one row expanded)."""
        shared = self.mask is None or self.mask.stride(0) == 0
        return [] if shared else [self.mask]

    def reorder(self, parents: torch.Tensor) -> None:
        """The rows' histories and masks follow their parents (B, beams)."""
        masks = self._own_mask()
        together = [m.contiguous() for m in masks]        # rows of a wider buffer: a copy
        ops.reorder_states([self.tokens, self.lengths] + together, parents)
        for mask, moved in zip(masks, together):
            if not mask.is_contiguous():
                mask.copy_(moved)

    def _saved(self) -> list:
        return [(t, t.clone()) for t in [self.tokens, self.lengths] + self._own_mask()]


class TiedEmbeddingSampler:
    """Token choice through an LM head tied to the input embedding (the
    Mamba language-model layout): logits = RMSNorm(y) E^T (the norm skipped
    when ``norm_weight`` is None), token = argmax (``temperature`` 0) or a
    sample of softmax(logits / temperature), optionally over the ``top_k``
    largest logits only (Gumbel-max with the device's default generator, so
    it can be captured in a graph).  ``rules`` adjust the logits first and keep
    the tokens chosen.  Returns (E[token], token)."""

    def __init__(self, embedding: torch.Tensor, temperature: float = 0.0,
                 top_k: Optional[int] = None, norm_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5, rules: Optional[LogitRules] = None):
        if embedding.dim() != 2:
            raise ValueError("embedding must be (vocab, d_model)")
        if temperature < 0:
            raise ValueError("temperature must be >= 0")
        self.E = embedding
        self.temperature = float(temperature)
        self.top_k = top_k
        self.norm_weight = norm_weight
        self.eps = eps
        self.rules = rules

    def logits(self, y: torch.Tensor) -> torch.Tensor:
        h = y
        if self.norm_weight is not None:
            h = F.rms_norm(y.float(), (y.shape[-1],), self.norm_weight.float(), self.eps)
        return h.float() @ self.E.float().t()

    def __call__(self, y: torch.Tensor) -> tuple:
        z = self.logits(y)
        if self.rules is not None:
            z = self.rules.adjust(z, self.temperature)
        elif self.temperature != 0.0:
            z = z / self.temperature
        if self.temperature == 0.0:
            tok = z.argmax(dim=-1)
        else:
            u = torch.rand_like(z).clamp_(min=1e-20, max=1.0 - 1e-7)
            g = z - torch.log(-torch.log(u))
            if self.top_k is not None and self.top_k < z.shape[-1]:
                kth = torch.topk(z, self.top_k, dim=-1).values[:, -1:]
                g = torch.where(z >= kth, g, torch.full_like(g, float("-inf")))
            tok = g.argmax(dim=-1)
        if self.rules is not None:
            self.rules.append(tok)
        return self.E[tok].to(y.dtype), tok


class DecodeLoop:
    """``steps_per_graph`` decode steps (model step + sampler) captured as one
    CUDA graph over a fixed state.  ``run(n)`` advances the state by n tokens
    and returns their ids (B, n): whole graph replays, then eager steps for
    the remainder (the same kernels, so the same bits).  The next input lives
    in ``self.x``; ``prefill`` sets it from a prompt."""

    def __init__(self, model, sampler, state, x0: torch.Tensor, steps_per_graph: int = 16):
        if steps_per_graph < 1:
            raise ValueError("steps_per_graph must be >= 1")
        self.model, self.sampler, self.state = model, sampler, state
        self.K = int(steps_per_graph)
        self.x = x0.detach().clone().contiguous()
        self.tokens = torch.empty(self.K, x0.shape[0], dtype=torch.long, device=x0.device)
        dev = self.x.device
        # warm-up on copies (library and sampler set-up outside the capture)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side), torch.no_grad():
            kept = _saved_rules(sampler)
            self._steps(self.x.clone(), _clone_state(state), torch.empty_like(self.tokens), 1)
            for t, before in kept:
                t.copy_(before)
        torch.cuda.current_stream(dev).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(self.graph):
            x_last = self._steps(self.x, self.state, self.tokens, self.K)
            self.x.copy_(x_last)

    def _steps(self, x, state, tokens, n):
        for k in range(n):
            y, _ = self.model.forward_step(x, state)
            x, tok = self.sampler(y)
            tokens[k].copy_(tok)
        return x

    @torch.no_grad()
    def run(self, n: int) -> torch.Tensor:
        out = []
        for _ in range(n // self.K):
            self.graph.replay()
            out.append(self.tokens.t().clone())
        r = n % self.K
        if r:
            tok = torch.empty(r, self.x.shape[0], dtype=torch.long, device=self.x.device)
            self.x.copy_(self._steps(self.x.clone(), self.state, tok, r))
            out.append(tok.t())
        if not out:
            return torch.empty(self.x.shape[0], 0, dtype=torch.long, device=self.x.device)
        return torch.cat(out, dim=1)


def _saved_rules(sampler) -> list:
    """What a step of the sampler changes in its rules, with copies."""
    rules = getattr(sampler, "rules", None)
    return [] if rules is None else rules._saved()


def _clone_state(state):
    if isinstance(state, dict):
        return {k: v.clone() for k, v in state.items()}
    return [_clone_state(s) for s in state]


@torch.no_grad()
def generate(model, sampler, prompt: torch.Tensor, max_new_tokens: int,
             steps_per_graph: int = 16) -> tuple:
    """Prefill ``prompt`` (B, T, d_model) with forward_with_final_state, pick
    the first token from its last position, then decode ``max_new_tokens`` - 1
    more on the GPU.  Returns (tokens (B, max_new_tokens), final state)."""
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be >= 1")
    y, state = model.forward_with_final_state(prompt)
    x, tok0 = sampler(y[:, -1])
    rest = max_new_tokens - 1
    if rest == 0:
        return tok0[:, None], state
    loop = DecodeLoop(model, sampler, state, x, min(steps_per_graph, rest))
    return torch.cat([tok0[:, None], loop.run(rest)], dim=1), state


class BeamLoop:
    """``steps_per_graph`` beam-search steps (model step, logits, selection over
    beams and vocabulary, reordering of the states) captured as one CUDA graph.

    state: the decode state of B * K sequences, beam j of request b in row
    b * K + j; ``tokens`` and ``scores`` (B, K): each beam's first token and its
    score.  A beam that emits ``eos_token`` is finished: it keeps its score and
    is padded with it.  ``run(n)`` takes n steps; ``result()`` returns the beams
    so far."""

    def __init__(self, model, sampler, state, tokens: torch.Tensor, scores: torch.Tensor,
                 eos_token: Optional[int] = None, steps_per_graph: int = 16,
                 dtype: Optional[torch.dtype] = None):
        if steps_per_graph < 1:
            raise ValueError("steps_per_graph must be >= 1")
        self.model, self.sampler, self.state = model, sampler, state
        self.K = int(steps_per_graph)
        self.dtype = sampler.E.dtype if dtype is None else dtype      # of the model's inputs
        self.eos = -1 if eos_token is None else int(eos_token)
        self.scores = scores.clone()
        self.last = tokens.clone()                    # each beam's newest token
        self.finished = self.last == self.eos
        self.history = [(None, tokens.clone())]       # (parents, tokens) of every step
        shape = (self.K,) + tuple(tokens.shape)
        self.parents = torch.empty(shape, dtype=torch.long, device=tokens.device)
        self.tokens = torch.empty_like(self.parents)
        dev = tokens.device
        self.graph = None
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side), torch.no_grad():
            # warm-up on copies (library set-up outside the capture)
            kept = self.state, self.scores, self.last, self.finished
            rules = _saved_rules(sampler)
            self.state = _clone_state(state)
            self.scores, self.last, self.finished = (t.clone() for t in kept[1:])
            self._steps(1)
            self.state, self.scores, self.last, self.finished = kept
            for t, before in rules:
                t.copy_(before)
        torch.cuda.current_stream(dev).wait_stream(side)

    def _steps(self, n):
        E, rules = self.sampler.E, getattr(self.sampler, "rules", None)
        B, K = self.scores.shape
        for i in range(n):
            x = E[self.last.flatten()].to(self.dtype)
            y, _ = self.model.forward_step(x, self.state)
            logits = self.sampler.logits(y)
            if rules is not None:
                logits = rules.adjust(logits)
            logits = logits.reshape(B, K, -1)
            best, par, tok = ops.beam_select(logits, self.scores, finished=self.finished,
                                             pad_token=max(self.eos, 0))
            ops.reorder_states(self.state, par)
            if rules is not None:
                rules.reorder(par)
                rules.append(tok.flatten())
            self.finished.copy_(self.finished.gather(1, par) | (tok == self.eos))
            self.scores.copy_(best)
            self.last.copy_(tok)
            self.parents[i].copy_(par)
            self.tokens[i].copy_(tok)

    def _keep(self, n):
        self.history += zip(self.parents[:n].clone().unbind(0), self.tokens[:n].clone().unbind(0))

    @torch.no_grad()
    def run(self, n: int) -> None:
        full, rest = divmod(n, self.K)
        if full and self.graph is None:
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self._steps(self.K)
        for _ in range(full):
            self.graph.replay()
            self._keep(self.K)
        if rest:
            self._steps(rest)
            self._keep(rest)

    def result(self) -> tuple:
        """(tokens (B, K, steps), scores (B, K)), each batch's best beam first."""
        B, K = self.scores.shape
        at = torch.arange(K, device=self.scores.device).expand(B, K)
        out = []
        for par, tok in reversed(self.history):
            out.append(tok.gather(1, at))
            if par is not None:
                at = par.gather(1, at)
        return torch.stack(out[::-1], -1), self.scores.clone()


def _repeat_state(state, n: int):
    if isinstance(state, dict):
        return {k: v.repeat_interleave(n, 0) for k, v in state.items()}
    return [_repeat_state(s, n) for s in state]


@torch.no_grad()
def beam_search(model, sampler, prompt: torch.Tensor, max_new_tokens: int, beams: int,
                eos_token: Optional[int] = None, length_penalty: float = 0.0,
                steps_per_graph: int = 16) -> tuple:
    """Beam search on the GPU: prefill ``prompt`` (B, T, d_model) once, then keep
    the ``beams`` best continuations of each request by total log probability
    (``sampler.logits``, adjusted by ``sampler.rules`` if it has any, through
    log-softmax), the beams' recurrent states and histories following them.  Beams that emit ``eos_token`` keep their score and are
    padded with it.  ``length_penalty`` a > 0 ranks the final beams by score /
    length^a, length counting up to the first ``eos_token``.

    Returns (tokens (B, beams, max_new_tokens), scores (B, beams)), the best
    beam of each request first."""
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be >= 1")
    if beams < 1:
        raise ValueError("beams must be >= 1")
    y, state = model.forward_with_final_state(prompt)
    logits = sampler.logits(y[:, -1])
    B, V = logits.shape
    if eos_token is not None and not 0 <= eos_token < V:
        raise ValueError(f"eos_token {eos_token} outside the vocabulary of {V}")
    if beams > V:
        raise ValueError(f"{beams} beams from a vocabulary of {V}")
    rules = getattr(sampler, "rules", None)
    if rules is not None:
        if rules.tokens.shape[0] != B * beams:
            raise ValueError(f"rules of {rules.tokens.shape[0]} rows for {B} x {beams} beams")
        logits = rules.adjust(logits, rows=slice(0, None, beams))
    start = torch.zeros(B, 1, device=logits.device)
    scores, _, tokens = ops.beam_select(logits.unsqueeze(1), start, num=beams)
    if rules is not None:
        rules.append(tokens.flatten())
    rest = max_new_tokens - 1
    loop = BeamLoop(model, sampler, _repeat_state(state, beams), tokens, scores, eos_token,
                    max(1, min(steps_per_graph, rest)), prompt.dtype)
    loop.run(rest)
    out, scores = loop.result()
    if length_penalty:
        done = out == (-1 if eos_token is None else eos_token)
        length = max_new_tokens - (done.cumsum(-1) > 0).sum(-1) + done.any(-1)
        order = (scores / length.to(scores.dtype) ** length_penalty).argsort(-1, descending=True)
        out = out.gather(1, order[..., None].expand_as(out))
        scores = scores.gather(1, order)
    return out, scores
