"""What every decoder of this package offers, whatever its model: the recorded step, and the calls that a generation loop,
the trace replay and the command line drive.

A decoder serves sequences through
    seq = decoder.open()                       a place for one sequence (its caches, states and position)
    rows = decoder.forward(seq, tokens, want)  runs the next tokens; logits of the wanted places among them
    ids = decoder.decode_greedy(seq, n)        n further tokens, arg-max fed back on the device
    ids = decoder.decode_sampled(seq, logits, n, sampling)  n further tokens, drawn on the device; the first from the last row of `logits`
    decoder.close(seq)                         gives the place back
Prompts may be fed in portions of any size; decode_greedy continues from the last place whose logits were asked for.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import ops


@dataclass
class Sampling:
    """How decode_sampled draws tokens (ops.sample); the same seed gives the same tokens.  A sequence's tokens use up the seed's random
    numbers one by one, over all of its calls: a reply drawn in pieces is the one drawn at once."""
    temperature: float = 1.0
    top_k: int = 0      # 0: all
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if not 0.0 <= self.temperature <= torch.finfo(torch.float32).max or not 0 <= self.top_k < 1 << 31 or not 0.0 <= self.top_p <= 1.0 or not 0.0 <= self.min_p <= 1.0:
            raise ValueError("a temperature of 0 or more (in 32 bits), a count top_k of 0 or more, and top_p and min_p from 0 to 1")

    def decode(self, logits: torch.Tensor, n: int, feed, drawn: int = 0) -> torch.Tensor:
        """int32 [n] on the device: the first token from the last row of `logits`, each further one from feed(the token before, a
        tensor of one element), which runs a step.  drawn: tokens that the sequence has drawn so far."""
        if logits is None:
            raise RuntimeError("ask for the logits of the last token first: the continuation is drawn from them")
        dev = logits.device
        kept = [torch.full((1,), v, dtype=t, device=dev) for v, t in ((self.temperature, torch.float32), (self.top_k, torch.int32),
                                                                       (self.top_p, torch.float32), (self.min_p, torch.float32))]
        u = torch.rand(drawn + n, device=dev, generator=torch.Generator(device=dev).manual_seed(self.seed))[drawn:]
        picks = torch.empty(n, dtype=torch.int32, device=dev)
        for i in range(n):
            rows = logits[-1:] if i == 0 else feed(picks[i - 1: i])
            ops.sample(rows, u[i: i + 1], temperature=kept[0], top_k=kept[1], top_p=kept[2], min_p=kept[3], tokens=picks[i: i + 1])
        return picks

    @staticmethod
    def ids(picks: torch.Tensor, status: torch.Tensor) -> list:
        """The drawn tokens on the host; waits for the device.  A step without a logit above minus infinity has no token, which is an
        error (and what the steps behind it leave in the decoder's status word, which is cleared, follows from it)."""
        ids = picks.cpu().tolist()
        none = next((i for i, t in enumerate(ids) if t < 0), None)
        if none is not None:
            st = int(status.item())
            status.zero_()
            raise RuntimeError(f"nothing to draw: token {none} of {len(ids)} has no logit above minus infinity" + (f" (status {st})" if st else ""))
        return ids


class RecordedStep:
    """A fixed sequence of launches over fixed device buffers: run eagerly, or recorded once into a CUDA graph and replayed."""

    def __init__(self, launches, device):
        self._launches, self._dev = launches, device
        self.graph = None

    def run(self) -> None:
        for f in self._launches:
            f()

    def capture(self) -> None:
        """Records the launches (call after at least one eager run; nothing is executed)."""
        torch.cuda.synchronize(self._dev)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self.run()
        self.graph = g

    def replay(self, n: int = 1) -> None:
        if self.graph is None:
            raise RuntimeError("capture() first")
        for _ in range(n):
            self.graph.replay()


@dataclass
class Request:
    prompt: list
    n_new: int
    tokens: list = field(default_factory=list)  # generated
    sampling: Sampling | None = None            # None: greedy


class RequestQueue:
    """First-come scheduler over a decoder: requests run one after the other, each prompt in portions of at most `portion`
    tokens (None: as the decoder cuts them), then greedy or sampled decoding; a finished request's place is reused by the next."""

    def __init__(self, decoder, portion: int | None = None):
        self.decoder, self.portion, self._waiting = decoder, portion, []

    def submit(self, prompt, n_new: int, sampling: Sampling | None = None) -> Request:
        r = Request([int(t) for t in prompt], int(n_new), sampling=sampling)
        if not r.prompt or r.n_new < 0:
            raise ValueError("a request needs a prompt and a count of new tokens that is not negative")
        self._waiting.append(r)
        return r

    def run(self) -> None:
        while self._waiting:
            r = self._waiting.pop(0)
            seq = self.decoder.open()
            try:
                step = self.portion or len(r.prompt)
                for at in range(0, len(r.prompt), step):
                    part = r.prompt[at: at + step]
                    last = at + step >= len(r.prompt)
                    logits = self.decoder.forward(seq, part, [len(part) - 1] if last else [])
                if r.n_new and r.sampling is not None:
                    r.tokens = self.decoder.decode_sampled(seq, logits, r.n_new, r.sampling)
                elif r.n_new:
                    r.tokens = self.decoder.decode_greedy(seq, r.n_new)
            finally:
                self.decoder.close(seq)


def generate(decoder, prompt, n_new: int, portion: int | None = None, sampling: Sampling | None = None) -> list:
    """Continuation of one prompt, greedy without `sampling`."""
    q = RequestQueue(decoder, portion)
    r = q.submit(prompt, n_new, sampling)
    q.run()
    return r.tokens
