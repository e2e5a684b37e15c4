"""Sampling: greedy and seeded temperature draws from float32 logits, on the device.

The reference samples greedily only (src/runner.ts:38-42: the first index with a strictly
greater value wins, so ties go to the lowest index; its device kernel refuses non-finite logits,
native/cuda-device.inc:97-115).  Temperature sampling is this engine's own: a row with
temperature T > 0 is drawn from softmax(logits / T) by inverse CDF at one uniform number, and that
number is a function of (seed, request id, output index) alone (``uniform_for``), so batching,
chunking, preemption and recomputation cannot change what a request generates.

``sample`` is the one place that launches the sampling kernels (csrc/sampling.cu).
"""
from __future__ import annotations

import hashlib

import torch

from .. import kernels


def uniform_for(seed: int, request_id: str, index: int) -> float:
    """The uniform number in [0, 1) that draws output token ``index`` of a request: a function of
    (seed, request id, index) alone.  24 bits, so that it is exact in float32 and below 1."""
    digest = hashlib.blake2b(f"{seed}:{request_id}:{index}".encode(), digest_size=8).digest()
    return (int.from_bytes(digest, "little") >> 40) / float(1 << 24)


def verify_uniforms(seed: int, request_id: str, index: int, tokens: int) -> tuple[list, list]:
    """The numbers that check ``tokens`` - 1 drafts from output token ``index`` of a request on: (accept, draw), one each per token of its
    step.  Functions of (seed, request id, index of the output token) alone; the draws are those of plain sampling (``uniform_for``).

    What comes out is distributed as the target's own tokens only if the drafts were drawn with other numbers than these: under the same
    seed and id a draft model sampled with ``uniform_for`` has the draws' own, and the token behind a draft that falls would follow from
    that draft.  ``draft_uniforms`` has numbers for the drafts."""
    return ([uniform_for(seed, f"{request_id}:accept", index + i) for i in range(tokens)],
            [uniform_for(seed, request_id, index + i) for i in range(tokens)])


def draft_uniforms(seed: int, request_id: str, index: int, drafts: int) -> list:
    """The numbers that draw a request's drafts for output tokens ``index`` on (``sample``'s ``uniforms`` on the draft model's logits): functions of
    (seed, request id, index of the output token) alone, and none of those that check the drafts (``verify_uniforms``)."""
    return [uniform_for(seed, f"{request_id}:draft", index + i) for i in range(drafts)]


def sample(logits: torch.Tensor, status: torch.Tensor, temperatures: torch.Tensor | None = None,
           uniforms: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Token ids (int32, on the device) from float32 logits [rows, vocab].

    Without ``temperatures`` every row is greedy; with them (float32 device tensors, one value per
    row, like ``uniforms``) a row is greedy where its temperature is 0 and drawn otherwise.  A
    non-finite logit sets a bit in the device ``status`` word instead of yielding a token."""
    if out is None:
        out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    kernels.sample(logits, out, status, temperatures, uniforms)
    return out


def verify(logits: torch.Tensor, drafts: torch.Tensor, row_start: torch.Tensor, status: torch.Tensor, draft_logits: torch.Tensor | None = None,
           temperatures: torch.Tensor | None = None, accept: torch.Tensor | None = None, draw: torch.Tensor | None = None):
    """Drafted tokens against the target's probabilities: ``(tokens, accepted)``, int32 on the device.

    ``tokens`` has a place per row of ``logits``: a request's drafts that stand, the token drawn after them, then -1 (so too in rows that are
    no request's); ``accepted`` says how many stand.  What is emitted is distributed as if drawn from the target alone, where the drafts were
    drawn from the draft model's distribution with numbers of their own (``draft_uniforms``), not with ``accept`` or ``draw``; a greedy request (temperature 0, or none given)
    gets the target's argmax at every place.  The arguments are those of ``kernels.verify_drafts`` (csrc/verify.cu), which this launches."""
    return kernels.verify_drafts(logits, drafts, row_start, status, draft_logits, temperatures, accept, draw)


__all__ = ["draft_uniforms", "sample", "uniform_for", "verify", "verify_uniforms"]
