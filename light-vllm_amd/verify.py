"""Verification of drafted tokens against the target model's probabilities.

light-vllm verifies draft trees greedily: a draft is accepted when it is the
target's most likely token (``GreedyTreeAcceptanceSampler``,
src/light_vllm/runtime/execution/speculative.py:220-257).  ``verify_drafts``
verifies them for sampled decoding: the tokens that come out follow the given
target probabilities, whatever was drafted.  It runs in the gfx950 kernels of
``liblvamd_hip.so`` on the device's probabilities; the random numbers are the
caller's.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch
from torch import Tensor

from light_vllm_amd import errors, native
from light_vllm_amd.interfaces import DraftTree
from light_vllm_amd.quantized_cache import _NOT_FAST, _raw_stream, on_device

_CODES = {torch.float32: native.DTYPE_F32, torch.float16: native.DTYPE_F16, torch.bfloat16: native.DTYPE_BF16}


class DraftBatch:
    """The draft trees of one step's requests, on the device.

    Made when the step is built (one upload), used by ``verify_drafts`` once the
    target's probabilities are there, on any stream that runs after the one it
    was made on.  It may be dropped after the call (a graph that captured such a
    call reads the batch's arrays: keep it as long).  A request without drafts has an empty
    tree.  Rows of probabilities are packed request by request: the root's (the
    distribution after the request's last formal token), then one per draft."""

    __slots__ = ("num_requests", "num_drafts", "num_rows", "path_width", "chains", "max_token", "counts", "device",
                 "_blob", "_stream", "_facts", "_verify")

    def __init__(self, drafts: Sequence[DraftTree], *, device: str | torch.device) -> None:
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise errors.ExecutionError("draft verification requires a GPU (cuda) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.counts = tuple(len(d) for d in drafts)
        arrays, self.chains, self.max_token = pack_drafts(drafts)
        self.num_requests = len(self.counts)
        self.num_drafts = sum(self.counts)
        self.num_rows = self.num_drafts + self.num_requests
        self.path_width = max((1, *self.counts))
        sizes = [a.size for a in arrays]
        blob = self._blob = torch.from_numpy(np.concatenate(arrays)).to(self.device)
        self._stream = _raw_stream(self.device.index)  # the allocator's, for the blob
        at = blob.data_ptr()
        # (Tokens first: int64, aligned.)
        tokens, starts, parents, siblings = (at + 4 * sum(sizes[:i]) for i in range(4))
        self._facts = (native.verify_entry(), self.device.index, self.num_rows, self.num_drafts, self.num_requests,
                       self.path_width, starts, tokens, parents, siblings, torch.float32, torch.float64, _raw_stream)
        self._verify = native.host().verify_tensors

    def __len__(self) -> int:
        return self.num_requests


def pack_drafts(drafts: Sequence[DraftTree]) -> tuple[list[np.ndarray], bool, int]:
    """int32 arrays [tokens as int64 pairs, first drafts per request, parents,
    earlier siblings], whether every tree is a chain, and the largest token."""

    starts, tokens, parents, siblings = [0], [], [], []
    chains, top = True, -1
    if not len(drafts):
        raise ValueError("draft verification needs at least one request")
    for tree in drafts:
        n = len(tree.token_ids)
        if n > native.VERIFY_MAX_DRAFTS:
            raise ValueError(f"draft verification takes at most {native.VERIFY_MAX_DRAFTS} drafts per request")
        last: dict[int, int] = {}
        for i, parent in enumerate(tree.parent_indices):
            siblings.append(last.get(parent, -1))
            last[parent] = i
            chains = chains and parent == i - 1
        parents.extend(tree.parent_indices)
        tokens.extend(tree.token_ids)
        starts.append(len(tokens))
        top = max((top, *tree.token_ids))
    if top >= 2**31:
        raise ValueError("draft tokens must be below 2**31")
    return [np.asarray(tokens, dtype=np.int64).view(np.int32), np.asarray(starts, dtype=np.int32),
            np.asarray(parents, dtype=np.int32), np.asarray(siblings, dtype=np.int32)], chains, top


@dataclass(frozen=True, slots=True)
class DraftVerdict:
    """What ``verify_drafts`` decided, on the device: per request how many drafts
    were accepted (int32), their indices in the tree, then -1 (int32
    ``[requests, longest tree]``), and the token that follows them (int64)."""

    counts: Tensor
    paths: Tensor
    tokens: Tensor

    def retained_query_indices(self, num_input_queries: Sequence[int]) -> tuple[tuple[int, ...], ...]:
        """Per request the query indices that ``compact`` keeps: the formal
        inputs, then the accepted path (light-vllm: speculative.py:399-401).
        Copies the verdict to the host."""

        counts, paths = self.counts.tolist(), self.paths.tolist()
        if len(num_input_queries) != len(counts):
            raise ValueError("num_input_queries needs one count per request")
        return tuple(tuple(range(n)) + tuple(n + i for i in path[:count])
                     for n, count, path in zip(num_input_queries, counts, paths))


def verify_drafts(batch: DraftBatch, target_probs: Tensor, node_uniforms: Tensor, sample_uniforms: Tensor, *,
                  draft_probs: Tensor | None = None) -> DraftVerdict:
    """Accept drafts and draw the token after them, on the current stream.

    ``target_probs`` ``[rows, vocab]`` (fp32, fp16 or bf16; any row stride): the
    target's probabilities at every node, packed as ``DraftBatch`` says.
    ``node_uniforms`` ``[rows]`` and ``sample_uniforms`` ``[requests]`` (fp32 or
    fp64): uniform numbers in [0, 1).  Without ``draft_probs`` the drafts are
    fixed tokens (an n-gram proposer's tree): at each node the children's
    probabilities are laid end to end, and the child whose interval holds the
    node's number is accepted.  With ``draft_probs`` ``[drafts, vocab]`` (the
    distribution that each draft was drawn from; chains only) draft x is accepted
    when u q(x) < p(x).  At the first node that accepts no child the request's
    token is drawn from what is left there: p without the children's tokens, or
    max(p - q, 0); p itself where nothing is left.  A row with no positive
    probability gives token -1.  Sums are in fp64.

    A probability that accepts a draft counts as given, the draw divides by the
    sum of what is left: where a row does not sum to one (by the rounding of fp16
    or bf16 rows, say), the tokens' distribution is off by as much.
    """

    vocab = target_probs.shape[1] if isinstance(target_probs, Tensor) and target_probs.ndim == 2 else 0
    code = _CODES.get(target_probs.dtype) if vocab else None
    if (code is None or vocab > 1 << 30 or batch.max_token >= vocab or batch.num_requests > 65535
            or (draft_probs is not None and not batch.chains)):
        _refuse(batch, target_probs, node_uniforms, sample_uniforms, draft_probs, vocab)
    n, device = batch.num_requests, batch.device
    with on_device(device):
        if _raw_stream(device.index) != batch._stream:
            # The caller may drop the batch while the kernels are pending: its
            # arrays are theirs until then.
            batch._blob.record_stream(torch.cuda.current_stream(device))
        counts = torch.empty(n, dtype=torch.int32, device=device)
        paths = torch.empty((n, batch.path_width), dtype=torch.int32, device=device)
        tokens = torch.empty(n, dtype=torch.int64, device=device)
        nbytes = native.load().lvamd_verify_drafts_workspace_size(n, batch.num_drafts, vocab, code)
        # (Of the call's own stream or graph: no two share one.)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        outputs = (counts.data_ptr(), paths.data_ptr(), tokens.data_ptr(), workspace.data_ptr(), nbytes)
        # One native call reads the tensors and launches when every rule holds.
        status = batch._verify(batch._facts, outputs, target_probs, node_uniforms, sample_uniforms, draft_probs, vocab,
                               target_probs.dtype, code)
        if status == _NOT_FAST:
            _refuse(batch, target_probs, node_uniforms, sample_uniforms, draft_probs, vocab)
            # Only the layout does not fit.
            rows = [t if t is None or t.stride(1) == 1 else t.contiguous() for t in (target_probs, draft_probs)]
            rows = [t if t is None or t.stride(1) == 1 else t.clone(memory_format=torch.contiguous_format) for t in rows]
            status = batch._verify(batch._facts, outputs, rows[0], node_uniforms.contiguous(),
                                   sample_uniforms.contiguous(), rows[1], vocab, target_probs.dtype, code)
        native.check(status, "lvamd_verify_drafts")
    return DraftVerdict(counts, paths, tokens)


def _refuse(batch: DraftBatch, target_probs, node_uniforms, sample_uniforms, draft_probs, vocab: int) -> None:
    """Raise the first broken rule's message."""

    def shape(t, *want) -> bool:
        return isinstance(t, Tensor) and tuple(t.shape) == want

    both = [target_probs] if draft_probs is None else [target_probs, draft_probs]
    rules = (
        (lambda: 0 < vocab <= 1 << 30 and shape(target_probs, batch.num_rows, vocab),
         f"target probabilities must have shape [{batch.num_rows}, vocab]"),
        (lambda: draft_probs is None or shape(draft_probs, batch.num_drafts, vocab),
         f"draft probabilities must have shape [{batch.num_drafts}, vocab]"),
        (lambda: draft_probs is None or batch.chains, "draft probabilities need chains of drafts, not trees"),
        (lambda: all(t.dtype in _CODES and t.dtype == target_probs.dtype for t in both),
         "probabilities must be float32, float16 or bfloat16, all of one dtype"),
        (lambda: shape(node_uniforms, batch.num_rows), f"node uniforms must have shape [{batch.num_rows}]"),
        (lambda: shape(sample_uniforms, batch.num_requests), f"sample uniforms must have shape [{batch.num_requests}]"),
        (lambda: node_uniforms.dtype == sample_uniforms.dtype and node_uniforms.dtype in (torch.float32, torch.float64),
         "uniforms must be float32 or float64, both of one dtype"),
        (lambda: all(t.device == batch.device for t in (*both, node_uniforms, sample_uniforms)),
         "probabilities and uniforms must be on the draft batch's device"),
        (lambda: batch.max_token < vocab, "a draft token lies outside the vocabulary"),
        (lambda: batch.num_requests <= 65535, "draft verification takes at most 65535 requests"),
    )
    for holds, message in rules:
        if not holds():
            raise ValueError(message)
