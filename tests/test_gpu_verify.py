"""GPU: ``verify_drafts`` against the fp64 oracle, decision for decision: trees
without draft probabilities and chains with them, every type, odd and small
vocabularies, strided rows, rows that leave nothing, and the numbers at the
ends of their range."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
from oracle import quantized_oracle as Q

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

DEV = torch.device("cuda:0")


def _trees(rng, sizes, vocab, chain):
    trees = []
    for n in sizes:
        parents = tuple(i - 1 if chain else int(rng.integers(-1, i)) if i else -1 for i in range(n))
        used, tokens = {}, []
        for p in parents:
            free = [t for t in rng.permutation(vocab)[:n + 1].tolist() if t not in used.get(p, ())]
            tokens.append(int(free[0]))
            used.setdefault(p, set()).add(tokens[-1])
        trees.append(lv.DraftTree(tuple(tokens), parents))
    return trees


def _probs(gen, rows, vocab, dtype, trees=None, weight=0.0):
    """Peaked rows; with trees, drafts get `weight` more mass at their parents."""
    x = (torch.randn((rows, vocab), generator=gen, device=DEV) * 2).softmax(dim=-1)
    if trees is not None:
        row = 0
        for t in trees:
            for token, parent in zip(t.token_ids, t.parent_indices):
                x[row + parent + 1, token] += weight
            row += len(t) + 1
    return (x / x.sum(dim=-1, keepdim=True)).to(dtype)


def _compare(trees, target, node, sample, verdict, draft_probs=None):
    counts, paths, tokens = (t.tolist() for t in (verdict.counts, verdict.paths, verdict.tokens))
    width = max((1, *map(len, trees)))
    row = first = 0
    for r, t in enumerate(trees):
        n = len(t)
        q = None if draft_probs is None else draft_probs[first : first + n].double().cpu().numpy()
        path, token = Q.verify(t.parent_indices, t.token_ids, target[row : row + n + 1].double().cpu().numpy(),
                               node[row : row + n + 1].double().tolist(), float(sample[r].double()), q)
        assert (counts[r], paths[r], tokens[r]) == (len(path), path + [-1] * (width - len(path)), token), r
        row, first = row + n + 1, first + n


@pytest.mark.parametrize("chain", (True, False), ids=("chain", "tree"))
@pytest.mark.parametrize("vocab,dtype,uniforms", [
    (32000, torch.float32, torch.float32), (151936, torch.float32, torch.float64), (100003, torch.bfloat16, torch.float32),
    (257, torch.float16, torch.float64), (37, torch.float32, torch.float32), (5000, torch.float16, torch.float32)])
def test_matches_the_oracle(vocab, dtype, uniforms, chain) -> None:
    rng = np.random.default_rng(vocab)
    for sizes in ([4], [0], [3, 0, 8, 1, 12, 5], [int(n) for n in rng.integers(0, 9, 70)] if vocab < 6000 else [2, 2]):
        print(f"[gpu] verify vocab {vocab} {dtype} chain={chain} {len(sizes)} requests", file=sys.stderr, flush=True)
        trees = _trees(rng, sizes, vocab, chain)
        batch = lv.DraftBatch(trees, device=DEV)
        gen = torch.Generator(device=DEV).manual_seed(vocab + len(sizes))
        target = _probs(gen, batch.num_rows, vocab, dtype, trees, 0.5)
        drafts = _probs(gen, batch.num_drafts, vocab, dtype) if chain else None
        node, sample = (torch.rand(n, generator=gen, device=DEV, dtype=uniforms) for n in (batch.num_rows, len(sizes)))
        verdict = lv.verify_drafts(batch, target, node, sample, draft_probs=drafts)
        _compare(trees, target, node, sample, verdict, drafts)


def test_vocabularies_of_a_few_tokens() -> None:
    rng = np.random.default_rng(1)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for vocab in (1, 2, 3, 7, 8, 9):
        print(f"[gpu] verify vocab {vocab}", file=sys.stderr, flush=True)
        trees = [lv.DraftTree((vocab - 1,), (-1,)), lv.DraftTree((), ()), lv.DraftTree((0,) * 5, tuple(range(-1, 4)))]
        batch = lv.DraftBatch(trees, device=DEV)
        for dtype in (torch.float32, torch.bfloat16):
            target, drafts = (_probs(gen, n, vocab, dtype) for n in (batch.num_rows, batch.num_drafts))
            node, sample = (torch.rand(n, generator=gen, device=DEV) for n in (batch.num_rows, 3))
            for q in (None, drafts):
                _compare(trees, target, node, sample, lv.verify_drafts(batch, target, node, sample, draft_probs=q), q)


@pytest.mark.parametrize("vocab,dtype", [(600001, torch.float32), (1200007, torch.bfloat16)])
def test_rows_of_many_chunks(vocab, dtype) -> None:
    """More chunks than the draw holds in registers; draws all along the row."""
    print(f"[gpu] verify vocab {vocab} {dtype}", file=sys.stderr, flush=True)
    rng = np.random.default_rng(vocab)
    gen = torch.Generator(device=DEV).manual_seed(vocab)
    trees = _trees(rng, [2, 0, 1, 0], vocab, True)
    batch = lv.DraftBatch(trees, device=DEV)
    target, drafts = (_probs(gen, n, vocab, dtype) for n in (batch.num_rows, batch.num_drafts))
    node = torch.rand(batch.num_rows, generator=gen, device=DEV, dtype=torch.float64)
    for values in ((0.05, 0.3, 0.55, 0.8), (0.45, 0.9, 0.99, 0.9999)):
        sample = torch.tensor(values, device=DEV, dtype=torch.float64)
        for q in (None, drafts):
            _compare(trees, target, node, sample, lv.verify_drafts(batch, target, node, sample, draft_probs=q), q)


def test_many_requests() -> None:
    print("[gpu] verify 5000 requests", file=sys.stderr, flush=True)
    rng = np.random.default_rng(9)
    gen = torch.Generator(device=DEV).manual_seed(9)
    trees = _trees(rng, [int(n) for n in rng.integers(0, 4, 5000)], 2100, False)
    batch = lv.DraftBatch(trees, device=DEV)
    target = _probs(gen, batch.num_rows, 2100, torch.bfloat16, trees, 0.3)
    node, sample = (torch.rand(n, generator=gen, device=DEV) for n in (batch.num_rows, 5000))
    verdict = lv.verify_drafts(batch, target, node, sample)
    _compare(trees, target, node, sample, verdict)


def test_strided_rows() -> None:
    print("[gpu] verify strided rows", file=sys.stderr, flush=True)
    rng = np.random.default_rng(2)
    gen = torch.Generator(device=DEV).manual_seed(2)
    trees = _trees(rng, [3, 5], 1001, True)
    batch = lv.DraftBatch(trees, device=DEV)
    wide = _probs(gen, 2 * batch.num_rows, 1003, torch.bfloat16)
    target, drafts = wide[::2, 1:1002], _probs(gen, 1001, batch.num_drafts, torch.bfloat16).t()
    node, sample = torch.rand(2 * batch.num_rows, generator=gen, device=DEV)[::2], torch.rand(2, generator=gen, device=DEV)
    for q in (None, drafts):
        _compare(trees, target, node, sample, lv.verify_drafts(batch, target, node, sample, draft_probs=q), q)


def test_one_request_with_strided_uniforms() -> None:
    """Vectors of one element keep their stride through ``contiguous()``."""
    print("[gpu] verify one request, strided uniforms", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(12)
    for uniforms in (torch.float32, torch.float64):
        for tree in (lv.DraftTree((5, 9), (-1, -1)), lv.DraftTree((), ())):
            batch = lv.DraftBatch([tree], device=DEV)
            target = _probs(gen, batch.num_rows, 33, torch.float32, [tree], 0.3)
            node = torch.rand((batch.num_rows, 4), generator=gen, device=DEV, dtype=uniforms)[:, 1]
            sample = torch.rand((1, 4), generator=gen, device=DEV, dtype=uniforms)[:, 2]
            assert sample.stride() == (4,)
            _compare([tree], target, node, sample, lv.verify_drafts(batch, target, node, sample))


def test_siblings_intervals_meet() -> None:
    """Numbers on the borders between siblings and one step beside them, where the
    sums of their probabilities round: each lies in one interval."""
    print("[gpu] verify borders of siblings", file=sys.stderr, flush=True)
    rng = np.random.default_rng(13)
    k, requests = 6, 2000
    trees = [lv.DraftTree(tuple(range(k)), (-1,) * k)] * requests
    batch = lv.DraftBatch(trees, device=DEV)
    probs = (rng.uniform(1, 2, (requests, k)) * np.exp2(-rng.integers(3, 45, (requests, k)))).astype(np.float32)
    target = torch.zeros((requests, k + 1, k + 2), device=DEV)
    target[:, 0, :k] = torch.from_numpy(probs).to(DEV)
    target[..., k] = 0.25
    target = target.view(-1, k + 2)
    borders = np.cumsum(probs.astype(np.float64), axis=1)
    sample = torch.full((requests,), 0.5, dtype=torch.float64, device=DEV)
    for j in range(k):
        for u in (borders[:, j], np.nextafter(borders[:, j], 0.0), np.nextafter(borders[:, j], 1.0)):
            node = torch.zeros((requests, k + 1), dtype=torch.float64)
            node[:, 0] = torch.from_numpy(u)
            node = node.view(-1).to(DEV)
            _compare(trees, target, node, sample, lv.verify_drafts(batch, target, node, sample))


def test_rows_that_leave_nothing() -> None:
    print("[gpu] verify empty residuals", file=sys.stderr, flush=True)
    vocab = 300
    trees = [lv.DraftTree((7,), (-1,))] * 5
    batch = lv.DraftBatch(trees, device=DEV)
    target = torch.zeros((10, vocab), device=DEV)
    drafts = torch.zeros((5, vocab), device=DEV)
    target[0, 7] = drafts[0, 7] = 1.0     # accepted, and the leaf's row is all zero: nothing to draw
    target[2, 7], drafts[1, 7] = 0.5, 1.0   # rejected, p <= q everywhere: drawn from p
    target[4] = float("nan")                # no row at all
    target[6, 3], target[6, 5], target[6, 9] = float("inf"), -1.0, 0.25  # entries that do not count
    target[8, 299] = 1e-30
    node, sample = torch.full((10,), 0.75, device=DEV), torch.full((5,), 0.5, device=DEV)
    for q in (None, drafts):
        verdict = lv.verify_drafts(batch, target, node, sample, draft_probs=q)
        _compare(trees, target, node, sample, verdict, q)
        assert verdict.tokens.tolist() == [-1, 7, -1, 9, 299]


def test_numbers_at_the_ends_of_their_range() -> None:
    print("[gpu] verify uniforms 0 and 1", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(4)
    trees = _trees(np.random.default_rng(4), [3] * 6, 50, False)
    batch = lv.DraftBatch(trees, device=DEV)
    target = _probs(gen, batch.num_rows, 50, torch.float32, trees, 0.3)
    target[:, :2] = 0
    target[:, 48:] = 0
    for value in (0.0, 1.0 - 2.0**-24, 1.0):
        node, sample = torch.full((batch.num_rows,), value, device=DEV), torch.full((6,), value, device=DEV)
        _compare(trees, target, node, sample, lv.verify_drafts(batch, target, node, sample))


def test_the_longest_tree() -> None:
    print("[gpu] verify 1024 drafts", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(5)
    trees = [lv.DraftTree(tuple(range(1024)), tuple(range(-1, 1023))),          # all accepted
             lv.DraftTree(tuple(range(1024)), (-1,) * 1024)]                     # siblings
    batch = lv.DraftBatch(trees, device=DEV)
    target = torch.full((batch.num_rows, 1100), 1.0 / 1100, device=DEV)
    target[torch.arange(1024), torch.arange(1024)] = 2.0
    node = torch.rand(batch.num_rows, generator=gen, device=DEV)
    node[1025] = 0.9
    sample = torch.rand(2, generator=gen, device=DEV)
    verdict = lv.verify_drafts(batch, target, node, sample)
    _compare(trees, target, node, sample, verdict)
    assert verdict.counts.tolist() == [1024, 1]
    assert verdict.retained_query_indices([2, 1])[0] == tuple(range(1026))
    with pytest.raises(ValueError, match="one count per request"):
        verdict.retained_query_indices([1])


def test_captured_and_on_another_stream() -> None:
    print("[gpu] verify in a graph and on a stream", file=sys.stderr, flush=True)
    rng = np.random.default_rng(6)
    gen = torch.Generator(device=DEV).manual_seed(6)
    trees = _trees(rng, [4, 2, 6], 30001, True)
    batch = lv.DraftBatch(trees, device=DEV)
    target, drafts = _probs(gen, batch.num_rows, 30001, torch.float32, trees, 0.4), _probs(gen, batch.num_drafts, 30001, torch.float32)
    node, sample = torch.rand(batch.num_rows, generator=gen, device=DEV), torch.rand(3, generator=gen, device=DEV)
    lv.verify_drafts(batch, target, node, sample, draft_probs=drafts)
    torch.cuda.synchronize()
    graphs, captured = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g, q in zip(graphs, (drafts, None)):
        with torch.cuda.graph(g):
            captured.append(lv.verify_drafts(batch, target, node, sample, draft_probs=q))
    stream = torch.cuda.Stream()
    for i in range(4):
        target.copy_(_probs(gen, batch.num_rows, 30001, torch.float32, trees, 0.4))
        for t in (node, sample):
            t.uniform_(generator=gen)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for q, verdict in zip((drafts, None), captured):
            _compare(trees, target, node, sample, verdict, q)
        with torch.cuda.stream(stream):
            _compare(trees, target, node, sample, lv.verify_drafts(batch, target, node, sample, draft_probs=drafts), drafts)


def test_a_batch_dropped_behind_another_stream() -> None:
    """The batch's arrays stay its own until a pending call on another stream has
    read them: a tensor that asks for their memory meanwhile gets other memory."""
    print("[gpu] verify, the batch dropped at once", file=sys.stderr, flush=True)
    rng = np.random.default_rng(14)
    gen = torch.Generator(device=DEV).manual_seed(14)
    trees = _trees(rng, [5, 0, 7, 3], 1000, True)
    batch = lv.DraftBatch(trees, device=DEV)
    target = _probs(gen, batch.num_rows, 1000, torch.float32, trees, 0.6)
    node, sample = torch.rand(batch.num_rows, generator=gen, device=DEV), torch.rand(4, generator=gen, device=DEV)
    stream, blob = torch.cuda.Stream(), batch._blob
    at, nbytes = blob.data_ptr(), 4 * blob.numel()
    del blob
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(50_000_000)
        verdict = lv.verify_drafts(batch, target, node, sample)
    del batch
    others = [torch.zeros(nbytes, dtype=torch.uint8, device=DEV) for _ in range(4)]
    assert at not in [t.data_ptr() for t in others]
    torch.cuda.synchronize()
    _compare(trees, target, node, sample, verdict)


def test_refusals() -> None:
    batch = lv.DraftBatch([lv.DraftTree((5, 6), (-1, -1)), lv.DraftTree((), ())], device=DEV)
    assert len(batch) == 2 and batch.num_rows == 4 and not batch.chains
    good = dict(target_probs=torch.ones((4, 10), device=DEV), node_uniforms=torch.ones(4, device=DEV),
                sample_uniforms=torch.ones(2, device=DEV))
    lv.verify_drafts(batch, **good)
    for bad, message in (
        (dict(target_probs=torch.ones((3, 10), device=DEV)), "target probabilities"),
        (dict(target_probs=torch.ones((4, 0), device=DEV)), "target probabilities"),
        (dict(target_probs=torch.ones((4, 10), device=DEV).double()), "float32, float16 or bfloat16"),
        (dict(target_probs=torch.ones((4, 10))), "on the draft batch's device"),
        (dict(target_probs=torch.ones((4, 6), device=DEV)), "outside the vocabulary"),
        (dict(node_uniforms=torch.ones(3, device=DEV)), "node uniforms"),
        (dict(sample_uniforms=torch.ones(3, device=DEV)), "sample uniforms"),
        (dict(sample_uniforms=torch.ones(2, device=DEV).double()), "both of one dtype"),
        (dict(draft_probs=torch.ones((3, 10), device=DEV)), "draft probabilities"),
        (dict(draft_probs=torch.ones((2, 10), device=DEV)), "chains"),
    ):
        with pytest.raises(ValueError, match=message):
            lv.verify_drafts(batch, **{**good, **bad})
    chain = lv.DraftBatch([lv.DraftTree((5,), (-1,))], device=DEV)
    with pytest.raises(ValueError, match="one dtype"):
        lv.verify_drafts(chain, torch.ones((2, 10), device=DEV), torch.ones(2, device=DEV), torch.ones(1, device=DEV),
                         draft_probs=torch.ones((1, 10), device=DEV).half())
