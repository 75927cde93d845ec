"""GPU: steps over the latent cache whose layers take several forms, and what a step
allocates."""

from __future__ import annotations

import pytest
import torch

import light_vllm_amd as lv
import test_gpu_latent as latent_space
import test_gpu_latent_layer as layer

pytestmark = pytest.mark.gpu

DEV, TREE = layer.DEV, layer.TREE


def _two_forms(second):
    """A cache of two layers, a step's metadata (anew at each call) and what runs it:
    layer 0 with weights of 128 + 128, layer 1 by ``second``."""
    cache, md, q, latent, rope_key, rotary, up = layer._step(4, 256, 64, 128, 128, 16, torch.bfloat16, [300, 40], [1, 5], seed=3)
    spec = lv.LatentKVCacheSpec(tuple(lv.LatentLayerSpec(f"layer{i}", 4, 256, 64) for i in range(2)))
    both = lv.LatentPagedKVCache(spec, cache.config)
    for i in range(2):
        both.layer(f"layer{i}").rows.copy_(cache.layer("layer0").rows)
    gen = torch.Generator(device=DEV).manual_seed(4)
    weights = lv.LatentWeights(*up)
    if second == "none":
        other, size = None, 256
    else:
        other, size = lv.LatentWeights(up[0][:, :64], up[1][:, :64]), 64
    q1 = torch.randn((6, 4, size + 64), generator=gen, device=DEV).to(torch.bfloat16)

    def metadata():
        return lv.PagedAttentionMetadata(block_tables=md.block_tables, num_computed_tokens=md.num_computed_tokens,
                                         query_layouts=md.query_layouts)

    def run(context):
        return [context.forward("layer0", q, latent, rope_key, scale=0.07, rotary=rotary, weights=weights),
                context.forward("layer1", q1, latent, rope_key, scale=0.07, rotary=rotary, weights=other)]

    return both, metadata, run


@pytest.mark.parametrize("second", ("none", "64"))
def test_a_cache_whose_layers_take_two_forms(second) -> None:
    """From its second step on, everything is planned and uploaded by create()."""
    latent_space._say(f"latent layers of two forms, {second}")
    cache, metadata, run = _two_forms(second)
    backend = lv.HipPagedAttentionBackend()
    want = run(backend.create(cache, metadata()))
    for _ in range(3):
        context = backend.create(cache, metadata())
        got = run(context)
        assert context.plan._late_blobs == []
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("second", ("none", "64"))
def test_a_step_of_two_forms_is_captured(second) -> None:
    latent_space._say(f"latent layers of two forms captured, {second}")
    cache, metadata, run = _two_forms(second)
    backend = lv.HipPagedAttentionBackend()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = run(backend.create(cache, metadata()))
    torch.cuda.current_stream().wait_stream(stream)
    context, graph = backend.create(cache, metadata()), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(context)
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        eager = run(backend.create(cache, metadata()))
        torch.cuda.synchronize()
        for a, b, c in zip(got, eager, want):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_a_plan_of_another_caches_layers_is_not_taken() -> None:
    """The same metadata on a cache of the same pool and other layers: its own forms are
    planned by create(), and captured."""
    latent_space._say("latent layers of another cache, the same metadata")
    cache, metadata, run = _two_forms("64")
    one = layer._step(2, 128, 32, 64, 64, 16, torch.bfloat16, [300, 40], [1, 5], seed=3)
    other = lv.LatentPagedKVCache(one[0].model_spec, cache.config)
    weights, backend = lv.LatentWeights(*one[6]), lv.HipPagedAttentionBackend()
    run_other = lambda c: c.forward("layer0", *one[2:5], scale=0.07, weights=weights)  # noqa: E731
    want, want_other = run(backend.create(cache, metadata())), run_other(backend.create(other, metadata()))
    md = metadata()
    run(backend.create(cache, md))
    context = backend.create(other, md)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run_other(context)
    graph.replay()
    again = run(backend.create(cache, md))
    torch.cuda.synchronize()
    assert torch.equal(out, want_other) and all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("known", (False, True))
def test_a_plan_whose_upload_is_pending_on_another_stream(known) -> None:
    """Two streams create contexts for the same metadata: the second waits for the lists
    that the first uploads."""
    latent_space._say(f"latent layers, lists pending on another stream, form known: {known}")
    cache, metadata, run = _two_forms("none")
    want = run(lv.HipPagedAttentionBackend().create(cache, metadata()))
    backend, md = lv.HipPagedAttentionBackend(), metadata()
    if known:
        run(backend.create(cache, metadata()))
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        torch.cuda._sleep(50_000_000)
        kept = backend.create(cache, md)
    with torch.cuda.stream(second):
        context = backend.create(cache, md)
        got = run(context)
    assert context.plan is kept.plan
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_short_requests_around_a_long_one_take_memory_for_themselves(monkeypatch) -> None:
    """Two decoding requests of 128 heads with a chunk of 8192 tokens between them: no
    scratch for the chunk's rows in latent space (2.1 GB)."""
    latent_space._say("latent layer, memory of short requests around a chunk")
    layer._force(monkeypatch, lambda n, linear: n >= 200)
    heads, chunk = 128, 8192
    cache, md, q, latent, rope_key, _, up = layer._step(heads, 512, 64, 128, 128, 16, torch.bfloat16, [40, 0, 90], [1, chunk, 2],
                                                        seed=3)
    weights, backend = lv.LatentWeights(*up), lv.HipPagedAttentionBackend()
    run = lambda: backend.create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07, weights=weights)  # noqa: E731
    want = run()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = run()
    torch.cuda.synchronize()
    took = torch.cuda.max_memory_allocated() - before
    result, expanded = q.shape[0] * heads * 128 * 2, chunk * heads * (128 + 128) * 2 + chunk * 64 * 2
    assert took < result + expanded + (64 << 20)  # (and the splits' partials, the short requests' own)
    assert torch.equal(got, want)


@pytest.mark.parametrize("expanded", (False, True))
def test_short_requests_anywhere_in_the_step(expanded, monkeypatch) -> None:
    """Short requests first, last, on both sides of long ones and alone: rows in latent
    space are theirs alone, tokens the step's."""
    latent_space._say(f"latent layer, places of short requests, expanded={expanded}")
    layer._force(monkeypatch, lambda n, linear: (n >= 70) & linear & expanded)
    for layouts in ([1, 80], [80, 1], [1, 80, TREE], [80, 3, 90], [2, 80, 1, 90, 1], [80, 1, TREE, 3, 70]):
        computed = [(37 * i) % 130 for i in range(len(layouts))]
        for rotary in (False, True):
            layer._run(layer._step(5, 256, 64, 64, 128, 16, torch.bfloat16, computed, layouts, seed=len(layouts)), rotary=rotary)


def test_uploads_are_not_captured() -> None:
    """What a replay would read from a reused staging buffer is refused: a context that
    is created inside a capture, moves of more tokens or blocks than a launch's arguments
    hold.  Fewer are captured and replay."""
    latent_space._say("latent steps, uploads in a capture")
    cache, metadata, run = _two_forms("none")
    backend = lv.HipPagedAttentionBackend()
    want = run(backend.create(cache, metadata()))
    wide = lv.LatentPagedKVCache(cache.model_spec, lv.PagedKVCacheConfig(num_blocks=80, block_size=16, dtype=torch.bfloat16,
                                                                         device=DEV))
    wide.copy_blocks([0], [1])  # (its table of layers is made at the first move)
    few = 32
    kept = tuple(range(2, 2 + few + 1))
    request = dict(block_ids=(0, 1, 2, 3), num_computed_tokens=10, num_query_tokens=40, num_reserved_query_tokens=40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(lv.ExecutionError, match="before the capture"):
            backend.create(cache, metadata())
        with pytest.raises(lv.ExecutionError, match="at most 32"):
            wide.copy_blocks(list(range(few + 1)), list(range(40, 40 + few + 1)))
        with pytest.raises(lv.ExecutionError, match="at most 32"):
            wide.compact(**request, retained_query_indices=kept)
        wide.copy_blocks(list(range(few)), list(range(40, 40 + few)))
        assert wide.compact(**request, retained_query_indices=kept[:few]) == few
    gen = torch.Generator(device=DEV).manual_seed(6)
    for _ in range(3):
        expect = {}
        for name in ("layer0", "layer1"):
            rows = wide.layer(name).rows
            rows.normal_(generator=gen)
            expect[name] = rows.clone()
            expect[name][40:40 + few] = rows[:few]
            flat = expect[name].view(-1, rows.shape[-1])
            flat[10:10 + few] = flat[12:12 + few].clone()
        graph.replay()
        got = run(backend.create(cache, metadata()))
        torch.cuda.synchronize()
        assert all(torch.equal(wide.layer(name).rows, x) for name, x in expect.items())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_framework_s_functions_move_latent_rows() -> None:
    """``hip_compact`` and ``hip_compact_many`` do what the cache's own methods do."""
    latent_space._say("latent compact through the functions")
    gen = torch.Generator(device=DEV).manual_seed(5)
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec("a", 4, 256, 64), lv.LatentLayerSpec("b", 4, 128, 32)))
    caches = [lv.LatentPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=12, block_size=8, dtype=torch.bfloat16, device=DEV))
              for _ in range(3)]
    for name in ("a", "b"):
        rows = caches[0].layer(name).rows
        rows.normal_(generator=gen)
        for cache in caches[1:]:
            cache.layer(name).rows.copy_(rows)
    requests = [dict(block_ids=(5, 2, 9), num_computed_tokens=11, num_query_tokens=9, num_reserved_query_tokens=9,
                     retained_query_indices=(0, 3, 4, 8)),
                dict(block_ids=(1, 7), num_computed_tokens=3, num_query_tokens=7, num_reserved_query_tokens=7,
                     retained_query_indices=(6, 1))]
    want = tuple(caches[0].compact(**r) for r in requests)
    assert lv.paged_cache.hip_compact_many(caches[1], requests) == want == (3, 1)
    assert tuple(lv.hip_compact(caches[2], **r) for r in requests) == want
    for cache in caches[1:]:
        assert all(torch.equal(cache.layer(name).rows, caches[0].layer(name).rows) for name in ("a", "b"))
