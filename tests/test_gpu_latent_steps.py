"""GPU: steps over the latent cache whose layers take several forms."""

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
