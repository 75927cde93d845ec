"""GPU: a backend that is dropped while its step's upload still waits on a busy
stream: the pinned buffer must not go to the next backend before it was read.

Both steps read the same pool through tables of their own, so a mixed-up upload
gives the other step's result, never an address out of range."""

from __future__ import annotations

import sys

import pytest
import torch

import light_vllm_amd as lv
from light_vllm_amd.plan import Staging

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

DEV = torch.device("cuda:0")


def test_dropped_backends_uploads_arrive_whole() -> None:
    print("[gpu] uploads of dropped backends", file=sys.stderr, flush=True)
    spec = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("a", 4, 2, 64),))
    cache = lv.PagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=64, block_size=16, dtype=torch.bfloat16, device=DEV))
    for pool in (cache.layer("a").keys, cache.layer("a").values):
        pool.normal_()
    q = torch.randn((1, 4, 64), device=DEV).to(torch.bfloat16)
    k, v = (torch.randn((1, 2, 64), device=DEV).to(torch.bfloat16) for _ in range(2))
    tables = [tuple(range(8 * i, 8 * i + 8)) for i in range(8)]
    steps = [lv.PagedAttentionMetadata(block_tables=(t,), num_computed_tokens=(100 + i,),
                                       query_layouts=(lv.linear_query_layout(1),), num_reserved_query_tokens=(28 - i,))
             for i, t in enumerate(tables)]
    want = []
    for md in steps:
        want.append(lv.HipPagedAttentionBackend().create(cache, md).forward("a", q, k, v, scale=0.125))
        torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)  # the uploads below wait behind this
    got = [lv.HipPagedAttentionBackend().create(cache, md).forward("a", q, k, v, scale=0.125) for md in steps]
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


def test_a_dropped_staging_ring_has_finished_its_copies() -> None:
    print("[gpu] a dropped staging ring", file=sys.stderr, flush=True)
    ring = Staging(DEV)
    torch.cuda._sleep(20_000_000)
    buf = ring.buffer(1024)
    buf[:] = 7
    dev = ring.upload(buf)
    event = ring._events[ring._slot]
    del ring, buf
    assert event.query()  # waited for
    assert bool((dev == 7).all())


def test_a_ring_dropped_in_a_capture_leaves_it_whole() -> None:
    print("[gpu] a staging ring dropped while a graph is captured", file=sys.stderr, flush=True)
    from light_vllm_amd import plan

    ring = Staging(DEV)
    buf = ring.buffer(1024)
    buf[:] = 7
    dev = ring.upload(buf).float()
    del buf
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        twice = dev * 2
        del ring
        out = twice + 1
    assert len(plan._LEFT) == 1
    for i in range(3):
        dev.fill_(float(i))
        graph.replay()
        torch.cuda.synchronize()
        assert bool((out == 2.0 * i + 1).all())
    Staging(DEV).buffer(16)  # the next ring's first use frees it
    assert not plan._LEFT
