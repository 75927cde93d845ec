"""GPU: attention over the latent cache where numbers end."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
import test_gpu_latent as latent_space
import test_gpu_latent_layer as layer
from light_vllm_amd import latent_attention, native

pytestmark = pytest.mark.gpu

DEV, TREE = layer.DEV, layer.TREE
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- a query all of whose scores are -inf: its softmax is NaN in every value ----------

@pytest.mark.parametrize("split", (False, True))
@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("heads, computed, layouts", [(16, [0, 40], [1, 3]), (5, [0, 1200], [TREE, 2]), (128, [70, 0], [1, 9])])
def test_scores_that_are_all_minus_infinity(heads, computed, layouts, dtype, wide, split, monkeypatch) -> None:
    """Some (query, head) rows hold -inf where every key is positive.  ``split``:
    each request's tiles go to many workgroups and are merged."""
    if wide:
        monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
    if split:
        computed = [c + 3000 for c in computed]
    latent_space._say(f"latent attention, scores of -inf, {heads} heads {computed} {dtype} wide={wide}")
    cache, md, q, latent, rope_key = latent_space._step(heads, 256, 64, 16, DTYPES[dtype], computed, layouts, seed=heads)
    flat = latent_space._flat(cache)
    flat[:, 3] = flat[:, 3].abs() + 0.5  # (NaN stays where no token is)
    latent = latent.clone()
    latent[:, 3] = latent[:, 3].abs() + 0.5
    q = q.clone()
    gone = [(0, 0), (q.shape[0] - 1, heads - 1), (q.shape[0] // 2, heads // 2)]
    for t, h in gone:
        q[t, h, 3] = -math.inf
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07)
    want, bound = latent_space._expected(cache, md, q, None, 0.07)
    nan = np.isnan(want).all(axis=2)
    assert sorted(set(gone)) == sorted(map(tuple, np.argwhere(nan).tolist())) and not np.isnan(want[~nan]).any()
    latent_space._check(out, want, bound, "scores of -inf")


@pytest.mark.parametrize("value", (math.inf, -math.inf))
@pytest.mark.parametrize("heads", (3, 40))
def test_a_first_token_whose_latent_is_infinite(heads, value) -> None:
    """One key, one score of either infinity or neither: NaN in every value."""
    latent_space._say(f"latent attention, a first token's latent holds {value}")
    cache, md, q, latent, rope_key = latent_space._step(heads, 256, 64, 16, torch.bfloat16, [0, 0, 50], [1, 4, 1], seed=3)
    latent = latent.clone()
    latent[0, 3] = value
    latent[1, 5] = value
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07)
    got = latent_space._np(out)
    assert np.isnan(got[:2]).all() and np.isfinite(got[5]).all()
    # (The second request's later queries have finite scores beside that one.)
    latent_space._check(out, *latent_space._expected(cache, md, q, None, 0.07), "an infinite latent")


@pytest.mark.parametrize("split", (False, True))
@pytest.mark.parametrize("expanded", (False, True))
@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
def test_scores_that_are_all_minus_infinity_with_weights(dtype, expanded, split, monkeypatch) -> None:
    latent_space._say(f"latent layer, scores of -inf, {dtype} expanded={expanded} split={split}")
    layer._force(monkeypatch, lambda n, linear: (n > 0) & expanded)
    computed, layouts = ([0, 33], [150, 70]) if not split else ([4000], [140])
    cache, md, q, latent, rope_key, _, up = layer._step(3, 256, 64, 64, 128, 16, DTYPES[dtype], computed, layouts, seed=5)
    flat = cache.layer("layer0").rows.view(-1, 320)
    flat[:, 300] = flat[:, 300].abs() + 0.5
    rope_key = rope_key.clone()
    rope_key[:, 300 - 256] = rope_key[:, 300 - 256].abs() + 0.5
    gone = [(0, 2), (131, 0), (q.shape[0] - 1, 1)]
    for t, h in gone:
        q[t, h, 64 + 300 - 256] = -math.inf
    context = lv.HipPagedAttentionBackend().create(cache, md)
    out = context.forward("layer0", q, latent, rope_key, scale=0.07, weights=lv.LatentWeights(*up))
    if split and expanded:
        assert any(shape.num_unit_jobs > 0 for shape in context.plan.launches.values())
    want, bound = layer._expected(cache, md, q, None, up, 0.07)
    nan = np.isnan(want).all(axis=2)
    assert sorted(gone) == sorted(map(tuple, np.argwhere(nan).tolist())) and not np.isnan(want[~nan]).any()
    layer._check(out, want, bound, "scores of -inf")


# ---- a chunk's keys or values past the type's largest ----------------------------------

@pytest.mark.parametrize("dtype, large", [("fp16", 60000.0), ("bf16", 3e38)])
@pytest.mark.parametrize("of", ("keys", "values"))
def test_a_chunks_keys_and_values_past_the_largest(of, dtype, large, monkeypatch) -> None:
    """A token whose key or value of one head is not representable: the queries that
    see it get NaN from that head, in every value; other queries and heads do not know
    of it."""
    latent_space._say(f"latent layer, {of} past {dtype}'s largest")
    layer._force(monkeypatch, lambda n, linear: n >= 200)
    t = DTYPES[dtype]
    cache, md, q, latent, rope_key, _, up = layer._step(4, 128, 32, 64, 64, 16, t, [20, 3], [300, 2], seed=6)
    # Head 1's key (value) of token 250 is the sum of magnitudes in one place; elsewhere
    # and for the other heads the weights are so small that nothing comes near.
    up = [w * 2.0**-12 for w in up]
    which = 0 if of == "keys" else 1
    up[which][1, 3] = torch.sign(up[which][1, 3]) * 0.5
    latent[250] = large * torch.sign(up[which][1, 3].float()).to(t)
    largest = torch.finfo(t).max
    per_head = [np.abs(latent_space._np(latent[250]) @ latent_space._np(w).transpose(0, 2, 1)).max(axis=1) for w in up]
    assert per_head[which][1] > 2 * largest
    others = [x for i, p in enumerate(per_head) for h, x in enumerate(p) if (i, h) != (which, 1)]
    assert max(others) < largest / 2
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=1e-3,
                                                                  weights=lv.LatentWeights(*up))
    got = latent_space._np(out)
    assert np.isnan(got[250:300, 1]).all()
    clean = [*range(250), 300, 301]
    assert np.isfinite(got[clean]).all()
    want, bound = layer._expected(cache, md, q, None, up, 1e-3)
    assert (np.abs(got - want)[clean] <= bound[clean]).all()
    if dtype == "fp16":  # (bf16's scores of that token pass fp32's largest for every head)
        rest = [0, 2, 3]
        assert (np.abs(got - want)[:, rest] <= bound[:, rest]).all()


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("value", (math.nan, math.inf, -math.inf))
def test_a_chunks_row_that_is_not_finite_reaches_every_query_that_sees_it(value, dtype, monkeypatch) -> None:
    latent_space._say(f"latent layer, {value} in a row of a chunk, {dtype}")
    layer._force(monkeypatch, lambda n, linear: n >= 200)
    cache, md, q, latent, rope_key, _, up = layer._step(4, 256, 64, 128, 128, 16, DTYPES[dtype], [20, 500], [400, 5], seed=5)
    latent[300, 7] = value
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07,
                                                                  weights=lv.LatentWeights(*up))
    got = latent_space._np(out)
    clean = [*range(300), *range(400, 405)]
    want, bound = layer._expected(cache, md, q, None, up, 0.07)
    assert np.isnan(got[300:400]).all() and np.isfinite(got[clean]).all()
    assert (np.abs(got - want)[clean] <= bound[clean]).all()


# ---- fp16 weights far below the largest ------------------------------------------------

def _tail(t, heads, rows, rope, tokens, scale):
    """Rows whose first score stands 2^26.4 above all others', which together weigh
    about rows * 2^-26.4: (latents, queries' value at latent 0, what comes out)."""
    latents = torch.zeros((rows, 128), device=DEV)
    latents[0, 0] = 40.0
    latents[1:, 1] = 1.0
    q0 = torch.tensor(26.4 * math.log(2) / (40.0 * scale)).to(t)
    w = math.exp(-float(q0) * 40.0 * scale)
    seen = rows - tokens + np.arange(tokens)  # of the others, by query
    return latents.to(t), float(q0), seen * w / (1 + seen * w)


@pytest.mark.parametrize("weighted", (None, "absorbed", "expanded"))
def test_many_small_fp16_weights(weighted, monkeypatch) -> None:
    """Thousands of keys, each weighing less than half of fp16's smallest step beside
    the largest weight, count.

    The weights are rounded as 2^7 and more times themselves (relative to the largest),
    so each is off by at most 2^-24 / 2 / 2^7 = 2^-32 or its half step: rows * 2^-32 +
    u |out|; the result, the attended latent and the value are rounded: 3 u |out|; the
    score is off by the fp32 sums' 128 * 2^-24 of 26.4 ln 2 (the numbers are chosen so
    that no product is rounded but the query's, which the formula takes as it is):
    1.5e-4 |out|."""
    latent_space._say(f"latent attention, many small fp16 weights, {weighted}")
    t, rows, tokens, scale = torch.float16, 8192, 200 if weighted == "expanded" else 2, 0.25
    # One workgroup for a request's whole length: pieces have maxima of their own.
    monkeypatch.setattr(native, "latent_decode_resident_groups", lambda *a: 1)
    monkeypatch.setattr(native, "latent_prefill_resident_units", lambda *a: 1)
    layer._force(monkeypatch, lambda n, linear: (n > 0) & (weighted == "expanded"))
    latents, q0, want = _tail(t, 2, rows, 32, tokens, scale)
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec("layer0", 2, 128, 32),))
    cache = lv.LatentPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=rows // 16, block_size=16, dtype=t, device=DEV))
    flat = cache.layer("layer0").rows.view(rows, 160)
    flat[: rows - tokens, :128] = latents[: rows - tokens]
    md = lv.PagedAttentionMetadata(block_tables=(tuple(range(rows // 16)),), num_computed_tokens=(rows - tokens,),
                                   query_layouts=(lv.linear_query_layout(tokens),))
    size = 128 if weighted is None else 64
    q = torch.zeros((tokens, 2, size + 32), dtype=t, device=DEV)
    q[..., 0] = q0
    weights = None
    if weighted:
        key_up, value_up = torch.zeros((2, 2, 64, 128), dtype=t, device=DEV)
        key_up[:, 0, 0] = 1
        value_up[:, 1, 1] = 1
        weights = lv.LatentWeights(key_up, value_up)
    context = lv.HipPagedAttentionBackend().create(cache, md)
    out = context.forward("layer0", q, latents[rows - tokens:], torch.zeros((tokens, 32), dtype=t, device=DEV), scale=scale,
                          weights=weights)
    assert not any(x.num_jobs or x.num_unit_jobs for x in context.plan.launches.values())
    got = latent_space._np(out)[..., 1]
    u = 2.0**-11
    assert (np.abs(got - want[:, None]) <= (rows * 2.0**-32 + (4 * u + 1.5e-4) * want)[:, None]).all()


@pytest.mark.parametrize("weighted", (None, "expanded"))
@pytest.mark.parametrize("lag", (7.9, 8.1, 40.0))
def test_fp16_weights_of_a_maximum_that_rises_late(lag, weighted, monkeypatch) -> None:
    """Scores that stand 2^lag above all earlier ones, below and above the 2^8 by which
    the running maximum may lag: no weight passes fp16's largest.

    Weights, result, attended latent and value are rounded: 5 u; a score is off by fp32
    sums of 128 * 2^-24 of lag: 2.2e-4."""
    latent_space._say(f"latent attention, fp16 weights of a maximum that rises by 2^{lag}, {weighted}")
    t, rows, tokens, scale = torch.float16, 1024, 200 if weighted else 2, 0.25
    monkeypatch.setattr(native, "latent_decode_resident_groups", lambda *a: 1)
    monkeypatch.setattr(native, "latent_prefill_resident_units", lambda *a: 1)
    layer._force(monkeypatch, lambda n, linear: n > 0)
    first = 512
    latents = torch.zeros((rows, 128), device=DEV)
    latents[first:, 0], latents[:first, 1], latents[first:, 2] = 40.0, 1.0, 1.0
    latents = latents.to(t)
    q0 = torch.tensor(lag * math.log(2) / (40.0 * scale)).to(t)
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec("layer0", 2, 128, 32),))
    cache = lv.LatentPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=rows // 16, block_size=16, dtype=t, device=DEV))
    cache.layer("layer0").rows.view(rows, 160)[: rows - tokens, :128] = latents[: rows - tokens]
    md = lv.PagedAttentionMetadata(block_tables=(tuple(range(rows // 16)),), num_computed_tokens=(rows - tokens,),
                                   query_layouts=(lv.linear_query_layout(tokens),))
    q = torch.zeros((tokens, 2, (64 if weighted else 128) + 32), dtype=t, device=DEV)
    q[..., 0] = q0
    key_up, value_up = torch.zeros((2, 2, 64, 128), dtype=t, device=DEV)
    key_up[:, 0, 0] = value_up[:, 1, 1] = value_up[:, 2, 2] = 1
    out = lv.HipPagedAttentionBackend().create(cache, md).forward(
        "layer0", q, latents[rows - tokens:], torch.zeros((tokens, 32), dtype=t, device=DEV), scale=scale,
        weights=lv.LatentWeights(key_up, value_up) if weighted else None)
    got, n = latent_space._np(out), rows - tokens + 1 + np.arange(tokens) - first
    w = math.exp(float(q0) * 40.0 * scale)
    for place, want in ((1, first / (first + n * w)), (2, n * w / (first + n * w))):
        off = np.abs(got[..., place] - want[:, None])
        assert (off <= ((5 * 2.0**-11 + 2.2e-4) * want + 2.0**-25)[:, None]).all()
