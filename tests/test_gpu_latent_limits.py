"""GPU: attention over the latent cache where numbers end."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
import test_gpu_latent as latent_space
import test_gpu_latent_layer as layer
from light_vllm_amd import latent_attention

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
