"""GPU: steps over the latent cache, with their heads' weights in both forms and in
latent space, held to the bound of ``latent_cases`` (the norm of each token's and head's
error; that mistakes pass it is tested on the CPU), and the rows that the step left in
the pool."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

import latent_cases as L
import light_vllm_amd as lv
from light_vllm_amd import latent_attention
from oracle import latent_oracle as Z

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

DEV = torch.device("cuda:0")


def _cache(step):
    cache = lv.LatentPagedKVCache(step["spec"], lv.PagedKVCacheConfig(
        num_blocks=step["num_blocks"], block_size=step["block"], dtype=step["dtype"], device=DEV))
    rows = cache.layer("layer0").rows
    rows.view(-1, rows.shape[-1]).copy_(step["rows"])
    return cache


def _check_pool(step, pool, rotary) -> None:
    """The step's latents as they came, its keys turned (each rounded once, behind fp32
    products: u |x| + 2^-22 (|a cos| + |b sin|)), every other row as it was."""

    layer, slots = step["spec"].layers[0], step["slots"]
    others = torch.ones(len(pool), dtype=torch.bool)
    others[slots] = False
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(pool[others]), bits(step["rows"][others]))
    got, size = pool[slots], layer.latent_size
    assert torch.equal(got[:, :size], step["latent"])
    key = step["rope_key"].double().numpy()
    if not rotary:
        assert torch.equal(got[:, size:], step["rope_key"])
        return
    c, s = (a.double().numpy() for a in step["rotary"])
    interleaved = layer.rotary_layout == "interleaved"
    want = Z.rotate(key, c, s, interleaved)
    # |a| |cos| + |b| |sin| and |b| |cos| + |a| |sin|: both of a pair are below this.
    pair = np.abs(key[:, 0::2]) + np.abs(key[:, 1::2]) if interleaved else np.abs(key[:, : key.shape[1] // 2]) + np.abs(
        key[:, key.shape[1] // 2:])
    pair = np.repeat(pair, 2, axis=1) if interleaved else np.concatenate((pair, pair), axis=1)
    u = torch.finfo(step["dtype"]).eps / 2
    assert (np.abs(got[:, size:].double().numpy() - want) <= u * np.abs(want) + 2.0**-22 * pair + 2.0**-25).all()


def _run(case, expanded, monkeypatch, *, dtype="bf16", seed=3, layout="interleaved", rotary=True, scale=None, heads=None):
    """``expanded(queries, linear)``: which requests take that form (None: by the rule)."""

    step = L.make(case, L.DTYPES[dtype], seed, layout)
    if expanded is not None:
        monkeypatch.setattr(latent_attention, "_expanded", lambda facts, *a: expanded(facts.q_lens, facts.vis_off < 0))
    scale = L.scale_of(case) if scale is None else scale
    print(f"[gpu] latent norms {case} {dtype} {layout} rotary={rotary} scale={scale:.3f}", file=sys.stderr, flush=True)
    cache, md, up = _cache(step), step["metadata"], step["up"]
    context = lv.HipPagedAttentionBackend().create(cache, md)
    out = context.forward("layer0", step["query"].to(DEV), step["latent"].to(DEV), step["rope_key"].to(DEV), scale=scale,
                          rotary=tuple(a.to(DEV) for a in step["rotary"]) if rotary else None,
                          weights=None if up is None else lv.LatentWeights(*(w.to(DEV) for w in up)))
    torch.cuda.synchronize()
    pool = cache.layer("layer0").rows.view(len(step["rows"]), -1)
    _check_pool(step, pool.cpu(), rotary)
    forms = [False] * len(md.query_layouts) if up is None else [bool(x) for x in latent_attention._expanded(
        md.facts, step["spec"].layers[0], case[3], case[4])]
    kw = dict(scale=scale, rotary=rotary, heads=heads)
    want, size = L.attend(step, pool, forms, **kw)
    assert want.isfinite().all()
    got = out.double() if heads is None else out[:, heads].double()
    assert got.shape == want.shape
    worst = ((got - want).norm(dim=-1) / L.bound(step, pool, forms, want, size, **kw)).max()
    print(f"[margin] latent norms: {100 * worst:.1f}% of the bound", file=sys.stderr, flush=True)
    assert worst <= 1.0
    return context, out


absorbed = lambda n, linear: n < 0  # noqa: E731
every = lambda n, linear: n > 0  # noqa: E731


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("case", L.SHORT)
def test_absorbed(case, dtype, monkeypatch) -> None:
    _run(case, absorbed, monkeypatch, dtype=dtype)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("case", L.LONG)
def test_expanded(case, dtype, monkeypatch) -> None:
    context, _ = _run(case, every, monkeypatch, dtype=dtype, layout="half")
    if case[6] == [9000]:
        assert any(shape.num_unit_jobs > 0 for shape in context.plan.launches.values())


@pytest.mark.parametrize("rotary", (True, False))
@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("case", L.MIXED)
def test_mixed(case, dtype, rotary, monkeypatch) -> None:
    _run(case, lambda n, linear: (n >= 400) & linear, monkeypatch, dtype=dtype, rotary=rotary)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("form", (absorbed, every))
def test_every_length(form, dtype, monkeypatch) -> None:
    _run(L.EVERY_LENGTH, form, monkeypatch, dtype=dtype)


@pytest.mark.parametrize("wide", (False, True))
def test_many_short_requests_around_a_long_one(wide, monkeypatch) -> None:
    """The wide tiles of the products with the weights; ``wide``: 128 columns a
    workgroup."""
    if wide:
        monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
    layouts = [1 + (i % 7 == 0) for i in range(151)]
    computed = [20 + (i * 5) % 41 for i in range(151)]
    layouts[60], computed[60] = 256, 10
    _run((128, 128, 32, 64, 64, 16, computed, layouts), lambda n, linear: n >= 200, monkeypatch, heads=[0, 31, 64, 127])


def test_heads_in_groups(monkeypatch) -> None:
    case = (5, 256, 64, 128, 64, 16, [40], [700])
    _, want = _run(case, every, monkeypatch)
    monkeypatch.setattr(latent_attention, "EXPANDED_BYTES", 1 << 20)
    _, got = _run(case, every, monkeypatch)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("scale", (1.0, -0.5, 0.0))
def test_scales(scale, dtype, monkeypatch) -> None:
    _run((4, 128, 32, 64, 64, 16, [200, 30], [300, 2]), lambda n, linear: n >= 200, monkeypatch, dtype=dtype, scale=scale)


def _random_case(rng):
    heads = int(rng.choice((1, 3, 5, 8, 16, 16, 20, 40, 64, 128)))
    latent, rope = int(rng.choice((512, 512, 384, 256, 128))), int(rng.choice((64, 32)))
    nope, value = (None, None) if rng.random() < 0.4 else (int(rng.choice((64, 128))), int(rng.choice((64, 128))))
    computed, layouts = [], []
    for _ in range(int(rng.integers(1, 9))):
        kind = rng.random()
        if kind < 0.5:
            n = int(rng.choice((1, 1, 1, 2, 5)))
            parents, far = n, 3000
        elif kind < 0.75:
            n = int(rng.integers(2, 40))
            parents, far = tuple([-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]), 1500
        else:
            parents, far = int(rng.integers(6, 420)), 900
        layouts.append(parents)
        computed.append(int(rng.choice((0, int(rng.integers(0, 70)), int(rng.integers(0, far))))))
    return heads, latent, rope, nope, value, int(rng.choice((16, 16, 1, 12, 32, 64))), computed, layouts


@pytest.mark.parametrize("seed", range(40))
def test_random_steps(seed, monkeypatch) -> None:
    """Any forms, widths, lengths, trees and blocks together, twice: the same bits."""
    rng = np.random.default_rng(seed)
    case = _random_case(rng)
    if seed % 3 == 0:
        monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
    kw = dict(dtype=str(rng.choice(("bf16", "fp16"))), layout=str(rng.choice(("interleaved", "half"))), seed=seed,
              rotary=bool(rng.random() < 0.7), heads=sorted({0, case[0] // 2, case[0] - 1}))
    _, first = _run(case, None, monkeypatch, **kw)
    _, again = _run(case, None, monkeypatch, **kw)
    assert torch.equal(first, again)
