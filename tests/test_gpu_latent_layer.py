"""GPU: a layer over the latent cache with its heads' weights (per-head queries in,
per-head values out), in both of its forms, against fp64.

Tolerance, for either form (u = eps / 2 of the step's type; B = attention of
sum_l |value_up[v, l]| |c_l|, at least that of |value|; Q = sum_n |q_n| |key_up[n, l]|):
* the softmax weights are rounded, and the sum that divides them counts them so:
  2 u B; what is rounded between (the attended latents, or every key's value): u
  B; the result: u |out|;
* a score is off by d = scale (u (sum_l |qa_l| |c_l| + sum_n |q_n| |k_n| + sum |q
  r|) + (L + N + P + 8) 2^-24 (sum_l Q_l |c_l| + sum |q r|)): the query in latent
  space or the key is rounded, the turned query is, and the sums are fp32; it moves
  the weights and their sum: 2 B (e^d - 1);
* fp32 sums: (keys / 16 + 64 + L) 2^-24 B.
"""

from __future__ import annotations

import math
import sys

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
from light_vllm_amd import latent_attention
from oracle import latent_oracle as Z

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

DEV = torch.device("cuda:0")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TREE = (-1, 0, 0, 1, 1, 2, 3, 0, 7)


def _say(text):
    print(f"[gpu] {text}", file=sys.stderr, flush=True)


def _np(t):
    return t.double().cpu().numpy()


def _step(heads, latent, rope, nope, value, bs, dtype, computed, layouts, seed, layout="interleaved"):
    """A cache with history (NaN wherever no token is), this step's tensors and the layer's weights."""
    rng = np.random.default_rng(seed)
    layouts = [p if isinstance(p, tuple) else tuple(range(-1, p - 1)) for p in layouts]
    need = [-(-(c + len(p)) // bs) for c, p in zip(computed, layouts)]
    free = [int(b) for b in rng.permutation(sum(need) + 3)]
    tables = []
    for n in need:
        tables.append(tuple(free[:n]))
        free = free[n:]
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec("layer0", heads, latent, rope, layout),))
    cache = lv.LatentPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=sum(need) + 3, block_size=bs, dtype=dtype, device=DEV))
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows = cache.layer("layer0").rows.view(-1, latent + rope)
    rows.fill_(math.nan)
    held = torch.cat([torch.tensor(t)[torch.arange(c) // bs] * bs + torch.arange(c) % bs for t, c in zip(tables, computed)]).to(DEV)
    rows[held] = torch.randn((len(held), latent + rope), generator=gen, device=DEV).to(dtype)
    t = sum(map(len, layouts))
    q = (1.5 * torch.randn((t, heads, nope + rope), generator=gen, device=DEV)).to(dtype)
    both = torch.randn((t, latent + rope), generator=gen, device=DEV).to(dtype)
    up = [(torch.randn((heads, n, latent), generator=gen, device=DEV) * latent**-0.5).to(dtype) for n in (nope, value)]
    metadata = lv.PagedAttentionMetadata(block_tables=tuple(tables), num_computed_tokens=tuple(computed),
                                         query_layouts=tuple(lv.QueryLayout(p) for p in layouts))
    rotary = lv.RotaryEmbedding(rope, device=DEV)(torch.randint(0, 100000, (t,), generator=gen, device=DEV))
    return cache, metadata, q, both[:, :latent], both[:, latent:], rotary, up


def _expected(cache, metadata, q, rotary, up, scale, heads=None):
    """(attention, its bound) for some heads over the cache's rows as they are now."""
    spec = cache.layer_spec("layer0")
    latent, rope, bs = spec.latent_size, spec.rope_size, cache.config.block_size
    u = torch.finfo(cache.config.dtype).eps / 2
    qn = _np(q)
    if rotary is not None:
        qn[..., -rope:] = Z.rotate(qn[..., -rope:], *(_np(t) for t in rotary), spec.rotary_layout == "interleaved")
    rows = _np(cache.layer("layer0").rows).reshape(-1, latent + rope)
    key_up, value_up = (_np(w) for w in up)
    heads = range(q.shape[1]) if heads is None else heads
    outs, bounds, t0 = [], [], 0
    for table, c, layout in zip(metadata.block_tables, metadata.num_computed_tokens, metadata.query_layouts):
        n = len(layout)
        at = np.arange(c + n)
        keys = rows[np.asarray(table, dtype=np.int64)[at // bs] * bs + at % bs]
        seen = Z.visible(layout.parent_indices, c)
        lat, rot = keys[:, :latent], keys[:, latent:]
        for h in heads:
            qh, wk, wv = qn[t0:t0 + n, h], key_up[h], value_up[h]
            qa = qh[:, :-rope] @ wk
            with np.errstate(invalid="ignore", over="ignore"):
                k, v = lat @ wk.T, lat @ wv.T
                s = np.where(seen, (qh[:, :-rope] @ k.T + qh[:, -rope:] @ rot.T) * scale, -np.inf)
                al, ar, aq = np.nan_to_num(np.abs(lat)), np.nan_to_num(np.abs(rot)), np.abs(qh)
                turned = aq[:, -rope:] @ ar.T
                d = u * (np.abs(qa) @ al.T + aq[:, :-rope] @ np.nan_to_num(np.abs(k)).T + turned) + (
                    latent + wk.shape[0] + rope + 8) * 2.0**-24 * ((aq[:, :-rope] @ np.abs(wk)) @ al.T + turned)
                d = np.where(seen, d * abs(scale), 0).max(axis=1)
                w = np.exp(s - s.max(axis=1, keepdims=True))
                w /= w.sum(axis=1, keepdims=True)
                size = np.abs(lat) @ np.abs(wv).T
                if np.isfinite(keys).all():
                    out, b = w @ v, w @ size
                else:
                    out = np.stack([w[i, seen[i]] @ v[seen[i]] for i in range(n)])
                    b = np.stack([w[i, seen[i]] @ size[seen[i]] for i in range(n)])
            outs.append(out)
            bounds.append(3 * u * b + u * np.abs(out) + 2 * b * np.expm1(d)[:, None]
                          + ((c + n) / 16 + 64 + latent) * 2.0**-24 * b + 2.0**-24)
        t0 += n
    def stack(parts):
        k = len(list(heads))
        return np.concatenate([np.stack(parts[i:i + k], axis=1) for i in range(0, len(parts), k)])
    return stack(outs), stack(bounds)


def _check(out, want, bound, what="layer"):
    got = out.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    worst = float((np.abs(got - want)[fine] / bound[fine]).max(initial=0))
    print(f"[margin] latent {what}: {100 * worst:.1f}% of the bound", file=sys.stderr, flush=True)
    assert worst <= 1.0


def _run(args, scale=None, rotary=True, heads=None, backend=None):
    cache, metadata, q, latent, rope_key, angles, up = args
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    angles = angles if rotary else None
    context = (backend or lv.HipPagedAttentionBackend()).create(cache, metadata)
    out = context.forward("layer0", q, latent, rope_key, scale=scale, rotary=angles, weights=lv.LatentWeights(*up))
    torch.cuda.synchronize()
    want, bound = _expected(cache, metadata, q, angles, up, scale, heads)
    _check(out if heads is None else out[:, heads], want, bound)
    return context, out


SHORT = [  # heads, latent, rope, nope, value, block, computed, layouts
    (16, 512, 64, 128, 128, 16, [0, 31, 700], [1, 1, 1]),
    (5, 128, 32, 64, 128, 12, [90, 0, 40], [TREE, 3, 1]),
    (40, 256, 32, 64, 64, 16, [300], [1]),
    (128, 384, 64, 128, 64, 1, [33, 7], [2, 1]),
]
LONG = [
    (4, 512, 64, 128, 128, 16, [0], [700]),
    (3, 512, 64, 128, 128, 16, [1000, 0], [513, 400]),
    (8, 128, 32, 64, 128, 12, [64, 5, 333], [129, 300, 191]),
    (2, 256, 32, 64, 64, 16, [130], [1025]),
    (5, 384, 64, 128, 64, 64, [63], [640]),
    (1, 256, 64, 64, 128, 1, [0], [833]),
]
MIXED = [
    (16, 256, 32, 64, 64, 16, [100, 0, 50, 3000, 20], [1, 500, TREE, 1, 400]),
    (4, 512, 64, 128, 128, 32, [0, 700, 1500], [600, 1, 450]),
]


def _force(monkeypatch, chosen):
    """Requests take the expanded form by ``chosen(queries, linear)``, not by the rule."""
    monkeypatch.setattr(latent_attention, "_expanded", lambda facts, *a: chosen(facts.q_lens, facts.vis_off < 0))


def test_the_rule_gives_each_form_its_requests() -> None:
    """Tokens, short runs and trees stay absorbed, long linear chunks do not."""
    args = _step(4, 512, 64, 128, 128, 16, torch.bfloat16, [500, 20, 0, 3000, 0], [1, 20, TREE, 1500, 900], seed=11)
    forms = latent_attention._expanded(args[1].facts, args[0].layer_spec("layer0"), 128, 128)
    assert forms.tolist() == [False, False, False, True, True]
    tree = _step(4, 512, 64, 128, 128, 16, torch.bfloat16, [0], [tuple([-1] + [0] * 899)], seed=11)
    assert not latent_attention._expanded(tree[1].facts, tree[0].layer_spec("layer0"), 128, 128).any()


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("case", SHORT)
def test_absorbed(case, dtype, monkeypatch) -> None:
    _say(f"latent layer, absorbed {case} {dtype}")
    _force(monkeypatch, lambda n, linear: n < 0)
    _run(_step(*case[:6], DTYPES[dtype], *case[6:], seed=case[0]))


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("case", LONG)
def test_expanded(case, dtype, monkeypatch) -> None:
    _say(f"latent layer, expanded {case} {dtype}")
    _force(monkeypatch, lambda n, linear: n > 0)
    _run(_step(*case[:6], DTYPES[dtype], *case[6:], seed=case[0], layout="half"))


@pytest.mark.parametrize("rotary", (True, False))
@pytest.mark.parametrize("case", MIXED)
def test_mixed(case, rotary, monkeypatch) -> None:
    _say(f"latent layer, mixed {case}")
    _force(monkeypatch, lambda n, linear: (n >= 400) & linear)
    _run(_step(*case[:6], torch.bfloat16, *case[6:], seed=case[0]), rotary=rotary)


@pytest.mark.parametrize("form", (True, False))
def test_each_form_at_lengths_that_the_rule_gives_the_other(form, monkeypatch) -> None:
    """Both forms hold at every length: one query, units that end anywhere."""
    _say(f"latent layer, expanded={form} at every length")
    _force(monkeypatch, lambda n, linear: np.full(n.shape, form))
    args = _step(3, 256, 64, 128, 64, 16, torch.bfloat16, [0, 63, 64, 500, 0, 1, 127], [1, 1, 2, 65, 128, 129, 256], seed=1)
    _run(args)


@pytest.mark.parametrize("long", (0, 256))
def test_many_short_requests(long, monkeypatch) -> None:
    """Rows enough for the wide tiles of the products with the weights, their last
    tile in part, with a long request's rows between them."""
    _say(f"latent layer, 151 short requests, a long one of {long}")
    _force(monkeypatch, lambda n, linear: n >= 200)
    layouts = [1 + (i % 7 == 0) for i in range(151)]
    computed = [(i * 5) % 41 for i in range(151)]
    if long:
        layouts[60], computed[60] = long, 10
    _run(_step(128, 128, 32, 64, 64, 16, torch.bfloat16, computed, layouts, seed=12))


def test_heads_in_groups(monkeypatch) -> None:
    _say("latent layer, heads in groups")
    _force(monkeypatch, lambda n, linear: n > 0)
    args = _step(5, 256, 64, 128, 64, 16, torch.bfloat16, [40], [700], seed=2)
    _, want = _run(args)
    monkeypatch.setattr(latent_attention, "EXPANDED_BYTES", 1 << 20)
    _, got = _run(args)
    assert torch.equal(got, want)


def test_split_units_of_a_long_history(monkeypatch) -> None:
    """Few units over many keys: pieces of units, merged."""
    _say("latent layer, split units")
    _force(monkeypatch, lambda n, linear: n > 0)
    args = _step(2, 512, 64, 128, 128, 16, torch.bfloat16, [9000], [300], seed=3)
    context, _ = _run(args, heads=[1])
    assert any(shape.num_unit_jobs > 0 for shape in context.plan.launches.values())


def test_large_and_negative_scales(monkeypatch) -> None:
    _say("latent layer, scales")
    _force(monkeypatch, lambda n, linear: n >= 200)
    for scale in (1.0, -0.5, 0.0):
        _run(_step(4, 128, 32, 64, 64, 16, torch.bfloat16, [200, 30], [300, 2], seed=4), scale=scale)


@pytest.mark.parametrize("value", (math.nan, math.inf, -math.inf))
def test_a_later_tokens_row_that_is_not_finite(value, monkeypatch) -> None:
    """It reaches the queries that see it and no others."""
    _say(f"latent layer, {value} in a later token's row")
    _force(monkeypatch, lambda n, linear: n >= 200)
    cache, md, q, latent, rope_key, rotary, up = args = _step(4, 256, 64, 128, 128, 16, torch.bfloat16, [20, 500],
                                                              [400, 5], seed=5)
    latent[300, 7] = value
    latent[403, 9] = value
    weights = lv.LatentWeights(*up)
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07, weights=weights)
    got = out.double().cpu().numpy()
    want, bound = _expected(cache, md, q, None, up, 0.07)
    clean = [*range(300), 400, 401, 402]
    assert np.isfinite(got[clean]).all()
    assert (np.abs(got - want)[clean] <= bound[clean]).all()
    if math.isnan(value):
        rest = [*range(300, 400), 403, 404]
        assert np.isnan(got[rest]).all() and np.isnan(want[rest]).all()
    else:
        assert not np.isfinite(got[300]).any()


def test_fp16_values_past_the_largest_are_held(monkeypatch) -> None:
    """A later token's row whose per-head values pass fp16's largest stays with the
    queries that see it."""
    _say("latent layer, fp16 values that overflow")
    _force(monkeypatch, lambda n, linear: n >= 200)
    cache, md, q, latent, rope_key, rotary, up = _step(2, 128, 32, 64, 64, 16, torch.float16, [20], [300], seed=6)
    latent[250] = 60000.0 * torch.sign(up[1][0, 3])
    weights = lv.LatentWeights(*up)
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.1, weights=weights)
    want, bound = _expected(cache, md, q, None, up, 0.1)
    got = out.double().cpu().numpy()
    assert (np.abs(got - want)[:250] <= bound[:250]).all()


def test_strided_queries_and_weights(monkeypatch) -> None:
    _say("latent layer, strided queries and weights")
    _force(monkeypatch, lambda n, linear: n >= 200)
    for computed, layouts in (([30, 64], [1, 5]), ([0], [300])):
        cache, md, q, latent, rope_key, rotary, up = _step(4, 128, 32, 64, 64, 16, torch.bfloat16, computed, layouts, seed=7)
        run = lambda q, up: lv.HipPagedAttentionBackend().create(cache, md).forward(  # noqa: E731
            "layer0", q, latent, rope_key, scale=0.1, rotary=rotary, weights=lv.LatentWeights(*up))
        want = run(q, up)
        # One up projection for keys and values, [heads, nope + value, latent], as models hold it.
        joined = torch.cat(up, dim=1)
        assert torch.equal(run(q, (joined[:, :64], joined[:, 64:])), want)
        assert torch.equal(run(q.transpose(0, 1).contiguous().transpose(0, 1), up), want)
        assert torch.equal(run(torch.cat((q[..., :1], q), dim=2)[..., 1:], [w.transpose(1, 2).contiguous().transpose(1, 2) for w in up]), want)


def test_refusals() -> None:
    cache, md, q, latent, rope_key, rotary, up = _step(4, 128, 32, 64, 64, 16, torch.bfloat16, [30], [2], seed=8)
    k, v = up
    for a, b, message in ((k[0], v, "three dimensions"), (k[:2], v, "agree"), (k[:, :, :64], v, "agree"),
                          (k[:, :32], v, "one of"), (k.half(), v, "one dtype"), (k.float(), v.float(), "bfloat16 or float16"),
                          (k.cpu(), v.cpu(), "GPU")):
        with pytest.raises(ValueError, match=message):
            lv.LatentWeights(a, b)
    good = lv.LatentWeights(k, v)
    for args, weights, message in (
        ((q, latent, rope_key), lv.LatentWeights(k[:2], v[:2]), "do not match the layer spec"),
        ((q, latent, rope_key), lv.LatentWeights(k.half(), v.half()), "weights dtype"),
        ((q[..., :64], latent, rope_key), good, "query shape"), ((q, latent, rope_key), None, "query shape"),
        ((q.half(), latent, rope_key), good, "query dtype"),
    ):
        with pytest.raises(lv.KVCacheError, match=message):
            lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", *args, scale=0.1, weights=weights)
    for rot, message in (((None, None), "cosines must have shape"), ((rotary[0], None), "sines must have shape")):
        with pytest.raises(lv.KVCacheError, match=message):
            lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.1, rotary=rot,
                                                                    weights=good)


def test_graph_replays(monkeypatch) -> None:
    """A mixed step captured after one eager run; a form that has not run refuses
    to be captured."""
    _say("latent layer, captured")
    _force(monkeypatch, lambda n, linear: n >= 200)
    cache, md, q, latent, rope_key, rotary, up = _step(4, 256, 64, 128, 64, 16, torch.bfloat16, [700, 40, 90], [1, 300, TREE], seed=9)
    weights, backend = lv.LatentWeights(*up), lv.HipPagedAttentionBackend()
    run = lambda c: c.forward("layer0", q, latent, rope_key, scale=0.07, rotary=rotary, weights=weights)  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fresh = backend.create(cache, md)
    torch.cuda.synchronize()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(lv.ExecutionError, match="once before it is captured"):
            run(fresh)
        torch.zeros(1, device=DEV)
    with torch.cuda.stream(stream):
        run(backend.create(cache, md))
    torch.cuda.current_stream().wait_stream(stream)
    context, graph = backend.create(cache, md), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(context)
    gen = torch.Generator(device=DEV).manual_seed(3)
    other = _step(4, 256, 64, 128, 64, 16, torch.bfloat16, [50], [200], seed=10)
    for i in range(4):
        for t in (q, latent, rope_key):
            t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        graph.replay()
        _run(other, backend=backend)
        torch.cuda.synchronize()
        _check(out, *_expected(cache, md, q, rotary, up, 0.07))
        assert torch.equal(run(backend.create(cache, md)), out)


def test_rows_past_32_bits_of_the_pool(monkeypatch) -> None:
    """A pool of 4.6e9 values (9.2 GB): the same step at its last blocks gives what a
    small pool gives, in both forms, and so do write, compact and block copies."""
    _say("latent layer, a pool of 9.2 GB")
    case = (16, 512, 64, 128, 128, 16, torch.bfloat16)
    computed, layouts = [40, 5, 100], [300, TREE, 1]
    big_blocks = 500_000
    large = lv.LatentPagedKVCache(_step(*case, [0], [1], seed=13)[0].model_spec, lv.PagedKVCacheConfig(
        num_blocks=big_blocks, block_size=16, dtype=torch.bfloat16, device=DEV))
    rows_large = large.layer("layer0").rows
    assert rows_large.numel() > 2**32
    _force(monkeypatch, lambda n, linear: n >= 200)
    for wide in (False, True):
        if wide:
            monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
        small, md, q, latent, rope_key, rotary, up = _step(*case, computed, layouts, seed=13)
        rows_small = small.layer("layer0").rows
        n = rows_small.shape[0]
        off = big_blocks - n
        rows_large[off:] = rows_small
        rows_large[:n] = 7
        far = lv.PagedAttentionMetadata(block_tables=tuple(tuple(b + off for b in t) for t in md.block_tables),
                                        num_computed_tokens=md.num_computed_tokens, query_layouts=md.query_layouts)
        outs = [lv.HipPagedAttentionBackend().create(cache, m).forward(
            "layer0", q, latent, rope_key, scale=0.07, rotary=rotary, weights=lv.LatentWeights(*up))
            for cache, m in ((small, md), (large, far))]
        assert torch.equal(outs[0], outs[1])

        def same():
            a, b = rows_small.view(torch.int16), rows_large[off:].view(torch.int16)  # (bits: some are NaN)
            assert torch.equal(a, b) and bool((rows_large[:n] == 7).all())

        same()
        slots = torch.tensor([3, 16 * n - 1], device=DEV)
        for cache, at in ((small, 0), (large, 16 * off)):
            cache.write("layer0", latent[:2], rope_key[:2], slots + at, rotary=(rotary[0][:2], rotary[1][:2]))
            cache.copy_blocks([at // 16], [at // 16 + 1])
            cache.compact(tuple(b + at // 16 for b in md.block_tables[1]), num_computed_tokens=5, num_query_tokens=9,
                          num_reserved_query_tokens=9, retained_query_indices=(0, 2, 5))
        same()


def test_steps_on_other_streams_than_their_plans() -> None:
    """A context whose lists lie on another stream may be dropped while its step is
    pending, and lists that a first forward uploads are there for every stream."""
    _say("latent layer, contexts used on other streams")
    args = _step(16, 256, 64, 128, 64, 16, torch.bfloat16, [300, 40], [1, 5], seed=14)
    cache, md, q, latent, rope_key, rotary, up = args
    weights = lv.LatentWeights(*up)
    call = dict(scale=0.07, rotary=rotary, weights=weights)
    want = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, **call)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for fresh in (True, False):
        backend = lv.HipPagedAttentionBackend()
        if not fresh:  # (the form is known: its lists are uploaded by create)
            backend.create(cache, md).forward("layer0", q, latent, rope_key, **call)
        torch.cuda.synchronize()
        contexts = [backend.create(cache, md) for _ in streams]
        torch.cuda.synchronize()
        outs = []
        for stream in streams:
            with torch.cuda.stream(stream):
                torch.cuda._sleep(2_000_000)
                outs.append(contexts.pop(0).forward("layer0", q, latent, rope_key, **call))
        backend._last = None  # (the last plan's keeper)
        junk = [torch.full((n,), -1, dtype=torch.int32, device=DEV) for n in (64, 256, 512, 1024, 4096, 1 << 16) for _ in range(8)]
        torch.cuda.synchronize()
        assert len(junk) and all(torch.equal(o, want) for o in outs)
