"""GPU: the latent cache, its rotary angles and the attention over it in latent
space, against fp64.

Tolerances, from the roundings on the way (u = eps / 2 of the step's type):
* a turned value is rounded once: u |x| + 2^-22 (|a cos| + |b sin|) (the fp32
  products and their sum);
* attention: the weights are rounded to T before the products, and the sum that
  divides them counts them as rounded, so they move the result by at most u (A +
  |out|) <= 2 u A, A being the attention of |value|; the result is rounded: u
  |out|.  A score is off by d = scale (u sum |q r| over the rotated part, where
  the append rounds the turned query, + (L + P + 4) 2^-24 sum |q k| for the fp32
  sums); it moves the weights by e^d - 1 and the sum that divides them too: 2 A
  (e^d - 1).  Exponentials (2^-22 each side) and the fp32 sums over N keys, added
  in tiles and pieces: (N / 16 + 64) 2^-24 A.
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


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _cache(heads, latent, rope, bs, blocks, dtype, layers=1, layout="interleaved"):
    spec = lv.LatentKVCacheSpec(tuple(lv.LatentLayerSpec(f"layer{i}", heads, latent, rope, layout) for i in range(layers)))
    return lv.LatentPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=blocks, block_size=bs, dtype=dtype, device=DEV))


def _flat(cache, layer="layer0"):
    rows = cache.layer(layer).rows
    return rows.view(-1, rows.shape[-1])


def _angles(n, rope, gen, far=1 << 17):
    positions = torch.randint(0, far, (n,), generator=gen, device=DEV)
    return lv.RotaryEmbedding(rope, device=DEV)(positions)


# ---- angles ------------------------------------------------------------------------

@pytest.mark.parametrize("scaling", (None, lv.RotaryScaling("linear", 3.0), lv.RotaryScaling("base", 8.0),
                                     lv.RotaryScaling("ramp", 40.0), lv.RotaryScaling("smooth", 8.0, 8192)))
@pytest.mark.parametrize("size, n, index", [(64, 1, torch.int64), (2, 3, torch.int32), (32, 1000, torch.int32),
                                            (128, 4099, torch.int64), (96, 255, torch.int64)])
def test_angles(size, n, index, scaling) -> None:
    """Off by the reduction (2^-51 of the turns), the reduced angle's fp32 value
    (2^-25 of at most pi / 4), the sums (four roundings of at most 2^-24, Taylor
    tails below 2^-29) and the product with the magnitude: under 2^-21 times it."""
    if size == 2 and scaling is not None and scaling.kind == "base":
        pytest.skip("one pair")
    _say(f"angles {size} x {n} {scaling}")
    gen = torch.Generator(device=DEV).manual_seed(size + n)
    positions = torch.randint(0, 1 << 21, (n,), generator=gen, device=DEV).to(index)
    positions[: n // 2] %= 9
    emb = lv.RotaryEmbedding(size, base=500000.0, scaling=scaling, device=DEV)
    freq, magnitude = lv.rotary_frequencies(size, 500000.0, scaling)
    angle = positions.cpu().double()[:, None] * freq
    for full in (False, True):
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            got = emb(positions, full=full, dtype=dtype)
            for t, want in zip(got, (angle.cos() * magnitude, angle.sin() * magnitude)):
                want = torch.cat((want, want), dim=1) if full else want
                assert t.shape == want.shape and t.dtype == dtype
                bound = 2.0**-21 * magnitude + (0 if dtype == torch.float32 else _u(dtype) * want.abs() + 2.0**-25)
                assert bool(((t.cpu().double() - want).abs() <= bound).all())
    assert all(t.shape == (0, size // 2) for t in emb(positions[:0]))
    if n > 4:  # a strided vector of positions
        assert torch.equal(emb(positions[::2])[0], emb(positions)[0][::2])


def test_angle_refusals() -> None:
    emb = lv.RotaryEmbedding(64, device=DEV)
    for bad, message in ((torch.zeros(3, device=DEV), "int32 or int64"), (torch.zeros((3, 1), dtype=torch.int64, device=DEV), "vector"),
                         (torch.zeros(3, dtype=torch.int64), "device")):
        with pytest.raises(ValueError, match=message):
            emb(bad)
    with pytest.raises(lv.KVCacheError, match="float32, float16"):
        emb(torch.zeros(3, dtype=torch.int64, device=DEV), dtype=torch.float64)


def test_full_angles_serve_the_per_head_cache() -> None:
    """The rows of ``full=True`` are the rotary= argument over a PagedKVCache."""
    _say("full angles through the 16-bit cache")
    spec = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("layer0", 4, 2, 64),))
    gen = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn((5, h, 64), generator=gen, device=DEV).to(torch.bfloat16) for h in (4, 2, 2))
    md = lv.PagedAttentionMetadata(block_tables=((2,),), num_computed_tokens=(0,), query_layouts=(lv.linear_query_layout(5),))
    rotary = lv.RotaryEmbedding(64, device=DEV)(torch.arange(5, device=DEV), full=True, dtype=torch.bfloat16)
    outs = []
    for turned in (False, True):
        cache = lv.PagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=3, block_size=16, dtype=torch.bfloat16, device=DEV))
        context = lv.HipPagedAttentionBackend().create(cache, md)
        if turned:
            outs.append(context.forward("layer0", q, k, v, scale=0.125, rotary=rotary))
        else:
            c, s = (t.double()[:, None, :] for t in rotary)
            half = lambda x: torch.cat((-x[..., 32:], x[..., :32]), dim=-1)  # noqa: E731
            qr, kr = ((x.double() * c + half(x.double()) * s).to(torch.bfloat16) for x in (q, k))
            outs.append(context.forward("layer0", qr, kr, v, scale=0.125))
    # (The 16-bit path rounds each product: keys and queries differ by up to 3 u of the products.)
    assert float((outs[0].float() - outs[1].float()).abs().max()) < 0.1


# ---- append ------------------------------------------------------------------------

def _expect_rows(want, latent, rope_key, slots, rotary, interleaved):
    """``want`` with the step's rows in place, and how far each value may be off."""
    size = latent.shape[1]
    off = np.zeros_like(want)
    lat, key = _np(latent), _np(rope_key)
    turned, most = key, 0 * key
    if rotary is not None:
        c, s = (_np(t) for t in rotary)
        turned = Z.rotate(key, c, s, interleaved)
        most = _u(latent.dtype) * np.abs(turned) + 2.0**-22 * Z.rotate(np.abs(key), np.abs(c), -np.abs(s), interleaved).clip(0)
        most = np.maximum(most, _u(latent.dtype) * np.abs(turned)) + 2.0**-22 * np.abs(key).max(initial=0)
    for t, slot in enumerate(slots):
        if slot >= 0:
            want[slot, :size], want[slot, size:] = lat[t], turned[t]
            off[slot, size:] = most[t]
    return want, off


def _check_rows(cache, want, off, layer="layer0"):
    got = _np(_flat(cache, layer))
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    assert np.all(same | (np.abs(got - want) <= off))


@pytest.mark.parametrize("rotary", (True, False))
@pytest.mark.parametrize("heads, latent, rope, bs, dtype, layout", [
    (16, 512, 64, 16, "bf16", "interleaved"), (5, 256, 32, 12, "fp16", "half"), (1, 128, 64, 1, "bf16", "half"),
    (40, 384, 32, 64, "fp16", "interleaved")])
@pytest.mark.parametrize("n", (1, 37, 700))
def test_append(heads, latent, rope, bs, dtype, layout, n, rotary) -> None:
    _say(f"latent append {n} tokens {latent}+{rope} blocks of {bs} {dtype} {layout} rotary={rotary}")
    t = DTYPES[dtype]
    gen = torch.Generator(device=DEV).manual_seed(n + latent)
    blocks = -(-n // bs) + 5
    cache = _cache(heads, latent, rope, bs, blocks, t, layout=layout)
    _flat(cache).normal_(generator=gen)
    before = _np(_flat(cache))
    slots = torch.randperm(blocks * bs, generator=gen, device=DEV)[:n]
    both = torch.randn((n, latent + rope), generator=gen, device=DEV).to(t)
    angles = _angles(n, rope, gen) if rotary else None
    cache.write("layer0", both[:, :latent], both[:, latent:], slots, rotary=angles)
    torch.cuda.synchronize()
    _check_rows(cache, *_expect_rows(before, both[:, :latent], both[:, latent:], slots.tolist(), angles,
                                     layout == "interleaved"))


@pytest.mark.parametrize("validate", (True, False))
def test_append_skips_tokens_and_takes_any_strides(validate) -> None:
    _say(f"latent append, skipped tokens, odd strides, validate={validate}")
    gen = torch.Generator(device=DEV).manual_seed(9)
    cache = _cache(4, 128, 32, 16, 4, torch.bfloat16)
    slots = torch.tensor([5, -1, 63, 0, -1, 17], device=DEV)
    if not validate:
        slots[4] = 64  # (out of range: not written)
    wide = torch.randn((6, 400), generator=gen, device=DEV).to(torch.bfloat16)
    cos, sin = _angles(6, 32, gen)
    odd_angles = tuple(torch.cat((x[:, :1], x), dim=1)[:, 1:] for x in (cos, sin))
    assert odd_angles[0].stride(0) == 17
    for lat, key, rot in ((wide[:, :128], wide[:, 128:160], (cos, sin)), (wide[:, 1:129], wide[:, 131:163], odd_angles),
                          (wide.t().contiguous().t()[:, :128], wide[:, 200:264:2], (cos, sin[:, :16])),
                          (wide[:1, :128].expand(6, 128), wide[:1, 3:35].expand(6, 32), None)):
        before = _np(_flat(cache))
        mapping = cache.prepare_write(slots if validate else slots, validate=validate) if not validate else cache.prepare_write(
            torch.where(slots >= 64, -1, slots))
        cache.write_prepared("layer0", lat, key, mapping, rotary=rot)
        torch.cuda.synchronize()
        kept = [s if s < 64 else -1 for s in slots.tolist()]
        _check_rows(cache, *_expect_rows(before, lat, key, kept, rot, True))
    before = _np(_flat(cache))
    cache.write("layer0", wide[:0, :128], wide[:0, 128:160], slots[:0])
    cache.write("layer0", wide[:2, :128], wide[:2, 128:160], torch.tensor([-1, -5], device=DEV))
    torch.cuda.synchronize()
    _check_rows(cache, before, 0 * before)


def test_write_refusals() -> None:
    cache = _cache(4, 128, 32, 16, 4, torch.bfloat16)
    x, r = torch.zeros((2, 128), dtype=torch.bfloat16, device=DEV), torch.zeros((2, 32), dtype=torch.bfloat16, device=DEV)
    slots = torch.tensor([0, 1], device=DEV)
    c = torch.zeros((2, 16), device=DEV)
    for bad, message in ((torch.tensor([0, 64], device=DEV), "out-of-range"), (torch.tensor([5, 5], device=DEV), "twice"),
                         (slots.cpu(), "device must match"), (slots.view(1, 2), "one entry per packed")):
        with pytest.raises(lv.KVCacheError, match=message):
            cache.write("layer0", x, r, bad)
    mapping = cache.prepare_write(slots)
    for a, b, rot, message in ((x.half(), r, None, "dtype and device"), (x, r.half(), None, "dtype and device"),
                               (x[:, :64], r, None, "latent_size"), (x, r[:, :16], None, "rope_size"),
                               (x, r[:1], None, "rope_size"), (x[:1], r[:1], None, "one entry per query"),
                               (x.cpu(), r.cpu(), None, "dtype and device"), (x, r, (c,), "a pair"),
                               (x, r, (c, c[:1]), "sines must have shape"), (x, r, (c.half(), c), "cosines must be float32"),
                               (x, r, (c, c.cpu()), "sines must be float32"),
                               (x, r, (None, None), "cosines must have shape"), (x, r, (c, None), "sines must have shape")):
        with pytest.raises(lv.KVCacheError, match=message):
            cache.write_prepared("layer0", a, b, mapping, rotary=rot)
    with pytest.raises(lv.KVCacheError, match="int64 vectors"):
        cache.write_prepared("layer0", x, r, lv.PagedKVWriteMapping(slots.int(), 2))
    with pytest.raises(lv.KVCacheError, match="not found"):
        cache.write("other", x, r, slots)
    from light_vllm_amd.paged_cache import hip_append

    with pytest.raises(lv.KVCacheError, match="its own write_prepared"):
        hip_append(cache, "layer0", x[:, None], x[:, None], 0, 0)


def test_append_passes_over_tokens_that_are_not_there() -> None:
    """Entries of a mapping made by hand whose token or slot is out of range."""
    _say("latent append, tokens and slots out of range")
    cache = _cache(4, 128, 32, 16, 4, torch.bfloat16)
    _flat(cache).fill_(7)
    x, r = torch.ones((2, 128), dtype=torch.bfloat16, device=DEV), torch.ones((2, 32), dtype=torch.bfloat16, device=DEV)
    mapping = lv.PagedKVWriteMapping(torch.tensor([3, 5, 9, 64, -1, 11], device=DEV), 2,
                                     torch.tensor([0, 2, -1, 1, 1, 1], device=DEV))
    cache.write_prepared("layer0", x, r, mapping)
    written = torch.zeros(64, dtype=torch.bool, device=DEV)
    written[[3, 11]] = True
    assert (_flat(cache)[written] == 1).all() and (_flat(cache)[~written] == 7).all()


# ---- compact and block copies --------------------------------------------------------

@pytest.mark.parametrize("requests", (1, 3, 20))
@pytest.mark.parametrize("latent, rope, bs, layers", [(512, 64, 16, 3), (128, 32, 12, 1)])
def test_compact(latent, rope, bs, layers, requests) -> None:
    _say(f"latent compact of {requests} requests, {layers} layers of {latent}+{rope}")
    rng = np.random.default_rng(requests)
    gen = torch.Generator(device=DEV).manual_seed(requests)
    blocks = requests * 4 + 3
    cache = _cache(4, latent, rope, bs, blocks, torch.bfloat16, layers)
    for i in range(layers):
        _flat(cache, f"layer{i}").normal_(generator=gen)
    want = [_np(_flat(cache, f"layer{i}")) for i in range(layers)]
    before = [w.copy() for w in want]
    ids, reqs, moved = rng.permutation(blocks).tolist(), [], []
    for r in range(requests):
        n, computed = int(rng.integers(1, 14)), int(rng.integers(0, 2 * bs))
        need = -(-(computed + n) // bs)
        table = tuple(ids.pop() for _ in range(need))
        kept = tuple(int(x) for x in rng.permutation(n)[: int(rng.integers(0, n + 1))])
        kept = kept if r % 2 else tuple(sorted(kept))
        reqs.append(dict(block_ids=table, num_computed_tokens=computed, num_query_tokens=n, num_reserved_query_tokens=n,
                         retained_query_indices=kept))
        at = lambda p: table[p // bs] * bs + p % bs  # noqa: E731
        moved.append(sum(k != i for i, k in enumerate(kept)))
        for i, k in enumerate(kept):
            for w, b in zip(want, before):
                w[at(computed + i)] = b[at(computed + k)]
    assert cache.compact_many(reqs) == tuple(moved) if requests > 1 else cache.compact(**reqs[0]) == moved[0]
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        np.testing.assert_array_equal(_np(_flat(cache, f"layer{i}")), w)


@pytest.mark.parametrize("pairs", (1, 9, 40))
def test_block_copy(pairs) -> None:
    _say(f"latent block copy of {pairs}")
    gen = torch.Generator(device=DEV).manual_seed(pairs)
    cache = _cache(4, 256, 64, 16, 2 * pairs + 1, torch.float16, 3)
    order = torch.randperm(2 * pairs, generator=torch.Generator().manual_seed(pairs)).tolist()
    want = []
    for i in range(3):
        rows = cache.layer(f"layer{i}").rows
        rows.normal_(generator=gen)
        w = rows.clone()
        w[order[pairs:]] = rows[order[:pairs]]
        want.append(w)
    if pairs == 9:
        lv.hip_block_copy(cache, order[:pairs], order[pairs:])
    else:
        cache.copy_blocks(order[:pairs], order[pairs:])
    for i, w in enumerate(want):
        assert torch.equal(cache.layer(f"layer{i}").rows, w)
    for src, dst, message in (((0,), (0,), "disjoint"), ((0, 1), (2, 2), "twice"), ((0,), (10**6,), "invalid")):
        with pytest.raises(lv.KVCacheError, match=message):
            cache.copy_blocks(src, dst)


# ---- attention -----------------------------------------------------------------------

def _step(heads, latent, rope, bs, dtype, computed, layouts, seed, layout="interleaved", prefix=0, spare=3, layers=1):
    """A cache with history (NaN wherever no token is), tables over a shuffled pool
    (the first ``prefix`` blocks shared), and this step's tensors."""
    rng = np.random.default_rng(seed)
    layouts = [p if isinstance(p, tuple) else tuple(range(-1, p - 1)) for p in layouts]
    need = [-(-(c + len(p)) // bs) for c, p in zip(computed, layouts)]
    total = prefix + sum(n - prefix for n in need) + spare
    free = [int(b) for b in rng.permutation(total)]
    shared, free = free[:prefix], free[prefix:]
    tables = []
    for n in need:
        tables.append(tuple(shared + free[: n - prefix]))
        free = free[n - prefix:]
    cache = _cache(heads, latent, rope, bs, total, dtype, layers, layout)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    held = torch.cat([torch.tensor(t)[torch.arange(c) // bs] * bs + torch.arange(c) % bs for t, c in zip(tables, computed)]).to(DEV)
    for i in range(layers):
        rows = _flat(cache, f"layer{i}")
        rows.fill_(math.nan)
        rows[held] = torch.randn((len(held), latent + rope), generator=gen, device=DEV).to(dtype)
    t = sum(map(len, layouts))
    q = torch.randn((t, heads, latent + rope), generator=gen, device=DEV).to(dtype)
    both = torch.randn((t, latent + rope), generator=gen, device=DEV).to(dtype)
    metadata = lv.PagedAttentionMetadata(block_tables=tuple(tables), num_computed_tokens=tuple(computed),
                                         query_layouts=tuple(lv.QueryLayout(p) for p in layouts),
                                         num_readonly_prefix_blocks=(prefix,) * len(need) if prefix else ())
    return cache, metadata, q, both[:, :latent], both[:, latent:]


def _expected(cache, metadata, q, rotary, scale, layer="layer0"):
    """(attention, its bound) over the cache's rows as they are now."""
    spec = cache.layer_spec(layer)
    latent, dtype = spec.latent_size, cache.config.dtype
    u = _u(dtype)
    qn = _np(q)
    if rotary is not None:
        qn[..., latent:] = Z.rotate(qn[..., latent:], *(_np(t) for t in rotary), spec.rotary_layout == "interleaved")

    def per_key(aq, ak):
        ak = np.nan_to_num(ak, nan=0, posinf=0)
        sums = (spec.row_size + 4) * 2.0**-24 * (aq @ ak.T)
        return sums + (u + 2.0**-21) * (aq[:, latent:] @ ak[:, latent:].T) if rotary is not None else sums

    parents = [p.parent_indices for p in metadata.query_layouts]
    out, size, d = Z.attention(qn, _np(_flat(cache, layer)), metadata.block_tables, metadata.num_computed_tokens, parents,
                               cache.config.block_size, latent, scale=scale, per_key_error=per_key)
    keys = np.concatenate([np.full(len(p), c + len(p)) for c, p in zip(metadata.num_computed_tokens, parents)])
    bound = u * (2 * size + np.abs(out)) + 2 * size * np.expm1(d)[..., None] + (
        (keys / 16 + 64) * 2.0**-24)[:, None, None] * size + 2.0**-24
    return out, bound


def _check(out, want, bound, what="attention"):
    got = out.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    worst = float((np.abs(got - want)[fine] / bound[fine]).max(initial=0))
    print(f"[margin] latent {what}: {100 * worst:.1f}% of the bound", file=sys.stderr, flush=True)
    assert worst <= 1.0


def _attend_and_check(cache, metadata, q, latent, rope_key, rotary=None, scale=None, backend=None):
    spec = cache.layer_spec("layer0")
    scale = 1.0 / math.sqrt(192) if scale is None else scale
    slots = metadata.slot_mapping(block_size=cache.config.block_size, device=torch.device("cpu")).tolist()
    want, off = _expect_rows(_np(_flat(cache)), latent, rope_key, slots, rotary, spec.rotary_layout == "interleaved")
    context = (backend or lv.HipPagedAttentionBackend()).create(cache, metadata)
    assert isinstance(context, lv.HipLatentPagedAttention) and context.supports_rotary
    out = context.forward("layer0", q, latent, rope_key, scale=scale, rotary=rotary)
    torch.cuda.synchronize()
    _check_rows(cache, want, off)  # rows behind the sequences as they were
    _check(out, *_expected(cache, metadata, q, rotary, scale))
    return out


CASES = [  # heads, latent, rope, block, computed, layouts
    (16, 512, 64, 16, [301], [1]),
    (16, 512, 64, 16, [0, 1, 15, 16, 31, 32, 33, 1000], [1] * 8),
    (128, 512, 64, 16, [0, 700, 64], [1, 1, 1]),
    (1, 512, 64, 12, [5, 900], [1, 1]),
    (5, 128, 32, 1, [40, 3], [1, 7]),
    (20, 384, 64, 64, [200, 0], [2, 3]),
    (40, 256, 32, 7, [333, 64], [1, 1]),
    (16, 512, 64, 16, [100, 2000, 31], [TREE, TREE, TREE]),
    (8, 256, 64, 16, [0, 50], [TREE, 4]),
    (16, 512, 32, 32, [0, 37], [70, 33]),
    (128, 128, 64, 16, [90], [9]),
    (3, 384, 32, 16, [20], [tuple([-1] + [max(0, i - 3) for i in range(1, 80)])]),
]


@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("heads, latent, rope, bs, computed, layouts", CASES)
def test_attention(heads, latent, rope, bs, computed, layouts, dtype, wide, monkeypatch) -> None:
    """``wide``: 128 columns to a workgroup wherever a request has more than 64."""
    if wide:
        monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
    _say(f"latent attention {heads} heads {latent}+{rope} blocks of {bs} {computed} {dtype} {wide}")
    args = _step(heads, latent, rope, bs, DTYPES[dtype], computed, layouts, seed=heads + bs)
    _attend_and_check(*args)


@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("heads, latent, rope, bs, computed, layouts", CASES[1:4] + CASES[7:9])
def test_attention_with_rotation(heads, latent, rope, bs, computed, layouts, layout, wide, monkeypatch) -> None:
    if wide:
        monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
    _say(f"latent attention with rotation {heads} heads {latent}+{rope} {layout}")
    args = _step(heads, latent, rope, bs, torch.bfloat16, computed, layouts, seed=heads + rope, layout=layout)
    gen = torch.Generator(device=DEV).manual_seed(1)
    _attend_and_check(*args, rotary=_angles(args[2].shape[0], rope, gen))


def test_many_requests_and_a_long_one() -> None:
    _say("latent attention, 300 requests; one of 9000 beside short ones")
    rng = np.random.default_rng(0)
    _attend_and_check(*_step(4, 128, 32, 16, torch.bfloat16, rng.integers(0, 90, 300).tolist(), [1] * 300, seed=1))
    _attend_and_check(*_step(16, 512, 64, 16, torch.bfloat16, [9000, 3, 40], [1, 2, 1], seed=2))


def test_shared_prefix_blocks() -> None:
    _say("latent attention, shared prefix blocks")
    _attend_and_check(*_step(16, 512, 64, 16, torch.bfloat16, [70, 64, 100], [1, 3, TREE], seed=3, prefix=4))


def test_scores_that_spread_far() -> None:
    """Large scores of both signs, so that the maximum moves at many tiles, and a
    scale that is negative or zero."""
    _say("latent attention, large scores")
    for scale in (2.0, -1.0, 0.0):
        cache, md, q, latent, rope_key = _step(16, 256, 64, 16, torch.bfloat16, [400, 90], [1, 5], seed=4)
        _attend_and_check(cache, md, q, latent, rope_key, scale=scale)


def test_strided_queries() -> None:
    _say("latent attention, strided queries")
    cache, md, q, latent, rope_key = _step(6, 256, 32, 16, torch.bfloat16, [30, 64], [1, 5], seed=5)
    want = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.1)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.cat((q[..., :1], q), dim=2)[..., 1:]
    every_other = torch.stack((q, q), dim=-1).flatten(2)[..., ::2]
    for view in (heads_first, odd, every_other):
        assert view.stride() != q.stride()
        assert torch.equal(lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", view, latent, rope_key, scale=0.1), want)


@pytest.mark.parametrize("value", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("wide", (False, True))
@pytest.mark.parametrize("heads, layouts", [(16, [TREE, 6]), (3, [tuple([-1] + [0] * 40), 40])])
def test_values_that_are_not_finite_stay_where_they_are_seen(heads, layouts, value, wide, monkeypatch) -> None:
    """A draft or later token whose row is not finite does not reach the queries
    that do not see it; those that see it follow the formula."""
    if wide:
        monkeypatch.setattr(latent_attention, "WIDE_TILES", 0)
    _say(f"latent attention, {value} in a masked row, {heads} heads")
    cache, md, q, latent, rope_key = _step(heads, 256, 64, 16, torch.bfloat16, [20, 33], layouts, seed=6)
    latent, rope_key = latent.clone(), rope_key.clone()
    n = len(md.query_layouts[0])
    latent[n - 2, 3] = value      # the first request's last but one
    rope_key[n + len(md.query_layouts[1]) - 1, 5] = value  # the second's last
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07)
    want, bound = _expected(cache, md, q, None, 0.07)
    assert np.isnan(want).any() and not np.isnan(want).all(axis=(1, 2)).all()
    _check(out, want, bound)


def test_two_layers_share_a_plan_and_layers_run_once() -> None:
    _say("latent attention, two layers, refusals")
    cache, md, q, latent, rope_key = _step(16, 512, 64, 16, torch.bfloat16, [40, 7], [1, 2], seed=7, layers=2)
    context = lv.HipPagedAttentionBackend().create(cache, md)
    outs = [context.forward(f"layer{i}", q, latent, rope_key, scale=0.07) for i in range(2)]
    for i in range(2):
        _check(outs[i], *_expected(cache, md, q, None, 0.07, f"layer{i}"))
    assert context.layer_ids == {"layer0", "layer1"}
    with pytest.raises(lv.KVCacheError, match="more than once"):
        context.forward("layer0", q, latent, rope_key, scale=0.07)
    with pytest.raises(lv.KVCacheError, match="not found"):
        context.forward("layer7", q, latent, rope_key, scale=0.07)
    c = torch.zeros((3, 32), device=DEV)
    for args, kw, message in (
        ((q[0], latent, rope_key), {}, "three dimensions"), ((q[:2], latent[:2], rope_key[:2]), {}, "token count"),
        ((q[:, :8], latent, rope_key), {}, "query shape"), ((q, latent[:2], rope_key[:2]), {}, "token dimensions"),
        ((q.half(), latent, rope_key), {}, "query dtype"), ((q, latent.half(), rope_key), {}, "update dtype"),
        ((q, latent, rope_key[:, :16]), {}, "rope_size"), ((q, latent, rope_key), dict(rotary=(c, c[:2])), "sines"),
    ):
        with pytest.raises(lv.KVCacheError, match=message):
            lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", *args, scale=0.07, **kw)
    bad = lv.PagedAttentionMetadata(block_tables=((0,), (10**6,)), num_computed_tokens=(3, 3),
                                    query_layouts=(lv.linear_query_layout(1),) * 2)
    with pytest.raises(lv.KVCacheError, match="out-of-range"):
        lv.HipPagedAttentionBackend().create(cache, bad)


def test_layers_of_both_rotary_layouts_share_a_plan() -> None:
    """Layers that differ in the layout alone take the same work lists, each its own turn."""
    _say("latent attention, layers of both layouts")
    layouts = ("interleaved", "half", "interleaved")
    one = {kind: _step(16, 256, 64, 16, torch.bfloat16, [33, 7], [1, TREE], seed=9, layout=kind) for kind in layouts}
    cache, md, q, latent, rope_key = one["half"]
    spec = lv.LatentKVCacheSpec(tuple(lv.LatentLayerSpec(f"layer{i}", 16, 256, 64, k) for i, k in enumerate(layouts)))
    many = lv.LatentPagedKVCache(spec, cache.config)
    for i in range(3):
        many.layer(f"layer{i}").rows.copy_(cache.layer("layer0").rows)
    rotary = _angles(q.shape[0], 64, torch.Generator(device=DEV).manual_seed(1))
    want = {kind: lv.HipPagedAttentionBackend().create(one[kind][0], md).forward(
        "layer0", q, latent, rope_key, scale=0.1, rotary=rotary) for kind in layouts[:2]}
    assert not torch.equal(want["half"], want["interleaved"])
    backend = lv.HipPagedAttentionBackend()
    for order in ((0, 1, 2), (1, 0, 2)):
        context = backend.create(many, md)
        for i in order:
            out = context.forward(f"layer{i}", q, latent, rope_key, scale=0.1, rotary=rotary)
            assert torch.equal(out, want[layouts[i]])
            a, b = (c.layer(name).rows.view(torch.int16) for c, name in ((many, f"layer{i}"), (one[layouts[i]][0], "layer0")))
            assert torch.equal(a, b)


def test_columns_past_32_bits_are_refused() -> None:
    cache, md, *_ = _step(1, 128, 32, 16, torch.bfloat16, [3], [2], seed=1)
    wide = lv.LatentPagedKVCache(lv.LatentKVCacheSpec((lv.LatentLayerSpec("layer0", 2**30, 128, 32, "half"),)), cache.config)
    with pytest.raises(lv.KVCacheError, match="below 2"):
        lv.HipPagedAttentionBackend().create(wide, md)


def test_graph_replays_and_streams() -> None:
    """A captured step replays with new inputs, with eager steps of the same
    backend between; two streams run steps of one backend at once."""
    _say("latent attention, captured and on two streams")
    cache, md, q, latent, rope_key = _step(16, 512, 64, 16, torch.bfloat16, [700, 1500, 90], [1, 3, TREE], seed=8)
    other = _step(16, 512, 64, 16, torch.bfloat16, [2500, 9], [1, 1], seed=9)
    gen = torch.Generator(device=DEV).manual_seed(3)
    rotary = _angles(q.shape[0], 64, gen)
    latent, rope_key = latent.clone(), rope_key.clone()
    backend = lv.HipPagedAttentionBackend()
    want_other = backend.create(other[0], other[1]).forward("layer0", *other[2:], scale=0.07)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        backend.create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07, rotary=rotary)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    context = backend.create(cache, md)
    with torch.cuda.graph(graph):
        out = context.forward("layer0", q, latent, rope_key, scale=0.07, rotary=rotary)
    for i in range(4):
        for t in (q, latent, rope_key):
            t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        graph.replay()
        got = backend.create(other[0], other[1]).forward("layer0", *other[2:], scale=0.07)
        torch.cuda.synchronize()
        assert torch.equal(got, want_other)
        _check(out, *_expected(cache, md, q, rotary, 0.07))
        eager = backend.create(cache, md).forward("layer0", q, latent, rope_key, scale=0.07, rotary=rotary)
        assert torch.equal(eager, out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [[backend.create(c, m) for _ in range(6)] for c, m in ((cache, md), (other[0], other[1]))]
    torch.cuda.synchronize()
    outs = [[], []]
    for k in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i == 0:
                    outs[0].append(contexts[0][k].forward("layer0", q, latent, rope_key, scale=0.07, rotary=rotary))
                else:
                    outs[1].append(contexts[1][k].forward("layer0", *other[2:], scale=0.07))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs[0]) and all(torch.equal(o, want_other) for o in outs[1])


def test_a_speculative_step_end_to_end() -> None:
    """Angles, write, tree attention, compact, and the next step on what was kept."""
    _say("latent speculative step")
    cache, md, q, latent, rope_key = _step(16, 512, 64, 16, torch.bfloat16, [37, 90], [TREE, TREE], seed=10)
    emb = lv.RotaryEmbedding(64, scaling=lv.RotaryScaling("ramp", 8.0), device=DEV)
    layout = md.query_layouts[0]
    positions = torch.tensor([p for c in md.num_computed_tokens for p in lv.semantic_positions(layout, prefix_length=c)], device=DEV)
    backend = lv.HipPagedAttentionBackend()
    _attend_and_check(cache, md, q, latent, rope_key, rotary=emb(positions), backend=backend)
    kept = (0, 1, 3, 6)
    held = [_flat(cache)[[t[(c + i) // 16] * 16 + (c + i) % 16 for i in kept]].clone()
            for t, c in zip(md.block_tables, md.num_computed_tokens)]
    moved = cache.compact_many([dict(block_ids=t, num_computed_tokens=c, num_query_tokens=9, num_reserved_query_tokens=9,
                                     retained_query_indices=kept) for t, c in zip(md.block_tables, md.num_computed_tokens)])
    assert moved == (2, 2)
    for rows, t, c in zip(held, md.block_tables, md.num_computed_tokens):
        assert torch.equal(_flat(cache)[[t[p // 16] * 16 + p % 16 for p in range(c, c + 4)]], rows)
    after = [c + 4 for c in md.num_computed_tokens]
    nxt = lv.PagedAttentionMetadata(block_tables=tuple(t[: -(-(c + 1) // 16)] for t, c in zip(md.block_tables, after)),
                                    num_computed_tokens=tuple(after), query_layouts=(lv.linear_query_layout(1),) * 2)
    positions = torch.tensor(after, device=DEV)
    _attend_and_check(cache, nxt, q[:2], latent[:2], rope_key[:2], rotary=emb(positions), backend=backend)
