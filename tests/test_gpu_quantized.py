"""GPU: the 8-bit paged cache against the fp64 oracle: the quantising append and
the compact code for code, attention over the cache, block copies, and a
speculative step through all of them.

Attention's tolerance, from the roundings on the way: probabilities are rounded
to the step's type before the products (half a step of their value, u = eps / 2),
so is the output; a sum of |p v| / sum p bounds what the first can move, and the
output's own value the second.  The fp32 scores are off by at most (D + 4) 2^-24
sum |q k| scale, which moves p by that share: 2^-12 of sum |p v| for the sizes
here (sum |q k| scale < 20).  In all: u (2 A + |out|) + 2^-12 A + 2^-24, with
A = attention of |v|.
"""

from __future__ import annotations

import math
import sys

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
from oracle import paged_kv_oracle as O
from oracle import quantized_oracle as Q

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

DEV = torch.device("cuda:0")
LARGEST = {torch.bfloat16: 1.875 * 2.0**127, torch.float16: 61440.0}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _cache(hq, hkv, d, bs, blocks, dtype, layers=1):
    spec = lv.ModelKVCacheSpec(tuple(lv.AttentionLayerSpec(f"layer{i}", hq, hkv, d) for i in range(layers)))
    return lv.QuantizedPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=blocks, block_size=bs, dtype=dtype, device=DEV))


def _fill(cache, seed):
    """Random codes (no NaN) and scales 2^-8 .. 2^2 in every block."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for spec in cache.model_spec.layers:
        layer = cache.layer(spec.layer_id)
        for codes, scales in ((layer.keys, layer.key_scales), (layer.values, layer.value_scales)):
            codes.copy_((torch.randn(codes.shape, generator=gen, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn))
            scales.copy_(torch.exp2(torch.randint(-8, 3, scales.shape, generator=gen, device=DEV).float()))


def _state(cache, layer_id="layer0"):
    layer = cache.layer(layer_id)
    return [[t.double().cpu().numpy() for t in pair]
            for pair in ((layer.keys, layer.key_scales), (layer.values, layer.value_scales))]


def _same(cache, want, layer_id="layer0"):
    for name, got, expect in zip("KV", _state(cache, layer_id), want):
        np.testing.assert_array_equal(got[1], expect[1], err_msg=f"{name} scales")
        np.testing.assert_array_equal(got[0], expect[0], err_msg=f"{name} codes")


def _write_and_compare(cache, key, value, slots, layer_id="layer0", **kw):
    want = _state(cache, layer_id)
    for (codes, scales), rows in zip(want, (key, value)):
        Q.append(codes, scales, rows.double().cpu().numpy(), slots.tolist(), LARGEST[key.dtype])
    mapping = cache.prepare_write(slots, **kw)
    cache.write_prepared(layer_id, key, value, mapping)
    torch.cuda.synchronize()
    _same(cache, want, layer_id)


def _rows(gen, n, heads, d, dtype, spread=3):
    x = torch.randn((n, heads, d), generator=gen, device=DEV)
    return (x * torch.exp2(torch.randint(-spread, spread + 1, (n, 1, 1), generator=gen, device=DEV).float())).to(dtype)


# ---- append --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("heads,d,bs", [(1, 32, 16), (4, 128, 16), (2, 80, 12), (3, 48, 4), (2, 256, 64), (5, 112, 1), (1, 240, 7), (2, 64, 100)])
def test_append_matches_the_oracle(heads, d, bs, dtype) -> None:
    print(f"[gpu] q8 append {heads}x{d} blocks of {bs} {dtype}", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(heads * 1000 + d + bs)
    cache = _cache(2 * heads, heads, d, bs, 24, DTYPES[dtype])
    _fill(cache, d)
    rng = np.random.default_rng(d + bs)
    runs = [(0, 1), (bs - 1, 1), (bs // 2, 2 * bs + 1), (3 * bs, bs), (bs // 3, 1)]  # (first offset, tokens) in own blocks
    blocks, slots = list(rng.permutation(24)), []
    for start, n in runs:
        need = -(-(start + n) // bs)
        own = [blocks.pop() for _ in range(min(need, len(blocks)))]
        slots += [own[p // bs] * bs + p % bs for p in range(start, start + n) if p // bs < len(own)]
    slots = torch.tensor(slots, device=DEV)
    k, v = (_rows(gen, len(slots), heads, d, DTYPES[dtype]) for _ in range(2))
    _write_and_compare(cache, k, v, slots)


@pytest.mark.parametrize("validate", (True, False))
def test_append_skips_negative_slots_and_takes_strided_rows(validate) -> None:
    print(f"[gpu] q8 append negative slots, strided rows, validate={validate}", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(5)
    cache = _cache(8, 2, 64, 16, 9, torch.bfloat16)
    _fill(cache, 1)
    slots = torch.tensor([-1, 3, 4, 5, -1, 17, -1, 32, 33, -1], device=DEV)
    packed = _rows(gen, len(slots), 12, 64, torch.bfloat16)  # a projection's Q, K and V
    _write_and_compare(cache, packed[:, 8:10], packed[:, 10:], slots, validate=validate)
    odd = _rows(gen, len(slots), 2, 65, torch.bfloat16)[:, :, 1:]  # rows of no 16-byte chunks
    _write_and_compare(cache, odd, odd, slots, validate=validate)
    _write_and_compare(cache, packed[:0, 8:10], packed[:0, 10:], slots[:0], validate=validate)


def test_one_token_of_an_odd_row() -> None:
    """One token and one kv head: strides of single elements, which no copy of
    theirs changes by itself, are no multiple of 16 bytes."""
    print("[gpu] q8 one token, one kv head, odd strides", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(31)
    cache = _cache(1, 1, 32, 16, 3, torch.bfloat16)
    x = _rows(gen, 1, 1, 133, torch.bfloat16).view(1, 133)
    odd = x[:, None, :32]
    assert odd.stride(1) % 8
    _write_and_compare(cache, odd, odd, torch.tensor([17], device=DEV))
    _write_and_compare(cache, x[:, None, 1:33], odd, torch.tensor([18], device=DEV))
    cache, md, q, k, v = _step(1, 1, 32, 16, torch.bfloat16, [40], [1], seed=31)
    want = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", odd.clone(), odd.clone(), odd.clone(), scale=0.2)
    for views in ((odd, odd, odd), (odd, odd.contiguous().view(-1)[None, None], odd)):
        assert torch.equal(lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", *views, scale=0.2), want)


def test_append_in_any_order_of_slots() -> None:
    print("[gpu] q8 append shuffled slots", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(6)
    cache = _cache(4, 2, 128, 16, 40, torch.bfloat16)
    _fill(cache, 2)
    order = torch.from_numpy(np.random.default_rng(3).permutation(640)[:300]).to(DEV)
    k, v = (_rows(gen, 300, 2, 128, torch.bfloat16) for _ in range(2))
    _write_and_compare(cache, k, v, order)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
def test_append_of_special_values(dtype) -> None:
    print(f"[gpu] q8 append special values {dtype}", file=sys.stderr, flush=True)
    t = DTYPES[dtype]
    cache = _cache(4, 2, 32, 16, 12, t)
    _fill(cache, 3)
    top = torch.finfo(t).max
    x = torch.zeros((12, 2, 32), dtype=t, device=DEV)
    x[1, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
    x[2] = math.nan                       # a row of NaN: the scale is that of zeros
    x[3, :, 0] = top                      # rounds past the largest value
    x[3, :, 1] = -top
    x[4, :, 2] = torch.finfo(t).tiny
    x[5, :, 3] = torch.finfo(t).smallest_normal / 4
    x[6] = 448.0
    x[7] = 449.0
    x[8] = -0.0
    x[9, 0] = 2.0**-100 if dtype == "bf16" else 2.0**-24
    x[10, 1] = torch.linspace(-1, 1, 32)
    x[11] = 1.0
    slots = torch.arange(12, device=DEV) * 16  # every row starts a block
    _write_and_compare(cache, x, x.flip(0), slots)
    _write_and_compare(cache, x.roll(1, 0), x, slots + 1)  # and meets one that is there


def test_token_by_token_append_equals_the_whole_prompt() -> None:
    print("[gpu] q8 append token by token", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(7)
    # (Magnitudes 1..2 times 2^-3..2^3: no code becomes subnormal.)
    x = (1 + torch.rand((40, 2, 64), generator=gen, device=DEV)) * torch.exp2(
        torch.randint(-3, 4, (40, 1, 1), generator=gen, device=DEV).float())
    x = x.to(torch.bfloat16)
    whole, one = (_cache(4, 2, 64, 16, 3, torch.bfloat16) for _ in range(2))
    slots = torch.arange(40, device=DEV)
    whole.write("layer0", x, x, slots)
    for i in range(40):
        one.write("layer0", x[i : i + 1], x[i : i + 1], slots[i : i + 1])
    torch.cuda.synchronize()
    _same(one, _state(whole))


def _bound(rows, scale):
    """What the cache states of a row's error at its block's scale."""
    return 2.0**-4 * rows.abs() + 2.0**-9 * scale


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
def test_growing_scales_stay_within_the_stated_bound(dtype) -> None:
    # A token at a time, each larger than those before: codes become subnormal.
    print(f"[gpu] q8 append, growing scales {dtype}", file=sys.stderr, flush=True)
    t = DTYPES[dtype]
    gen = torch.Generator(device=DEV).manual_seed(34)
    cache = _cache(8, 4, 64, 16, 2, t)
    size = torch.exp2(torch.rand((16, 4, 1), generator=gen, device=DEV).mul(14).sort(dim=0).values)
    x = ((torch.rand((16, 4, 64), generator=gen, device=DEV) * 2 - 1) * size).to(t)
    for i in range(16):
        _write_and_compare(cache, x[i : i + 1], x[i : i + 1].flip(2), torch.tensor([i], device=DEV))
    layer = cache.layer("layer0")
    for codes, scales, rows in ((layer.keys, layer.key_scales, x), (layer.values, layer.value_scales, x.flip(2))):
        scale = scales[0, :, None]
        err = (codes[0].float() * scale - rows.float()).abs()
        assert float((err / _bound(rows.float(), scale)).max()) < 1.0
        assert float((err / _bound(rows.float(), 0 * scale)).nan_to_num().max()) > 1.0  # (the second term counts)


def test_a_rejected_drafts_scale_stays() -> None:
    """A draft that is far larger than the history of its block raises the block's
    scale for all its rows, and its rejection does not lower it: the history keeps
    the stated bound, at that scale.  Other blocks and heads are as they were."""
    print("[gpu] q8 a rejected draft of 2^14", file=sys.stderr, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(35)
    cache = _cache(4, 2, 64, 16, 3, torch.bfloat16)
    x = torch.randn((26, 2, 64), generator=gen, device=DEV).to(torch.bfloat16)
    cache.write("layer0", x, x, torch.arange(26, device=DEV))
    layer = cache.layer("layer0")
    before = [t.clone() for t in (layer.keys.float(), layer.key_scales)]
    drafts = torch.randn((3, 2, 64), generator=gen, device=DEV).to(torch.bfloat16)
    drafts[2, 0, 7] = 2.0**14
    md = lv.PagedAttentionMetadata(block_tables=((0, 1),), num_computed_tokens=(26,), query_layouts=(lv.QueryLayout((-1, 0, 0)),))
    q = torch.randn((3, 4, 64), generator=gen, device=DEV).to(torch.bfloat16)
    want = _state(cache)
    for codes, scales in want:
        Q.append(codes, scales, drafts.double().cpu().numpy(), [26, 27, 28], LARGEST[torch.bfloat16])
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, drafts, drafts, scale=0.125)
    _same(cache, want)
    _check(out[:2], *(e[:2] for e in _expected(cache, md, q, want)), torch.bfloat16)
    assert cache.compact(block_ids=(0, 1), num_computed_tokens=26, num_query_tokens=3, num_reserved_query_tokens=3,
                         retained_query_indices=(0, 1)) == 0
    torch.cuda.synchronize()
    scale = layer.key_scales
    assert float(scale[1, 0]) == 64.0 and float(scale[1, 1]) == float(before[1][1, 1])
    assert torch.equal(scale[0], before[1][0]) and torch.equal(layer.keys.float()[0], before[0][0])
    held = layer.keys[1, :10].float() * scale[1][None, :, None]
    err = (held - x[16:].float()).abs()
    assert float((err / _bound(x[16:].float(), scale[1][None, :, None])).max()) < 1.0
    assert float(err[:, 0].max()) > 0.03125  # the price: steps of 2^-9 x 64 instead of 2^-9 x 2^-6


def test_write_refusals() -> None:
    cache = _cache(4, 2, 64, 16, 4, torch.bfloat16)
    x = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=DEV)
    slots = torch.tensor([0, 1], device=DEV)
    for bad, message in ((torch.tensor([0, 64], device=DEV), "out-of-range"), (torch.tensor([5, 5], device=DEV), "twice"),
                         (slots.cpu(), "device must match"), (slots.view(1, 2), "one entry per packed")):
        with pytest.raises(lv.KVCacheError, match=message):
            cache.write("layer0", x, x, bad)
    mapping = cache.prepare_write(slots)
    for k, v, m, message in ((x.half(), x.half(), mapping, "dtype and device"), (x, x.half(), mapping, "same dtype"),
                             (x[:, :1], x[:, :1], mapping, "must have shape"), (x[:1], x[:1], mapping, "one entry per query"),
                             (x, x, lv.PagedKVWriteMapping(slots, 2), "of its own prepare_write")):
        with pytest.raises(lv.KVCacheError, match=message):
            cache.write_prepared("layer0", k, v, m)
    with pytest.raises(lv.KVCacheError, match="not found"):
        cache.write("other", x, x, slots)


# ---- attention -------------------------------------------------------------------

def _step(hq, hkv, d, bs, dtype, computed, layouts, seed, layers=1, spare=7, prefix=0):
    """A cache with history in every block, tables over a shuffled pool (the
    first ``prefix`` blocks shared), and this step's tensors."""
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
    cache = _cache(hq, hkv, d, bs, total, dtype, layers)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for spec in cache.model_spec.layers:
        layer = cache.layer(spec.layer_id)
        for codes, scales in ((layer.keys, layer.key_scales), (layer.values, layer.value_scales)):
            x = torch.randn(codes.shape, generator=gen, device=DEV)
            scales.copy_(torch.exp2(torch.randint(-9, -6, scales.shape, generator=gen, device=DEV).float()))
            codes.copy_((x / scales[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn))
    t = sum(map(len, layouts))
    q = torch.randn((t, hq, d), generator=gen, device=DEV).to(dtype)
    k, v = (torch.randn((t, hkv, d), generator=gen, device=DEV).to(dtype) for _ in range(2))
    metadata = lv.PagedAttentionMetadata(block_tables=tuple(tables), num_computed_tokens=tuple(computed),
                                         query_layouts=tuple(lv.QueryLayout(p) for p in layouts),
                                         num_readonly_prefix_blocks=(prefix,) * len(need) if prefix else ())
    return cache, metadata, q, k, v


def _slots(metadata, bs):
    return metadata.slot_mapping(block_size=bs, device=torch.device("cpu"))


def _expected(cache, metadata, q, state):
    """(attention, attention of |v|) in fp64 over the cache's state."""
    (k, ks), (v, vs) = state
    k, v = k * ks[:, None, :, None], v * vs[:, None, :, None]
    parents = [l.parent_indices for l in metadata.query_layouts]
    qn = q.double().cpu().numpy()
    scale = 1.0 / math.sqrt(q.shape[2])
    args = (metadata.block_tables, metadata.num_computed_tokens, parents)
    return (O.dense_attention(qn, k, v, *args, scale=scale), O.dense_attention(qn, k, np.abs(v), *args, scale=scale))


def _check(out, expect, size, dtype):
    u = torch.finfo(dtype).eps / 2
    err = np.abs(out.double().cpu().numpy() - expect)
    bound = u * (2 * size + np.abs(expect)) + 2.0**-12 * size + 2.0**-24
    worst = float((err / bound).max())
    print(f"[margin] q8 attention: {100 * worst:.1f}% of the bound", file=sys.stderr, flush=True)
    assert worst <= 1.0


def _attend_and_check(cache, metadata, q, k, v, dtype, backend=None):
    bs = cache.config.block_size
    want = _state(cache)
    for (codes, scales), rows in zip(want, (k, v)):
        Q.append(codes, scales, rows.double().cpu().numpy(), _slots(metadata, bs).tolist(), LARGEST[dtype])
    context = (backend or lv.HipPagedAttentionBackend()).create(cache, metadata)
    assert isinstance(context, lv.HipQuantizedPagedAttention) and not context.supports_rotary
    out = context.forward("layer0", q, k, v, scale=1.0 / math.sqrt(q.shape[2]))
    torch.cuda.synchronize()
    _same(cache, want)  # code for code, rows behind the sequences as they were
    _check(out, *_expected(cache, metadata, q, want), dtype)
    return out


TREE = (-1, 0, 0, 1, 1, 2, 3, 0, 7)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("hq,hkv,d,bs,computed,layouts", [
    (28, 4, 128, 16, [0, 1, 15, 16, 63, 64, 700, 2000], [1] * 8),     # decode around block and tile borders
    (14, 2, 64, 16, [37, 128, 511, 0], [1, 1, 1, 1]),
    (8, 8, 64, 4, [5, 130, 33], [1, 2, 3]),                             # group 1, short runs
    (16, 2, 80, 12, [100, 255, 7], [1, 2, 1]),
    (8, 2, 256, 64, [300, 31], [1, 1]),
    (32, 1, 64, 16, [200, 90], [1, 1]),                                 # one kv head of 32: the prefill kernel
    (16, 1, 32, 16, [1000, 3], [1, 1]),
    (12, 2, 128, 16, [0, 100, 511], [65, 128, 40]),                     # prompts, whole and continued
    (12, 2, 128, 16, [300, 64, 1000], [TREE, TREE, TREE]),
    (4, 2, 96, 1, [50, 9], [TREE, 17]),                                 # blocks of one token
    (6, 2, 112, 100, [250, 30], [(-1, 0, 0), 5]),
    (4, 4, 176, 16, [90, 400], [33, 1]),
])
def test_attention_matches_the_oracle(hq, hkv, d, bs, computed, layouts, dtype) -> None:
    print(f"[gpu] q8 attention {hq}/{hkv}x{d} bs {bs} {dtype} {computed} {layouts}", file=sys.stderr, flush=True)
    _attend_and_check(*_step(hq, hkv, d, bs, DTYPES[dtype], computed, layouts, seed=d + bs + len(computed)), DTYPES[dtype])


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("hq,hkv,d,bs,computed,layouts", [
    (8, 2, 128, 16, [0, 1, 15, 16, 47, 63, 64, 700], [1, 2, 3, 4, 1, 4, 4, 1]),
    (4, 4, 64, 32, [0, 5, 31, 120, 127, 128, 1000], [16, 16, 9, 16, 16, 1, 1]),     # runs over a block's and a tile's end
    (4, 4, 32, 1, [3, 127, 200], [16, 7, 1]),                                         # sixteen blocks of one token
    (6, 2, 80, 64, [10, 60, 130], [(-1, 0, 0), 5, 1]),
    (4, 2, 256, 4, [30, 29, 700], [8, 1, 3]),
    (3, 3, 112, 8, [50, 100], [(-1, 0, 0, 1, 1, 2, 3, 0, 7), 12]),
    (2, 2, 64, 128, [100, 200], [16, 1]),
])
def test_append_inside_the_decode_launch(monkeypatch, hq, hkv, d, bs, computed, layouts, dtype) -> None:
    """The same codes, scales and rows, bit for bit, as with a launch for the
    append, for tokens that raise their block's scale by 2^-1 .. 2^12 or not at all."""
    print(f"[gpu] q8 decode appends {hq}/{hkv}x{d} bs {bs} {dtype}", file=sys.stderr, flush=True)
    t = DTYPES[dtype]
    cache, metadata, q, k, v = _step(hq, hkv, d, bs, t, computed, layouts, seed=d + bs)
    gen = torch.Generator(device=DEV).manual_seed(d)
    k, v = (x * torch.exp2(torch.randint(-8, 5, (x.shape[0], hkv, 1), generator=gen, device=DEV).float()).to(t) for x in (k, v))
    q = q / 16  # (keys of up to 2^4 times the usual: the scores' bound holds)
    layer = cache.layer("layer0")
    parts = (layer.keys.view(torch.uint8), layer.key_scales, layer.values.view(torch.uint8), layer.value_scales)
    before = [p.clone() for p in parts]
    found = []
    for units in (1 << 20, 0):
        for p, b in zip(parts, before):
            p.copy_(b)
        monkeypatch.setattr(sys.modules["light_vllm_amd.backend"], "_APPEND_UNITS", units)
        found.append([_attend_and_check(cache, metadata, q, k, v, t).view(torch.int16).clone()] + [p.clone() for p in parts])
    for a, b in zip(*found):
        assert torch.equal(a, b)
    # NaN and infinities among the tokens: the same once more.
    k[0, 0, 1], v[-1, 0, 2], v[0, -1, 3], v[0, -1, 4] = math.nan, math.nan, math.inf, -math.inf
    found = []
    for units in (1 << 20, 0):
        for p, b in zip(parts, before):
            p.copy_(b)
        monkeypatch.setattr(sys.modules["light_vllm_amd.backend"], "_APPEND_UNITS", units)
        out = lv.HipPagedAttentionBackend().create(cache, metadata).forward("layer0", q, k, v, scale=1 / math.sqrt(d))
        found.append([torch.nan_to_num(out, nan=-7.0)] + [p.clone() for p in parts])
    assert bool((found[0][0] == -7.0).any())
    for a, b in zip(*found):
        assert torch.equal(a, b)


@pytest.mark.parametrize("d", range(32, 257, 16))
def test_every_head_size(d) -> None:
    print(f"[gpu] q8 attention head size {d}", file=sys.stderr, flush=True)
    for dtype in (torch.bfloat16, torch.float16):
        _attend_and_check(*_step(6, 2, d, 16, dtype, [333, 70, 90], [1, (-1, 0, 0), 50], seed=d), dtype)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("d", (80, 96, 112, 128))
def test_units_of_256_columns(monkeypatch, d, dtype) -> None:
    """Chunks and trees in units of 256 columns (large chunks only, by the backend's
    rule): more and fewer columns than a unit, split key ranges, NaN."""
    print(f"[gpu] q8 attention, 256 columns, head size {d} {dtype}", file=sys.stderr, flush=True)
    t = DTYPES[dtype]
    monkeypatch.setattr(sys.modules["light_vllm_amd.backend"], "_quantized_columns", lambda *a: 256)
    rng = np.random.default_rng(d)
    tree = tuple([-1] + [int(rng.integers(0, i)) for i in range(1, 70)])
    _attend_and_check(*_step(12, 2, d, 16, t, [0, 100, 1500, 7], [130, 41, tree, 1], seed=d), t)
    _attend_and_check(*_step(4, 1, d, 12, t, [5000], [90], seed=d + 1), t)
    _attend_and_check(*_step(12, 2, d, 16, t, [256 + 5 * i for i in range(6)], [50] * 6, seed=d + 2, prefix=16), t)
    cache, metadata, q, k, v = _step(6, 2, d, 16, t, [40], [60], seed=d + 3)
    v[50, 1, 5] = math.nan
    out = lv.HipPagedAttentionBackend().create(cache, metadata).forward("layer0", q, k, v, scale=1 / math.sqrt(d))
    nan = torch.isnan(out)
    assert bool(nan[50:, 3:, 5].all()) and int(nan.sum()) == 10 * 3


def test_unit_width_rule() -> None:
    import light_vllm_amd.backend as B

    def width(c, n, hq=28, hkv=4, d=128, requests=1):
        spec = lv.AttentionLayerSpec("l", hq, hkv, d)
        blocks = -(-(c + n) // 64)
        md = lv.PagedAttentionMetadata(
            block_tables=tuple(tuple(range(i * blocks, (i + 1) * blocks)) for i in range(requests)),
            num_computed_tokens=(c,) * requests, query_layouts=(lv.QueryLayout(tuple(range(-1, n - 1))),) * requests)
        return B._quantized_columns(B.facts_of(md), spec, 2)

    assert width(5000, 1) == width(100, 9) == 64 and width(100, 10) == 128
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert width(14336, 2048) == width(0, 4096) == width(2048, 512, requests=4) == 256
        assert width(0, 2048) == width(14336, 1536) == width(14336, 2048, d=64) == width(14336, 2048, d=144) == 128


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
def test_weights_are_summed_as_they_are_multiplied(dtype) -> None:
    """Values of 0.5 and 0.5625: the sum that divides is that of the rounded weights,
    so a weight's rounding moves the result o by its share of v - o, not of v.

    Bound: the output's rounding, half a step in [0.5, 1), which is u / 2; the
    weights', u A with A = sum p |v - o| / sum p, and as in the module's bound 2^-12 A
    for the scores; a few sums in fp32, 2^-20; and (1 + 2 u) for the divisor."""
    print(f"[gpu] q8 attention, nearly equal values {dtype}", file=sys.stderr, flush=True)
    t = DTYPES[dtype]
    u = torch.finfo(t).eps / 2
    for computed, layouts in (([0, 1, 2, 3, 4, 5, 6, 9] * 4, [1] * 32), ([1, 2, 70], [2, 1, 4]), ([0, 3, 500], [20, 30, 17])):
        cache, md, q, k, v = _step(8, 4, 64, 16, t, computed, layouts, seed=32)
        layer = cache.layer("layer0")
        gen = torch.Generator(device=DEV).manual_seed(33)
        pick = lambda shape: 0.5 + 0.0625 * torch.randint(0, 2, shape, generator=gen, device=DEV).float()  # noqa: E731
        layer.values.copy_((pick(layer.values.shape) / layer.value_scales[:, None, :, None]).to(torch.float8_e4m3fn))
        v = pick(v.shape).to(t)
        want = _state(cache)
        for (codes, scales), rows in zip(want, (k, v)):
            Q.append(codes, scales, rows.double().cpu().numpy(), _slots(md, 16).tolist(), LARGEST[t])
        out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, k, v, scale=0.125).double().cpu().numpy()
        keys, values = (codes * scales[:, None, :, None] for codes, scales in want)
        args = (md.block_tables, md.num_computed_tokens, [l.parent_indices for l in md.query_layouts])
        expect = O.dense_attention(q.double().cpu().numpy(), keys, values, *args, scale=0.125)
        # sum p |v - o| / sum p: the share of 0.5625 is x = (o - 0.5) / 0.0625, so 2 x (1 - x) 0.0625.
        assert expect.min() > 0.5 - 1e-12 and expect.max() < 0.5625 + 1e-12
        x = (expect - 0.5) / 0.0625
        bound = u / 2 + (1 + 2 * u) * (u + 2.0**-12) * 0.125 * x * (1 - x) + 2.0**-20
        worst = float((np.abs(out - expect) / bound).max())
        print(f"[margin] q8 nearly equal values: {100 * worst:.1f}% of the bound", file=sys.stderr, flush=True)
        assert worst <= 1.0


def test_long_tree_and_deep_split() -> None:
    print("[gpu] q8 attention trees of 40 and 70 queries, one long sequence", file=sys.stderr, flush=True)
    rng = np.random.default_rng(8)
    trees = [tuple([-1] + [int(rng.integers(0, i)) for i in range(1, n)]) for n in (40, 70)]
    _attend_and_check(*_step(4, 2, 64, 16, torch.bfloat16, [100, 333], trees, seed=9), torch.bfloat16)
    _attend_and_check(*_step(7, 1, 128, 16, torch.bfloat16, [9000, 20], [1, 1], seed=10), torch.bfloat16)


@pytest.mark.parametrize("seed", range(24))
def test_random_steps(seed) -> None:
    """Any mix of decode rows, runs, prompts and trees, over any head layout, block
    size and shared prefix; and the same bits when it runs again."""
    rng = np.random.default_rng(1000 + seed)
    hkv = int(rng.integers(1, 6))
    group = int(rng.choice([1, 2, 3, 4, 7, 8, 16, 17, 40]))
    d, bs = 16 * int(rng.integers(2, 17)), int(rng.choice([1, 3, 8, 16, 16, 32, 64, 100, 128]))
    dtype = (torch.bfloat16, torch.float16)[seed % 2]
    n = int(rng.integers(1, 9))
    prefix = int(rng.integers(0, 4)) if rng.random() < 0.3 else 0
    computed = [prefix * bs + int(np.exp2(rng.uniform(0, 10.5))) - 1 for _ in range(n)]
    layouts = []
    for _ in range(n):
        m = int(np.exp2(rng.uniform(0, 7.5)))
        kind = rng.random()
        layouts.append(1 if kind < 0.4 else m if kind < 0.7 else
                       tuple([-1] + [int(rng.integers(max(-1, i - 9), i)) for i in range(1, m)]))
    print(f"[gpu] q8 random step {seed}: {hkv * group}/{hkv}x{d} bs {bs} {dtype} prefix {prefix} {computed} "
          f"{[x if isinstance(x, int) else -len(x) for x in layouts]}", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(hkv * group, hkv, d, bs, dtype, computed, layouts, seed=seed, prefix=prefix)
    layer = cache.layer("layer0")
    parts = (layer.keys.view(torch.uint8), layer.key_scales, layer.values.view(torch.uint8), layer.value_scales)
    before = [p.clone() for p in parts]
    out = _attend_and_check(cache, md, q, k, v, dtype)
    after = [p.clone() for p in parts]
    for p, b in zip(parts, before):
        p.copy_(b)
    again = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, k, v, scale=1.0 / math.sqrt(d))
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))
    for p, b in zip(parts, after):
        assert torch.equal(p, b)


def test_shared_prefix_spans_and_options() -> None:
    print("[gpu] q8 attention shared prefix", file=sys.stderr, flush=True)
    args = _step(12, 2, 128, 16, torch.bfloat16, [256 + 5 * i for i in range(6)], [TREE] * 6, seed=11, prefix=16)
    out = _attend_and_check(*args, torch.bfloat16)
    for options in (dict(shared_prefix=False), dict(split_prefill=False), dict(use_prefill_kernel=False),
                    dict(decode_col_tiles=4, prefill_waves=8, decode_workgroups=False)):
        other = lv.HipPagedAttentionBackend(**options).create(args[0], args[1]).forward("layer0", *args[2:], scale=1 / math.sqrt(128))
        # Both within the bound of the exact result: 2^-8 per rounding.
        assert float((other.float() - out.float()).abs().max()) < 0.05


@pytest.mark.parametrize("layouts", ([1, 1], [(-1, 0, 0), 3], [40, 70], [TREE * 1, TREE]))
def test_nan_reaches_only_the_queries_that_see_it(layouts) -> None:
    # The last token of request 0 (a leaf: only its own query sees it) has NaN
    # in V and one in K of another token; request 1 is untouched.
    print(f"[gpu] q8 attention NaN in a masked row {layouts}", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(6, 2, 64, 16, torch.bfloat16, [100, 90], layouts, seed=12)
    n0 = len(md.query_layouts[0].parent_indices)
    v[n0 - 1, 0, 5] = math.nan
    v[n0 - 1, 1, 63] = math.inf
    if n0 > 1:
        k[n0 - 1, 1, 3] = math.nan
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, k, v, scale=0.125).isnan().cpu()
    want = torch.zeros_like(out)
    want[n0 - 1, 0:3, 5] = True   # kv head 0: one channel
    want[n0 - 1, 3:6, 63] = True
    if n0 > 1:
        want[n0 - 1, 3:6] = True  # a NaN score: all of kv head 1
    assert torch.equal(out, want)


def test_nan_in_the_history_reaches_every_query_of_its_request() -> None:
    print("[gpu] q8 attention NaN in the history", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(4, 2, 64, 16, torch.bfloat16, [3000, 90, 100], [1, 1, 30], seed=13)
    layer = cache.layer("layer0")
    block = md.block_tables[0][0]
    layer.keys.view(torch.uint8)[block, 2, 0, 0] = 0x7F     # request 0, kv head 0: NaN scores
    layer.values.view(torch.uint8)[md.block_tables[2][1], 3, 1, 9] = 0xFF
    out = lv.HipPagedAttentionBackend().create(cache, md).forward("layer0", q, k, v, scale=0.125).isnan().cpu()
    want = torch.zeros_like(out)
    want[0, 0:2] = True
    want[2:, 2:4, 9] = True
    assert torch.equal(out, want)


def test_stale_rows_behind_a_sequence_are_not_read() -> None:
    # NaN codes and huge scales wherever no sequence reaches.
    print("[gpu] q8 attention stale rows", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(6, 2, 64, 16, torch.bfloat16, [100, 90, 18], [1, 9, TREE], seed=14)
    used = torch.zeros(cache.config.num_blocks * 16, dtype=torch.bool)
    for table, c, layout in zip(md.block_tables, md.num_computed_tokens, md.query_layouts):
        for pos in range(c + len(layout.parent_indices)):
            used[table[pos // 16] * 16 + pos % 16] = True
    layer = cache.layer("layer0")
    for codes in (layer.keys, layer.values):
        codes.view(torch.uint8).view(-1, 2, 64)[(~used).to(DEV)] = 0x7F
    _attend_and_check(cache, md, q, k, v, torch.bfloat16)


def test_pool_past_32_bits_of_bytes() -> None:
    print("[gpu] q8 attention over a pool of 5 GiB", file=sys.stderr, flush=True)
    heads, d, bs = 8, 256, 16
    blocks = 5 * 2**30 // (heads * d * bs)
    spec = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("layer0", 16, heads, d),))
    cache = lv.QuantizedPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=blocks, block_size=bs, dtype=torch.bfloat16, device=DEV))
    small = _step(16, heads, d, bs, torch.bfloat16, [70, 40], [1, 20], seed=15)
    md = small[1]
    far = {b: blocks - 1 - 37 * i for i, b in enumerate(sorted({b for t in md.block_tables for b in t}))}
    src, dst = cache.layer("layer0"), small[0].layer("layer0")
    for big, little in ((src.keys, dst.keys), (src.values, dst.values), (src.key_scales, dst.key_scales),
                        (src.value_scales, dst.value_scales)):
        for b, to in far.items():
            big.view(torch.uint8)[to].copy_(little.view(torch.uint8)[b])
    moved = lv.PagedAttentionMetadata(block_tables=tuple(tuple(far[b] for b in t) for t in md.block_tables),
                                      num_computed_tokens=md.num_computed_tokens, query_layouts=md.query_layouts)
    scale = 1.0 / math.sqrt(d)
    a = lv.HipPagedAttentionBackend().create(small[0], md).forward("layer0", *small[2:], scale=scale)
    b = lv.HipPagedAttentionBackend().create(cache, moved).forward("layer0", *small[2:], scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    for i, (big, little) in enumerate(((src.keys, dst.keys), (src.values, dst.values))):
        for block, to in far.items():
            assert torch.equal(big.view(torch.uint8)[to], little.view(torch.uint8)[block]), i
    # Compact and copies across the far end.
    req = dict(block_ids=moved.block_tables[1], num_computed_tokens=40, num_query_tokens=20, num_reserved_query_tokens=20,
               retained_query_indices=(0, 5, 19))
    assert cache.compact(**req) == small[0].compact(**{**req, "block_ids": md.block_tables[1]}) == 2
    cache.copy_blocks((moved.block_tables[0][0],), (3,))
    torch.cuda.synchronize()
    for block, to in far.items():
        assert torch.equal(src.keys.view(torch.uint8)[to], dst.keys.view(torch.uint8)[block])
    assert torch.equal(src.values.view(torch.uint8)[3], dst.values.view(torch.uint8)[md.block_tables[0][0]])
    assert torch.equal(src.key_scales[3], dst.key_scales[md.block_tables[0][0]])


def test_strided_queries_and_the_general_path() -> None:
    print("[gpu] q8 attention strided inputs", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(6, 2, 64, 16, torch.bfloat16, [100, 90], [1, 20], seed=16)
    backend = lv.HipPagedAttentionBackend()
    out = backend.create(cache, md).forward("layer0", q, k, v, scale=0.125)
    packed = torch.cat((q, k, v), dim=1)
    views = packed[:, :6], packed[:, 6:8], packed[:, 8:]
    odd = torch.zeros((21, 10, 65), dtype=torch.bfloat16, device=DEV)
    odd[:, :, 1:] = packed
    for qkv in (views, (odd[:, :6, 1:], odd[:, 6:8, 1:], odd[:, 8:, 1:])):
        assert torch.equal(backend.create(cache, md).forward("layer0", *qkv, scale=0.125), out)


def test_refusals_of_the_context() -> None:
    cache, md, q, k, v = _step(6, 2, 64, 16, torch.bfloat16, [100], [1], seed=17)
    context = lv.HipPagedAttentionBackend().create(cache, md)
    with pytest.raises(lv.KVCacheError, match="rotated"):
        context.forward("layer0", q, k, v, scale=1.0, rotary=(q[:, 0], q[:, 0]))
    with pytest.raises(lv.KVCacheError, match="dtype and device"):
        context.forward("layer0", q.half(), k.half(), v.half(), scale=1.0)
    context = lv.HipPagedAttentionBackend().create(cache, md)
    context.forward("layer0", q, k, v, scale=1.0)
    with pytest.raises(lv.KVCacheError, match="more than once"):
        context.forward("layer0", q, k, v, scale=1.0)
    with pytest.raises(lv.ExecutionError, match="8-bit"):
        context.decode_launch("layer0", q, q, scale=1.0)
    with pytest.raises(lv.ExecutionError, match="8-bit"):
        context.prefill("layer0", q, q, scale=1.0)


def test_one_backend_serves_both_kinds_of_cache() -> None:
    # The same metadata object over a 16-bit and an 8-bit cache of one geometry.
    print("[gpu] q8 and 16-bit caches, one backend", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(6, 2, 64, 16, torch.bfloat16, [100, 300], [1, 20], seed=18)
    plain = lv.PagedKVCache(cache.model_spec, cache.config)
    layer, to = cache.layer("layer0"), plain.layer("layer0")
    backend = lv.HipPagedAttentionBackend()
    outs = []
    for _ in range(2):
        outs.append(backend.create(cache, md).forward("layer0", q, k, v, scale=0.125))
        for codes, scales, pool in ((layer.keys, layer.key_scales, to.keys), (layer.values, layer.value_scales, to.values)):
            pool.copy_((codes.float() * scales[:, None, :, None]).to(torch.bfloat16))
        slots = md.slot_mapping(block_size=16, device=DEV)
        stored = [t.view(-1, 2, 64)[slots] for t in (to.keys, to.values)]
        outs.append(backend.create(plain, md).forward("layer0", q, *stored, scale=0.125))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    assert float((outs[0].float() - outs[1].float()).abs().max()) < 0.05


def test_captured_step_replays() -> None:
    # Append, decode, merge and prefill in a graph: replays with new inputs in
    # place, eager work between them, against the eager result each time.
    print("[gpu] q8 attention in a graph", file=sys.stderr, flush=True)
    cache, md, q, k, v = _step(14, 2, 128, 16, torch.bfloat16, [900, 90, 700], [1, 30, TREE], seed=19)
    backend = lv.HipPagedAttentionBackend()
    start = [t.clone() for t in (cache.layer("layer0").keys.view(torch.uint8), cache.layer("layer0").values.view(torch.uint8),
                                 cache.layer("layer0").key_scales, cache.layer("layer0").value_scales)]

    def reset():
        layer = cache.layer("layer0")
        for t, s in zip((layer.keys.view(torch.uint8), layer.values.view(torch.uint8), layer.key_scales, layer.value_scales), start):
            t.copy_(s)

    backend.create(cache, md).forward("layer0", q, k, v, scale=0.1)  # plan, workspace
    context = backend.create(cache, md)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = context.forward("layer0", q, k, v, scale=0.1)
    gen = torch.Generator(device=DEV).manual_seed(20)
    for i in range(4):
        for t in (q, k, v):
            t.normal_(generator=gen)
        reset()
        eager = backend.create(cache, md).forward("layer0", q, k, v, scale=0.1).clone()
        state = _state(cache)
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager), i
        _same(cache, state)


def test_two_streams() -> None:
    print("[gpu] q8 attention on another stream", file=sys.stderr, flush=True)
    args = [_step(6, 2, 64, 16, torch.bfloat16, [400, 90], [1, 20], seed=s) for s in (21, 22)]
    want = [lv.HipPagedAttentionBackend().create(a[0], a[1]).forward("layer0", *a[2:], scale=0.125) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in args], []
    backends = [lv.HipPagedAttentionBackend() for _ in args]
    for _ in range(5):
        got = []
        for s, b, a in zip(streams, backends, args):
            with torch.cuda.stream(s):
                got.append(b.create(a[0], a[1]).forward("layer0", *a[2:], scale=0.125))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


# ---- compact, block copies, the whole step ---------------------------------------

@pytest.mark.parametrize("dtype,bs,shapes", [("bf16", 16, [(12, 2, 128)] * 2), ("fp16", 4, [(4, 2, 64), (4, 4, 32), (8, 1, 128)]),
                                             ("bf16", 12, [(4, 2, 80)]), ("bf16", 1, [(4, 1, 48)]), ("fp16", 64, [(4, 2, 256)])])
def test_compact_matches_the_oracle(dtype, bs, shapes) -> None:
    print(f"[gpu] q8 compact bs {bs} {shapes} {dtype}", file=sys.stderr, flush=True)
    rng = np.random.default_rng(bs)
    spec = lv.ModelKVCacheSpec(tuple(lv.AttentionLayerSpec(f"layer{i}", *s) for i, s in enumerate(shapes)))
    computed = [0, 5, 3 * bs - 1, 2 * bs, 17]
    retained = [(0, 2, 5), (1, 3, 4, 8), (8,), (7, 0, 3), tuple(range(9))]  # one out of order, one that moves nothing
    need = [-(-(c + 9) // bs) for c in computed]
    free = [int(b) for b in rng.permutation(sum(need) + 3)]
    tables = []
    for n in need:
        tables.append(tuple(free[:n]))
        free = free[n:]
    cache = lv.QuantizedPagedKVCache(spec, lv.PagedKVCacheConfig(num_blocks=sum(need) + 3, block_size=bs, dtype=DTYPES[dtype], device=DEV))
    _fill(cache, 23)
    src, dst = [], []
    for t, c, kept in zip(tables, computed, retained):
        for i, j in enumerate(kept):
            if i != j:
                src.append(t[(c + j) // bs] * bs + (c + j) % bs)
                dst.append(t[(c + i) // bs] * bs + (c + i) % bs)
    want = {}
    for s in spec.layers:
        want[s.layer_id] = _state(cache, s.layer_id)
        for codes, scales in want[s.layer_id]:
            Q.compact(codes, scales, src, dst)
    requests = [dict(block_ids=t, num_computed_tokens=c, num_query_tokens=9, num_reserved_query_tokens=9,
                     retained_query_indices=kept, num_readonly_prefix_blocks=0) for t, c, kept in zip(tables, computed, retained)]
    moved = lv.hip_compact(cache, **requests[0]) if len(shapes) == 1 else cache.compact(**requests[0])
    assert (moved, *cache.compact_many(iter(requests[1:]))) == tuple(sum(i != j for i, j in enumerate(kept)) for kept in retained)
    torch.cuda.synchronize()
    for layer_id, state in want.items():
        _same(cache, state, layer_id)


@pytest.mark.parametrize("requests,nodes", [(40, 5), (128, 5), (300, 5), (3, 45), (2, 20)])
def test_compact_of_many_requests(requests, nodes) -> None:
    """Chunks in one launch (33 to 384 pairs), the workspace's two launches (more,
    or a request of more than 32 moved rows)."""
    print(f"[gpu] q8 compact of {requests} requests, paths of {nodes}", file=sys.stderr, flush=True)
    rng = np.random.default_rng(requests)
    bs, n = 16, 2 * nodes
    computed = [int(c) for c in rng.integers(0, 40, requests)]
    need = [-(-(c + n) // bs) for c in computed]
    free = [int(b) for b in rng.permutation(sum(need) + 3)]
    tables = []
    for m in need:
        tables.append(tuple(free[:m]))
        free = free[m:]
    cache = _cache(4, 2, 64, bs, sum(need) + 3, torch.bfloat16, layers=2)
    _fill(cache, requests)
    src, dst, calls = [], [], []
    for t, c in zip(tables, computed):
        kept = (0, *sorted(rng.choice(np.arange(1, n), nodes - 1, replace=False).tolist()))
        for i, j in enumerate(kept):
            if i != j:
                src.append(t[(c + j) // bs] * bs + (c + j) % bs)
                dst.append(t[(c + i) // bs] * bs + (c + i) % bs)
        calls.append(dict(block_ids=t, num_computed_tokens=c, num_query_tokens=n, num_reserved_query_tokens=n,
                          retained_query_indices=kept, num_readonly_prefix_blocks=0))
    want = {f"layer{i}": _state(cache, f"layer{i}") for i in range(2)}
    for state in want.values():
        for codes, scales in state:
            Q.compact(codes, scales, src, dst)
    assert sum(cache.compact_many(calls)) == len(src)
    torch.cuda.synchronize()
    for layer_id, state in want.items():
        _same(cache, state, layer_id)


def test_compact_refuses_a_block_of_two_requests() -> None:
    cache = _cache(4, 2, 64, 16, 4, torch.bfloat16)
    one = dict(block_ids=(0,), num_computed_tokens=2, num_query_tokens=3, num_reserved_query_tokens=3, retained_query_indices=(2,))
    two = dict(block_ids=(0,), num_computed_tokens=8, num_query_tokens=3, num_reserved_query_tokens=3, retained_query_indices=(2,))
    with pytest.raises(lv.KVCacheError, match="same block of an 8-bit cache"):
        cache.compact_many((one, two))
    with pytest.raises(ValueError, match="unique"):
        cache.compact(**{**one, "retained_query_indices": (1, 1)})
    assert cache.compact_many(()) == ()


@pytest.mark.parametrize("n", (1, 5, 40))
def test_block_copies_take_codes_and_scales(n) -> None:
    print(f"[gpu] q8 block copy n={n}", file=sys.stderr, flush=True)
    cache = _cache(6, 3, 48, 12, 100, torch.float16, layers=2)
    _fill(cache, 24)
    order = [int(b) for b in np.random.default_rng(n).permutation(100)]
    src, dst = order[:n], order[n : 2 * n]
    want = {i: _state(cache, f"layer{i}") for i in range(2)}
    for state in want.values():
        for codes, scales in state:
            codes[dst], scales[dst] = codes[src], scales[src]
    (lv.hip_block_copy if n == 5 else type(cache).copy_blocks)(cache, src, dst)
    torch.cuda.synchronize()
    for i, state in want.items():
        _same(cache, state, f"layer{i}")
    with pytest.raises(lv.KVCacheError, match="invalid physical block"):
        cache.copy_blocks((0,), (100,))


def test_speculative_steps_end_to_end() -> None:
    # Prompt, then rounds of: tree step over the cache, verification, compact,
    # next token; every forward against the oracle over the oracle's cache.
    print("[gpu] q8 speculative steps", file=sys.stderr, flush=True)
    hq, hkv, d, bs, vocab, layers = 6, 2, 64, 16, 211, ("layer0",)
    rng = np.random.default_rng(25)
    gen = torch.Generator(device=DEV).manual_seed(25)
    cache = _cache(hq, hkv, d, bs, 40, torch.bfloat16)
    backend = lv.HipPagedAttentionBackend()
    want = _state(cache)
    perm = [int(b) for b in rng.permutation(40)]
    tables, computed, scale = (tuple(perm[:14]), tuple(perm[14:28]), tuple(perm[28:])), [0, 0, 0], 0.125

    def step(layouts):
        need = [-(-(c + len(p)) // bs) for c, p in zip(computed, layouts)]
        md = lv.PagedAttentionMetadata(block_tables=tuple(t[:n] for t, n in zip(tables, need)),
                                       num_computed_tokens=tuple(computed), query_layouts=tuple(map(lv.QueryLayout, layouts)))
        t = sum(map(len, layouts))
        q, k, v = (torch.randn((t, h, d), generator=gen, device=DEV).to(torch.bfloat16) for h in (hq, hkv, hkv))
        for (codes, scales), rows in zip(want, (k, v)):
            Q.append(codes, scales, rows.double().cpu().numpy(), _slots(md, bs).tolist(), LARGEST[torch.bfloat16])
        out = backend.create(cache, md).forward(layers[0], q, k, v, scale=scale)
        torch.cuda.synchronize()
        _same(cache, want)
        _check(out, *_expected(cache, md, q, want), torch.bfloat16)

    step([tuple(range(-1, n - 1)) for n in (50, 33, 4)])
    computed = [50, 33, 4]
    for turn in range(4):
        trees = [lv.DraftTree(tuple(int(x) for x in rng.permutation(vocab)[:n]),
                              tuple(int(rng.integers(-1, i)) if i else -1 for i in range(n))) for n in (8, 0, 5)]
        batch = lv.DraftBatch(trees, device=DEV)
        layouts = [lv.append_draft_layout(1, t).parent_indices for t in trees]
        step(layouts)
        target = torch.rand((batch.num_rows, vocab), generator=gen, device=DEV)
        row = 0
        for t in trees:  # drafts that are often right
            for i, (token, parent) in enumerate(zip(t.token_ids, t.parent_indices)):
                target[row + parent + 1, token] += 40
            row += len(t) + 1
        target /= target.sum(dim=1, keepdim=True)
        node, sample = torch.rand(batch.num_rows, generator=gen, device=DEV), torch.rand(3, generator=gen, device=DEV)
        verdict = lv.verify_drafts(batch, target, node, sample)
        kept = verdict.retained_query_indices([1] * 3)
        row = 0
        for r, t in enumerate(trees):
            path, token = Q.verify(t.parent_indices, t.token_ids, target[row : row + len(t) + 1].double().cpu().numpy(),
                                   node[row : row + len(t) + 1].tolist(), float(sample[r]))
            assert kept[r] == (0, *(1 + i for i in path)) and int(verdict.tokens[r]) == token
            row += len(t) + 1
        src, dst = [], []
        for t, c, indices in zip(tables, computed, kept):
            for i, j in enumerate(indices):
                if i != j:
                    src.append(t[(c + j) // bs] * bs + (c + j) % bs)
                    dst.append(t[(c + i) // bs] * bs + (c + i) % bs)
        for codes, scales in want:
            Q.compact(codes, scales, src, dst)
        requests = [dict(block_ids=t[: -(-(c + len(p)) // bs)], num_computed_tokens=c, num_query_tokens=len(p),
                         num_reserved_query_tokens=len(p), retained_query_indices=indices)
                    for t, c, p, indices in zip(tables, computed, layouts, kept)]
        assert sum(cache.compact_many(requests)) == len(src)
        torch.cuda.synchronize()
        _same(cache, want)
        computed = [c + len(indices) for c, indices in zip(computed, kept)]
    step([(-1,)] * 3)
