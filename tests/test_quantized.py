"""CPU tests of the 8-bit cache and draft verification: the oracle against
torch's e4m3 and against the distribution it must keep, the drafts' packing,
refusals, and the C entry points' argument checks (before any HIP call)."""

from __future__ import annotations

import ctypes
import dataclasses

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
from light_vllm_amd import native
from light_vllm_amd.verify import pack_drafts
from oracle import quantized_oracle as Q

X = ctypes.c_void_p(16)  # an address that no check dereferences


def test_oracle_rounding_is_torchs_e4m3() -> None:
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[every.isfinite()].unique()
    middle = (every[1:] + every[:-1]) / 2  # ties
    rng = np.random.default_rng(0)
    x = torch.cat([every, middle, torch.from_numpy(rng.uniform(-448, 448, 4000).astype(np.float32)),
                   torch.from_numpy((rng.standard_normal(4000) * 0.01).astype(np.float32))])
    np.testing.assert_array_equal(Q.round_e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("amax,e", [(0.0, -100), (448.0, 0), (448.1, 1), (449.0, 1), (224.0, -1), (1.0, -8), (1e-38, -100), (3.3e38, 120)])
def test_scale_of_a_largest_magnitude(amax, e) -> None:
    assert Q.scale_of(np.float32(amax)) == 2.0**e


def test_token_at_a_time_gives_what_a_whole_prompt_gives() -> None:
    # Exponent-only re-scaling: the same codes unless one became subnormal
    # (magnitudes below 2^-6 of the block's final scale).
    rng = np.random.default_rng(1)
    rows = np.exp2(rng.integers(-3, 4, (16, 1, 1))) * rng.choice([-1, 1], (16, 2, 32)) * rng.uniform(1, 2, (16, 2, 32))
    whole, ws = np.zeros((1, 16, 2, 32)), np.full((1, 2), 2.0**-100)
    one, os_ = whole.copy(), ws.copy()
    Q.append(whole, ws, rows, range(16), 61440.0)
    for i in range(16):
        Q.append(one, os_, rows[i : i + 1], [i], 61440.0)
    np.testing.assert_array_equal(one, whole)
    np.testing.assert_array_equal(os_, ws)


def test_growing_scales_stay_within_the_stated_bound() -> None:
    """A row is rounded when it is written (half a step of its value, 2^-4 of it, or
    half the smallest subnormal code, 2^-10 of the scale then) and again at each
    growth that makes its code subnormal: 2^-10 of scales that at least double, in
    all less than 2^-9 of the last one.  One rounding's bound does not hold."""
    rng = np.random.default_rng(3)
    worst = one_rounding = 0.0
    for _ in range(100):
        sizes = np.exp2(np.sort(rng.uniform(0, 14, 12)))
        rows = rng.uniform(-1, 1, (12, 1, 64)) * sizes[:, None, None]
        rows[:, 0, 0] = sizes
        codes, scales = np.zeros((1, 16, 1, 64)), np.full((1, 1), 2.0**-100)
        for i in range(12):
            Q.append(codes, scales, rows[i : i + 1], [i], 1.875 * 2.0**127)
        err = np.abs(codes[0, :12] * scales[0, 0] - rows)
        worst = max(worst, float((err / (2.0**-4 * np.abs(rows) + 2.0**-9 * scales[0, 0])).max()))
        one_rounding = max(one_rounding, float((err / np.maximum(2.0**-4 * np.abs(rows), 2.0**-10 * scales[0, 0])).max()))
    assert worst < 1.0 < one_rounding


@pytest.mark.parametrize("mode", ("chain", "tree"))
def test_verified_tokens_follow_the_target(mode) -> None:
    # The first emitted token over a grid of uniforms (and, for the chain, every
    # drafted token with its draft probability) against p: each cell's share is
    # exact to the grid's step per interval border.
    rng = np.random.default_rng(2)
    p, q = rng.dirichlet(np.ones(6)), rng.dirichlet(np.ones(6))
    grid = (np.arange(200) + 0.5) / 200
    found = np.zeros(6)
    drafts = [((-1,), (t,), q[t]) for t in range(6)] if mode == "chain" else [((-1, -1, 0), (4, 1, 2), 1.0)]
    target = np.stack([p] * 4)
    for parents, tokens, weight in drafts:
        probs = np.stack([q]) if mode == "chain" else None
        for u in grid:
            for s in grid:
                path, token = Q.verify(parents, tokens, target, [u] * 4, s, probs)
                found[tokens[path[0]] if path else token] += weight / grid.size**2
    # Borders: one of u per drafted token, up to six of u'.
    np.testing.assert_allclose(found, p, atol=7 / 200)


def test_drafts_are_packed_with_their_earlier_siblings() -> None:
    trees = [lv.DraftTree((7, 9, 8, 5), (-1, -1, 0, -1)), lv.DraftTree((), ()), lv.DraftTree((3, 4), (-1, 0))]
    (tokens, starts, parents, siblings), chains, top = pack_drafts(trees)
    assert tokens.view(np.int64).tolist() == [7, 9, 8, 5, 3, 4]
    assert starts.tolist() == [0, 4, 4, 6]
    assert parents.tolist() == [-1, -1, 0, -1, -1, 0]
    assert siblings.tolist() == [-1, 0, -1, 1, -1, -1]
    assert not chains and top == 9
    assert pack_drafts(trees[1:])[1]
    with pytest.raises(ValueError, match="at least one request"):
        pack_drafts([])
    n = native.VERIFY_MAX_DRAFTS
    pack_drafts([lv.DraftTree(tuple(range(n)), tuple(range(-1, n - 1)))])
    with pytest.raises(ValueError, match="at most 1024 drafts"):
        pack_drafts([lv.DraftTree(tuple(range(n + 1)), tuple(range(-1, n)))])
    with pytest.raises(ValueError, match="below 2"):
        pack_drafts([lv.DraftTree((2**31,), (-1,))])


def test_refusals_without_a_gpu() -> None:
    spec = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("a", 4, 2, 64),))
    config = lambda **kw: lv.PagedKVCacheConfig(**{**dict(num_blocks=4, block_size=16, dtype=torch.bfloat16, device="cuda:0"), **kw})  # noqa: E731
    with pytest.raises(lv.KVCacheError, match="requires a GPU"):
        lv.QuantizedPagedKVCache(spec, config(device="cpu"))
    with pytest.raises(lv.KVCacheError, match="bfloat16 or float16"):
        lv.QuantizedPagedKVCache(spec, config(dtype=torch.float32))
    with pytest.raises(lv.KVCacheError, match="at most 2"):
        lv.QuantizedPagedKVCache(spec, config(num_blocks=2**27))
    odd = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("a", 4, 2, 40),))
    with pytest.raises(lv.KVCacheError, match="head sizes"):
        lv.QuantizedPagedKVCache(odd, config())
    with pytest.raises(lv.ExecutionError, match="requires a GPU"):
        lv.DraftBatch([lv.DraftTree((), ())], device="cpu")
    mixed = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("a", 4, 2, 64), lv.AttentionLayerSpec("b", 4, 1, 128)))
    assert lv.quantized_kv_cache_bytes_per_block(mixed, block_size=16) == 2 * (2 * (16 * 64 + 4) + 16 * 128 + 4)


def test_16_bit_appends_refuse_an_8_bit_cache() -> None:
    # Their rows are twice as long as the pool's.  (Nothing to append: the calls
    # reach no kernel either way.)
    from light_vllm_amd import paged_cache

    spec = lv.AttentionLayerSpec("a", 4, 2, 64)
    rows = torch.zeros((0, 1, 2, 64), dtype=torch.bfloat16)

    class Cache:
        quantized = True

        def layer(self, layer_id):
            return lv.QuantizedPagedLayerCache(rows, rows, rows, rows)

        def layer_spec(self, layer_id):
            return spec

    q, k = torch.zeros((0, 4, 64), dtype=torch.bfloat16), rows[:, 0]
    angles = torch.zeros((0, 64), dtype=torch.bfloat16)
    with pytest.raises(lv.KVCacheError, match="8-bit KV cache"):
        paged_cache.hip_append(Cache(), "a", k, k, 0, 0)
    with pytest.raises(lv.KVCacheError, match="8-bit KV cache"):
        paged_cache.hip_append_rotary(Cache(), "a", q, k, k, (angles, angles), 0, 0)


def test_a_mappings_tensors_are_checked_where_it_is_made() -> None:
    # The launch reads int64 slots, and as many sources, on the cache's device.
    slots = torch.tensor([3, 4], dtype=torch.long)
    good = lv.QuantizedKVWriteMapping(slots, 4, slots, (4, 16))
    assert good.geometry == (4, 16)
    lv.QuantizedKVWriteMapping(slots, 2, None, (4, 16))
    for bad in ((slots.int(), 2, None), (slots.view(1, 2), 2, None), (slots, 3, None), (slots.repeat(2)[::2], 2, None),
                (slots, 4, slots[:1]), (slots, 4, slots.int()), (slots, 4, slots.repeat(2)[::2]), (slots, 1, slots),
                (slots, 4, slots.to("meta"))):
        with pytest.raises(lv.KVCacheError, match="slots and source indices"):
            lv.QuantizedKVWriteMapping(*bad, (4, 16))
    with pytest.raises(lv.KVCacheError, match="slots and source indices"):
        dataclasses.replace(good, source_indices=slots.to("meta"))


def test_append_entry_point_checks() -> None:
    lib = native.load()

    def call(key=X, strides=(256, 128), pool=X, n=4, heads=2, d=128, bs=16, dtype=2):
        return lib.lvamd_kv_append_q8(key, *strides, X, 256, 128, pool, X, X, X, X, None, n, heads, d, bs, dtype, None)

    assert call(n=0) == 0
    assert call(dtype=0) == -2 and call(dtype=7) == -2 and call(d=40) == -2 and call(d=272) == -2
    for bad in (dict(key=None), dict(pool=None), dict(n=-1), dict(heads=0), dict(bs=0), dict(strides=(4, 128)),
                dict(strides=(256, 12)), dict(key=ctypes.c_void_p(8)), dict(pool=ctypes.c_void_p(24))):
        assert call(**bad) == -1, bad


def test_attention_entry_point_checks() -> None:
    lib = native.load()
    f = ctypes.c_float(0.1)

    none = (None, 0, 0, None, 0, 0)
    new = (X, 512, 128, X, 512, 128)

    def decode(q=X, waves=1, slots=0, heads=4, group=7, d=128, bs=16, dtype=2, qs=(3584, 128), part=None, kv=none):
        return lib.lvamd_paged_decode_q8(q, *qs, *kv, X, X, X, X, X, 3584, 128, X, X, waves, X, X, part, part, slots, heads,
                                         group, d, bs, f, dtype, None)

    def prefill(q=X, units=1, slots=0, heads=4, group=7, d=128, bs=16, dtype=2, qs=(3584, 128), part=None, columns=128):
        return lib.lvamd_paged_prefill_q8(q, *qs, X, X, X, X, X, 3584, 128, X, X, X, units, part, part, slots, heads, group, d,
                                          columns, bs, f, dtype, None)

    for call, count in ((decode, "waves"), (prefill, "units")):
        assert call(**{count: 0}) == 0
        assert call(dtype=0) == -2 and call(d=24) == -2 and call(d=264) == -2
        for bad in (dict(q=None), dict(heads=0), dict(group=0), dict(bs=0), dict(qs=(3580, 128)), {count: -1}):
            assert call(**bad) == -1, bad
        assert call(slots=3) == -3
    assert decode(group=17) == -1
    # The decode launch's append: both tensors, aligned rows, whole blocks per tile.
    for kv in ((X, 512, 128, None, 512, 128), (X, 508, 128, X, 512, 128), (ctypes.c_void_p(8), 512, 128, X, 512, 128)):
        assert decode(kv=kv) == -1, kv
    assert decode(kv=new, bs=12) == -1 and decode(kv=new, bs=128) == -1
    assert prefill(columns=32) == -2 and prefill(columns=512) == -2 and prefill(columns=256, d=64) == -2 and prefill(columns=64, q=None) == -1
    merge = lambda dtype, jobs, cols=1: lib.lvamd_paged_attention_merge_q8(X, X, X, 0, 0, X, jobs, 4, 7, 128, cols, 16, dtype, None)  # noqa: E731
    assert merge(2, 0) == 0 and merge(0, 1) == -2 and merge(2, -1) == -1 and merge(1, 1, 17) == -2
    for d in (32, 64, 80, 128, 256):
        assert lib.lvamd_paged_decode_q8_tile_tokens(2, d) * d <= 8192
        assert lib.lvamd_paged_prefill_q8_key_tokens(1, d) == (64 if d <= 128 else 32)
    assert lib.lvamd_paged_decode_q8_tile_tokens(0, 128) == -2 and lib.lvamd_paged_prefill_q8_key_tokens(2, 40) == -2
    plan = native.AttentionPlanQ8(base=native.AttentionPlan(num_kv_heads=4, group=7, head_size=128, block_size=16, dtype=2))
    empty = (None, 0, 0, None, 0, 0)
    call = lambda p, kv=empty, pool=X: lib.lvamd_paged_attention_q8(p, X, 0, 0, *kv, pool, X, X, 0, 0, f, None)  # noqa: E731
    assert call(None) == -1
    assert call(ctypes.addressof(plan)) == 0  # nothing to append, no rows
    assert call(ctypes.addressof(plan), pool=None) == -1
    assert call(ctypes.addressof(plan), kv=(X, 0, 0, None, 0, 0)) == -1
    plan.scale_offset = 24
    assert call(ctypes.addressof(plan)) == -1


def test_prefill_takes_a_positive_scale_only() -> None:
    # Its running maximum is that of the unscaled scores, its masked ones -inf.
    lib = native.load()
    units = native.AttentionPlanQ8(base=native.AttentionPlan(num_units=1, num_kv_heads=4, group=7, head_size=128, block_size=16,
                                                             dtype=2, prefill_col_tiles=8))
    empty = (None, 0, 0, None, 0, 0)
    for scale in (0.0, -0.125, float("nan")):
        f = ctypes.c_float(scale)
        assert lib.lvamd_paged_prefill_q8(X, 3584, 128, X, X, X, X, X, 3584, 128, X, X, X, 1, None, None, 0, 4, 7, 128, 128, 16, f,
                                          2, None) == -1
        assert lib.lvamd_paged_attention_q8(ctypes.addressof(units), X, 3584, 128, *empty, X, X, X, 3584, 128, f, None) == -1


def test_compact_entry_point_checks() -> None:
    lib = native.load()

    def call(keys=X, layers=2, heads=2, d=128, bs=16, offset=1024, n=3, groups=1, ws=X, nbytes=1 << 20):
        return lib.lvamd_kv_compact_q8(keys, X, layers, heads, d, bs, offset, X, X, n, X, groups, ws, nbytes, None)

    assert call(n=0, groups=0) == 0
    assert call(d=40) == -2
    for bad in (dict(keys=None), dict(layers=0), dict(heads=0), dict(bs=0), dict(offset=-4), dict(offset=2), dict(n=-1),
                dict(groups=0), dict(groups=4), dict(n=0, groups=1)):
        assert call(**bad) == -1, bad
    need = lib.lvamd_kv_compact_q8_workspace_size(3, 2, 2, 128)
    assert need == 3 * 2 * 2 * 2 * (128 + 4) and lib.lvamd_kv_compact_q8_workspace_size(0, 2, 2, 128) == 0
    assert call(ws=None) == -3 and call(nbytes=need - 1) == -3 and call(ws=ctypes.c_void_p(8)) == -3


def test_compact_few_entry_point_checks() -> None:
    lib = native.load()
    assert int(lib.lvamd_kv_compact_q8_few_pairs()) == 32
    most = int(lib.lvamd_kv_compact_q8_few_call_pairs())
    assert most == 384
    pairs = np.arange(most + 1, dtype=np.int64)

    def call(keys=X, layers=2, heads=2, d=128, bs=16, offset=1024, src=pairs, dst=pairs, n=32, chunks=(0, 32), count=None):
        starts = np.asarray(chunks, dtype=np.int32)
        return lib.lvamd_kv_compact_q8_few(keys, X, layers, heads, d, bs, offset, src.ctypes.data, dst.ctypes.data, n,
                                           starts.ctypes.data, len(starts) - 1 if count is None else count, None)

    assert call(n=0) == 0
    assert call(d=40) == -2
    for bad in (dict(keys=None), dict(layers=0), dict(heads=0), dict(bs=0), dict(offset=-4), dict(offset=2), dict(n=-1),
                dict(n=33), dict(n=33, chunks=(0, 33)), dict(n=33, chunks=(0, 32, 32, 33)), dict(n=33, chunks=(1, 33)),
                dict(n=34, chunks=(0, 32, 33)), dict(n=32, count=0), dict(n=32, chunks=range(34), count=33),
                dict(n=most + 1, chunks=(*range(0, most, 32), most, most + 1)), dict(src=pairs - 1), dict(dst=pairs + 2**31)):
        assert call(**bad) == -1, bad


def test_compact_chunks() -> None:
    chunks = native.host().compact_chunks
    packed = lambda *slots: np.asarray(slots, dtype=np.int64).tobytes()  # noqa: E731

    def cut(moved, src, dst, most=4, bs=16):
        found = chunks(packed(*moved), packed(*src), packed(*dst), bs, most)
        return None if found is None else np.frombuffer(found, dtype=np.int32).tolist()

    assert cut((3, 0, 1), (5, 6, 7, 40), (2, 3, 4, 33)) == [0, 4]
    assert cut((3, 2), (5, 6, 7, 40, 41), (2, 3, 4, 33, 34)) == [0, 3, 5]
    assert cut((4, 4, 1), (5, 6, 7, 8, 37, 38, 39, 40, 70), (1, 2, 3, 4, 33, 34, 35, 36, 66)) == [0, 4, 8, 9]
    assert cut((5,), (5, 6, 7, 8, 9), (1, 2, 3, 4, 5)) is None                                   # a longer request
    assert cut((3, 2), (5, 6, 7, 40, 9), (2, 3, 4, 33, 34)) is None                              # reads a block the first writes
    assert cut((3, 2), (5, 40, 7, 41, 42), (2, 3, 4, 33, 34)) is None                            # and the other way round
    assert cut((3, 2), (5, 6, 7, 8, 9), (2, 3, 4, 0, 1)) is None                                 # both write one block
    assert cut((2, 2), (5, 6, 8, 9), (2, 3, 0, 1)) == [0, 4]                                     # in one chunk that is no matter
    assert cut((), (), ()) == [0, 0]
    for bad in (((3,), (1, 2), (3, 4)), ((-1,), (1,), (2,))):
        with pytest.raises(ValueError):
            cut(*bad)
    with pytest.raises(ValueError):
        chunks(packed(1), packed(1, 2), packed(1), 16, 4)


def test_block_runs() -> None:
    runs = native.host().block_runs
    packed = lambda *slots: np.asarray(slots, dtype=np.int64).tobytes()  # noqa: E731
    twice, starts = runs(packed(3, 0, 4), packed(33, 34, 48, 5, 6, 15, 16), 16)
    assert not twice and np.frombuffer(starts, dtype=np.int64).tolist() == [0, 2, 3, 6, 7]
    assert runs(packed(1, 1), packed(33, 34), 16)[0] == 1
    assert runs(packed(3), packed(33, 48, 34), 16)[0] == 1
    assert np.frombuffer(runs(b"", b"", 16)[1], dtype=np.int64).tolist() == [0]
    for bad in ((packed(1), packed(1), 0), (packed(1), packed(1, 2), 4), (packed(2), packed(1), 4), (packed(-1, 2), packed(1), 4)):
        with pytest.raises(ValueError):
            runs(*bad)


def test_verify_entry_point_checks() -> None:
    lib = native.load()

    def call(target=X, stride=100, vocab=100, dtype=0, starts=X, n=2, drafts=3, width=1, ws=X, nbytes=1 << 20):
        return lib.lvamd_verify_drafts(target, stride, None, 0, vocab, dtype, starts, X, X, X, n, drafts, X, X, 0, X, X, width, X,
                                       ws, nbytes, None)

    assert call(n=0) == 0
    assert call(dtype=3) == -2
    for bad in (dict(target=None), dict(starts=None), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(n=-1), dict(n=65536),
                dict(width=0), dict(stride=-1), dict(drafts=-1)):
        assert call(**bad) == -1, bad
    need = lib.lvamd_verify_drafts_workspace_size(2, 3, 100, 0)
    assert need > 0 and call(nbytes=need - 1) == -3 and call(ws=None) == -3 and call(ws=ctypes.c_void_p(4)) == -3


@pytest.mark.parametrize("kernel,count", [("q8_append_kernel", 2), ("q8_compact_few_kernel", 2), ("q8_gather_kernel", 1),
                                          ("q8_scatter_kernel", 1), ("q8_decode_kernel", 60), ("q8_prefill_kernel", 68),
                                          ("verify_sums_kernel", 6), ("verify_draw_kernel", 6)])
def test_kernels_hold_their_registers(kernel, count) -> None:
    pytest.importorskip("msgpack")
    from test_kernel_resources import _kernels

    found = {n: k for n, k in _kernels().items() if kernel in n}
    assert len(found) == count
    assert not {n for n, k in found.items() if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
