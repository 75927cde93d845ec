"""Host tests of the latent cache, its planner and the rotary frequencies (CPU)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
from light_vllm_amd import native
from light_vllm_amd.plan import StepPlan
from oracle import latent_oracle as Z

CPU = torch.device("cpu")


def test_layer_spec_rules() -> None:
    spec = lv.LatentLayerSpec("a", 16, 512, 64)
    assert spec.row_size == 576 and spec.rotary_layout == "interleaved"
    for kw, message in (
        (dict(layer_id=""), "layer_id"), (dict(num_query_heads=0), "num_query_heads"),
        (dict(num_query_heads=True), "num_query_heads"), (dict(latent_size=500), "latent_size"),
        (dict(latent_size=640), "latent_size"), (dict(rope_size=48), "rope_size"), (dict(rotary_layout="x"), "rotary_layout"),
    ):
        with pytest.raises(ValueError, match=message):
            lv.LatentLayerSpec(**{**dict(layer_id="a", num_query_heads=16, latent_size=512, rope_size=64), **kw})
    with pytest.raises(ValueError, match="at least one layer"):
        lv.LatentKVCacheSpec(())
    with pytest.raises(ValueError, match="unique"):
        lv.LatentKVCacheSpec((spec, spec))
    two = lv.LatentKVCacheSpec([spec, lv.LatentLayerSpec("b", 8, 256, 32)])
    assert lv.latent_kv_cache_bytes_per_block(two, block_size=16, dtype=torch.bfloat16) == (576 + 288) * 16 * 2


def test_cache_refuses_what_it_cannot_hold() -> None:
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec("a", 16, 512, 64),))
    for config, message in (
        (lv.PagedKVCacheConfig(num_blocks=4, block_size=16, dtype=torch.bfloat16), "requires a GPU"),
        (lv.PagedKVCacheConfig(num_blocks=4, block_size=16, dtype=torch.float32, device="cuda"), "bfloat16 or float16"),
        (lv.PagedKVCacheConfig(num_blocks=2**27, block_size=16, dtype=torch.float16, device="cuda"), "at most"),
    ):
        with pytest.raises(lv.KVCacheError, match=message):
            lv.LatentPagedKVCache(spec, config)
    heads = lv.ModelKVCacheSpec((lv.AttentionLayerSpec("a", 16, 1, 128),))
    with pytest.raises(lv.KVCacheError, match="LatentKVCacheSpec"):
        lv.LatentPagedKVCache(heads, lv.PagedKVCacheConfig(num_blocks=4, block_size=16, dtype=torch.float16, device="cuda"))


def test_the_library_refuses_bad_arguments() -> None:
    """Checked before any HIP call."""
    lib = native.load()
    one = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(one) + 15) // 16 * 16
    append = lambda **k: lib.lvamd_latent_append(*{**dict(  # noqa: E731
        latent=p, ls=8, rope=p, rs=8, pool=p, slots_n=16, slots=p, sources=None, n=1, cos=None, sin=None, angle=4, il=1,
        q=None, qt=8, qh=8, rot=None, tokens=1, heads=1, size=512, rsize=64, dtype=native.DTYPE_BF16, stream=None), **k}.values())
    for bad, status in ((dict(size=500), -2), (dict(rsize=16), -2), (dict(dtype=native.DTYPE_F32), -2), (dict(n=-1), -1),
                        (dict(latent=None), -1), (dict(latent=p + 2), -1), (dict(ls=9), -1), (dict(rope=p + 8), -1),
                        (dict(slots=None), -1), (dict(pool=None), -1), (dict(cos=p), -1), (dict(q=p, rot=p), -1),
                        (dict(cos=p, sin=p, q=p, rot=None), -1), (dict(cos=p + 4, sin=p), -1),
                        (dict(cos=p, sin=p, angle=6), -1), (dict(cos=p, sin=p, q=p, rot=p, qh=4), -1),
                        (dict(slots_n=2**31), -1), (dict(n=2**31), -1)):
        assert append(**bad) == status, bad
    assert append(n=0) == 0
    assert lib.lvamd_rotary_angles(p, 3, 1, p, 32, 1.0, p, p, 1, 0, None) == -1
    assert lib.lvamd_rotary_angles(p, 8, 1, p, 32, 1.0, p, p, 3, 0, None) == -1
    assert lib.lvamd_rotary_angles(p, 8, 1, p, 32, 1.0, p, p, 1, 9, None) == -1
    assert lib.lvamd_rotary_angles(p, 8, 2**31, p, 32, 1.0, p, p, 1, 0, None) == -1
    assert lib.lvamd_rotary_angles(None, 8, 0, None, 32, 1.0, None, None, 1, 0, None) == 0
    few = lib.lvamd_latent_move_few_pairs()
    assert few == 32 and lib.lvamd_latent_move_few(p, 1, 1152, p, p, few + 1, None) == -1
    assert lib.lvamd_latent_move_few(p, 1, 1150, p, p, 1, None) == -1
    assert lib.lvamd_latent_move_few(None, 1, 1152, None, None, 0, None) == 0
    assert lib.lvamd_latent_move_workspace_size(3, 2, 1152) == 3 * 2 * 1152
    assert lib.lvamd_latent_move(p, 2, 1152, p, p, 3, p, 3 * 2 * 1152 - 1, None) == -3
    assert lib.lvamd_latent_move(p, 2, 1152, p, None, 3, None, 0, None) == -1
    decode = lambda **k: lib.lvamd_latent_decode(*{**dict(  # noqa: E731
        q=p, qt=8, qh=8, qr=p, rt=8, rh=8, lat=None, ls=0, rk=None, rs=0, cos=None, sin=None, angle=0, il=1, pool=p, out=p, ot=8, oh=8, pieces=p, groups=1, jobs=None, njobs=0,
        cols=1, tables=p, vis=p, acc=None, ml=None, slots=0, heads=1, size=512, rope=64, tiles=1, block=16, scale=1.0,
        dtype=native.DTYPE_F16, stream=None), **k}.values())
    for bad, status in ((dict(size=576), -2), (dict(dtype=native.DTYPE_F32), -2), (dict(tiles=3), -2), (dict(groups=-1), -1),
                        (dict(heads=0), -1), (dict(block=0), -1), (dict(q=None), -1), (dict(q=p + 8), -1), (dict(rt=4), -1),
                        (dict(out=p + 4), -1), (dict(ot=2), -1), (dict(pool=None), -1), (dict(pieces=None), -1),
                        (dict(njobs=1), -1), (dict(slots=1), -3), (dict(vis=None), -1), (dict(lat=p), -1),
                        (dict(lat=p, ls=4, rk=p), -1), (dict(cos=p), -1), (dict(cos=p, sin=p + 8), -1),
                        (dict(cos=p, sin=p, angle=2), -1),
                        (dict(lat=p, ls=8, rk=p, rs=8, tiles=8), -2)):
        assert decode(**bad) == status, bad
    assert decode(groups=0) == 0


# ---- frequencies -----------------------------------------------------------------

def test_frequencies_follow_their_definitions() -> None:
    freq, magnitude = lv.rotary_frequencies(64, 10000.0)
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert magnitude == 1.0 and np.allclose(freq, want, rtol=1e-14, atol=0)
    freq, _ = lv.rotary_frequencies(64, 10000.0, lv.RotaryScaling("linear", 4.0))
    assert np.allclose(freq, np.array(want) / 4, rtol=1e-14, atol=0)
    freq, _ = lv.rotary_frequencies(64, 10000.0, lv.RotaryScaling("base", 8.0))
    assert freq[0] == 1.0 and math.isclose(freq[-1], want[-1] / 8, rel_tol=1e-13)
    scaling = lv.RotaryScaling("ramp", 32.0, 4096)
    freq, magnitude = lv.rotary_frequencies(64, 10000.0, scaling)
    turns = 4096 * np.array(want) / (2 * math.pi)
    ratio = freq.numpy() / want
    assert math.isclose(magnitude, 0.1 * math.log(32) + 1)
    assert np.all(ratio[turns > 40] == 1.0) and np.allclose(ratio[turns < 0.7], 1 / 32)
    assert np.all(np.diff(ratio) <= 0)
    freq, magnitude = lv.rotary_frequencies(64, 500000.0, lv.RotaryScaling("smooth", 8.0, 8192))
    want = 500000.0 ** (-np.arange(0, 64, 2) / 64)
    turns = 8192 * want / (2 * math.pi)
    ratio = freq.numpy() / want
    assert magnitude == 1.0 and np.all(ratio[turns > 4] == 1) and np.allclose(ratio[turns < 1], 1 / 8)
    mid = (turns > 1) & (turns < 4)
    share = (turns[mid] - 1) / 3
    assert mid.any() and np.allclose(ratio[mid], share + (1 - share) / 8)
    assert lv.rotary_frequencies(64, 1e4, lv.RotaryScaling("ramp", 32.0, magnitude=1.0))[1] == 1.0


@pytest.mark.parametrize("make, message", [
    (lambda: lv.RotaryScaling("other", 2.0), "must be one of"),
    (lambda: lv.RotaryScaling("linear", 0.0), "positive number"),
    (lambda: lv.RotaryScaling("linear", math.nan), "positive number"),
    (lambda: lv.RotaryScaling("ramp", 2.0, 0), "positive integer"),
    (lambda: lv.RotaryScaling("smooth", 2.0, 4096, slow=4.0, fast=4.0), "slow < fast"),
    (lambda: lv.RotaryScaling("ramp", 2.0, magnitude=math.inf), "must be a number"),
    (lambda: lv.rotary_frequencies(63, 1e4), "even integer"),
    (lambda: lv.rotary_frequencies(64, 1.0), "above 1"),
    (lambda: lv.rotary_frequencies(2, 1e4, lv.RotaryScaling("base", 2.0)), "more than one pair"),
])
def test_rotary_refusals(make, message) -> None:
    with pytest.raises(ValueError, match=message):
        make()


def test_rotary_needs_a_gpu() -> None:
    with pytest.raises(lv.ExecutionError, match="GPU"):
        lv.RotaryEmbedding(64, device="cpu")


# ---- the planner -------------------------------------------------------------------

@pytest.mark.parametrize("seed", range(12))
def test_pieces_cover_every_column_group_once(seed) -> None:
    rng = np.random.default_rng(seed)
    bs, heads = int(rng.choice((1, 12, 16, 64))), int(rng.choice((1, 5, 16, 128)))
    tiles, resident = int(rng.choice((1, 2, 4, 8))), int(rng.choice((3, 64, 512)))
    computed, layouts = [], []
    for _ in range(int(rng.integers(1, 9))):
        n = int(rng.choice((1, 1, 2, 9, 33, 70)))
        tree = rng.random() < 0.4
        layouts.append(tuple([-1] + [int(rng.integers(0, i)) for i in range(1, n)] if tree else range(-1, n - 1)))
        computed.append(int(rng.choice((0, 1, 31, 32, 500, 4000))))
    need = [-(-(c + len(p)) // bs) for c, p in zip(computed, layouts)]
    ids = iter(rng.permutation(sum(need)).tolist())
    tables = tuple(tuple(next(ids) for _ in range(n)) for n in need)
    md = lv.PagedAttentionMetadata(block_tables=tables, num_computed_tokens=tuple(computed),
                                   query_layouts=tuple(lv.QueryLayout(p) for p in layouts))
    plan = StepPlan(md, block_size=bs, device=CPU, num_blocks=sum(need))
    xcds = int(rng.choice((1, 4, 8)))
    found = native.host().latent_work(plan._req_meta, plan.facts.flat, heads, tiles, resident, bs, 32, 256, xcds)
    pieces, jobs, groups, slots, most, depth = found
    pieces = np.frombuffer(pieces, np.int32).reshape(-1, native.PIECE_FIELDS)
    jobs = np.frombuffer(jobs, np.int32).reshape(-1, native.MERGE_FIELDS)
    assert groups <= resident or groups * 32 * 256 >= sum(c + len(p) for c, p in zip(computed, layouts))
    order = []  # as the workgroups walk them
    for w in range(groups):
        while w >= 0:
            order.append(w)
            w = int(pieces[w][11])
    assert sorted(order) == list(range(len(pieces)))
    by_segment: dict = {}
    for x in pieces[order]:
        off, lb = sum(need[:x[0]]), x[2] // bs
        if (x[2] % bs + 31) // bs >= 4:
            assert (x[12:] == -1).all()
        else:
            table = tables[x[0]][lb:-(-int(x[3]) // bs)][:4]
            assert tuple(x[12:12 + len(table)]) == table
        by_segment.setdefault((int(x[0]), int(x[1])), []).append(x)
        off = sum(need[:x[0]])
        assert x[5] == off and x[6] == computed[x[0]] and x[7] == len(layouts[x[0]])
    for got in by_segment.values():
        got.sort(key=lambda x: x[2])  # (the workgroups are dealt to the XCDs)
    want = set()
    for r, (c, p) in enumerate(zip(computed, layouts)):
        columns = len(p) * heads
        for g in range(-(-columns // (16 * tiles))):
            want.add((r, g))
            linear = p == tuple(range(-1, len(p) - 1))
            last = (min(columns, (g + 1) * 16 * tiles) - 1) // heads if linear else len(p) - 1
            got = by_segment[(r, g)]
            assert got[0][2] == 0 and got[-1][3] == c + last + 1
            assert all(a[3] == b[2] and a[3] % 32 == 0 for a, b in zip(got, got[1:])) and all(x[2] < x[3] for x in got)
            if len(got) == 1:
                assert got[0][4] == -1
            else:
                assert [int(x[4]) for x in got] == list(range(got[0][4], got[0][4] + len(got)))
    assert want == set(by_segment)
    split = {k: v for k, v in by_segment.items() if len(v) > 1}
    assert slots == sum(map(len, split.values())) and len(jobs) == len(split)
    for j in jobs:
        v = split[(int(j[0]), int(j[1]))]
        assert j[2] == v[0][4] and j[3] == len(v) <= depth
        columns = len(layouts[j[0]]) * heads - int(j[1]) * 16 * tiles
        assert min(columns, 16 * tiles) <= most


def test_column_groups_of_the_same_tokens_share_an_xcd() -> None:
    """Four column groups per request, four shares each: the workgroups over the same
    tokens of a request differ by whole rounds of the XCDs."""
    md = lv.PagedAttentionMetadata(block_tables=tuple(tuple(range(64 * r, 64 * r + 64)) for r in range(16)),
                                   num_computed_tokens=(1023,) * 16, query_layouts=(lv.linear_query_layout(1),) * 16)
    plan = StepPlan(md, block_size=16, device=CPU, num_blocks=1024)
    pieces, _, groups, *_ = native.host().latent_work(plan._req_meta, plan.facts.flat, 64, 1, 256, 16, 32, 256, 8)
    pieces = np.frombuffer(pieces, np.int32).reshape(-1, native.PIECE_FIELDS)
    assert groups == 256 == len(pieces)
    where: dict = {}
    for w, x in enumerate(pieces):
        where.setdefault((int(x[0]), int(x[2])), []).append((int(x[1]), w % 8))
    assert len(where) == 64
    for found in where.values():
        assert sorted(g for g, _ in found) == [0, 1, 2, 3] and len({xcd for _, xcd in found}) == 1


def test_latent_work_refuses_nonsense() -> None:
    meta, flat = np.zeros(8, np.int32), np.zeros(1, np.int32)
    for args in ((0, 1, 4, 16, 32, 256, 8), (16, 0, 4, 16, 32, 256, 8), (16, 1, 0, 16, 32, 256, 8), (16, 1, 4, 0, 32, 256, 8),
                 (16, 1, 4, 16, 32, 256, 0)):
        with pytest.raises(ValueError, match="inconsistent"):
            native.host().latent_work(meta, flat, *args)


# ---- the oracle --------------------------------------------------------------------

def test_oracle_forms_agree() -> None:
    """The absorbed queries over the rows, times value_up, are the per-head form."""
    rng = np.random.default_rng(3)
    latent, rope, heads, nope, value, bs = 24, 8, 3, 10, 6, 4
    rows = rng.standard_normal((40, latent + rope))
    key_up, value_up = rng.standard_normal((heads, nope, latent)), rng.standard_normal((heads, value, latent))
    tables, computed, parents = ((3, 1, 7), (0, 9)), (5, 0), ((-1, 0, 0, 1), (-1, 0, 1))
    q = rng.standard_normal((7, heads, nope + rope))
    absorbed = np.concatenate((np.einsum("thn,hnl->thl", q[..., :nope], key_up), q[..., nope:]), axis=2)
    args = (rows, tables, computed, parents, bs, latent)
    u, _, _ = Z.attention(absorbed, *args, scale=0.3)
    want, _, _ = Z.attention(q, *args, scale=0.3, key_up=key_up, value_up=value_up)
    assert np.allclose(np.einsum("thl,hvl->thv", u, value_up), want, rtol=1e-12, atol=1e-12)


def test_oracle_rotation_keeps_lengths_and_angles_add() -> None:
    rng = np.random.default_rng(4)
    x = rng.standard_normal((5, 2, 8))
    a, b = rng.standard_normal((2, 5, 4))
    for interleaved in (True, False):
        y = Z.rotate(Z.rotate(x, np.cos(a), np.sin(a), interleaved), np.cos(b), np.sin(b), interleaved)
        assert np.allclose(y, Z.rotate(x, np.cos(a + b), np.sin(a + b), interleaved))
        assert np.allclose(np.linalg.norm(y, axis=-1), np.linalg.norm(x, axis=-1))


def test_column_tiles_of_a_step() -> None:
    """The widest request's columns; 128 only where the workgroups of 64 would have
    many tiles each."""
    from light_vllm_amd.latent_attention import TILE_ROWS, WIDE_TILES, choose_col_tiles

    def tiles(heads, q, total, resident=256):
        return choose_col_tiles(np.asarray(q), np.asarray(total), heads, lambda t: resident)

    assert [tiles(h, [1, 1], [9, 9]) for h in (1, 16, 17, 32, 33, 64, 65, 128)] == [1, 1, 2, 2, 4, 4, 4, 4]
    assert tiles(16, [1, 3], [5000, 7]) == 4
    enough = TILE_ROWS * WIDE_TILES * 256  # of one request with 65 to 128 columns: two groups of 64
    assert tiles(128, [1], [enough // 2]) == 8
    assert tiles(128, [1], [enough // 2 - TILE_ROWS]) == 4
    assert tiles(16, [9], [enough // 3 + TILE_ROWS]) == 8
