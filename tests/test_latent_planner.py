"""Host tests of the latent kernel's work lists at the tile of every width (CPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import light_vllm_amd as lv
from light_vllm_amd import native
from light_vllm_amd.plan import StepPlan


def _lists(seed):
    rng = np.random.default_rng(seed)
    bs, heads = int(rng.choice((1, 12, 16, 64))), int(rng.choice((1, 5, 16, 40, 128)))
    tiles, resident = int(rng.choice((1, 2, 4, 8))), int(rng.choice((3, 64, 512)))
    unit = int(native.load().lvamd_latent_decode_tile_tokens(tiles))
    computed, layouts = [], []
    for _ in range(int(rng.integers(1, 9))):
        n = int(rng.choice((1, 1, 2, 9, 33, 70)))
        tree = rng.random() < 0.4
        layouts.append(tuple([-1] + [int(rng.integers(0, i)) for i in range(1, n)] if tree else range(-1, n - 1)))
        computed.append(int(rng.choice((0, 1, 31, 32, 63, 64, 500, 4000))))
    need = [-(-(c + len(p)) // bs) for c, p in zip(computed, layouts)]
    ids = iter(rng.permutation(sum(need)).tolist())
    tables = tuple(tuple(next(ids) for _ in range(n)) for n in need)
    md = lv.PagedAttentionMetadata(block_tables=tables, num_computed_tokens=tuple(computed),
                                   query_layouts=tuple(lv.QueryLayout(p) for p in layouts))
    plan = StepPlan(md, block_size=bs, device=torch.device("cpu"), num_blocks=sum(need))
    found = native.host().latent_work(plan._req_meta, plan.facts.flat, heads, tiles, resident, bs, unit, 256, int(rng.choice((1, 8))))
    pieces = np.frombuffer(found[0], np.int32).reshape(-1, native.PIECE_FIELDS)
    jobs = np.frombuffer(found[1], np.int32).reshape(-1, native.MERGE_FIELDS)
    return bs, heads, 16 * tiles, unit, tables, computed, layouts, pieces, jobs, int(found[2]), int(found[3])


def test_tiles_of_every_width() -> None:
    assert [native.load().lvamd_latent_decode_tile_tokens(t) for t in (1, 2, 4, 8)] == [32, 32, 64, 32]


@pytest.mark.parametrize("seed", range(40))
def test_pieces_cover_and_append_every_row(seed) -> None:
    """Each column group's pieces follow one another over all rows that a column sees,
    cut at whole tiles; the group that holds a token's first column has that token's row
    (it writes the row to the pool); the first blocks are the table's."""
    bs, heads, columns, unit, tables, computed, layouts, pieces, jobs, groups, slots = _lists(seed)
    walked = []
    for w in range(groups):
        while w >= 0:
            walked.append(w)
            w = int(pieces[w][11])
    assert sorted(walked) == list(range(len(pieces)))
    by_group: dict = {}
    for x in pieces:
        by_group.setdefault((int(x[0]), int(x[1])), []).append(x)
        blocks = tables[x[0]][x[2] // bs:-(-int(x[3]) // bs)]
        if (x[2] % bs + unit - 1) // bs >= 4:
            assert (x[12:] == -1).all()
        else:
            assert tuple(x[12:12 + min(4, len(blocks))]) == blocks[:4]
    taken = []
    for r, (c, parents) in enumerate(zip(computed, layouts)):
        n, linear = len(parents), parents == tuple(range(-1, len(parents) - 1))
        appended = set()
        for g in range(-(-n * heads // columns)):
            mine = sorted(by_group.pop((r, g)), key=lambda x: x[2])
            last = (min(n * heads, (g + 1) * columns) - 1) // heads if linear else n - 1
            assert mine[0][2] == 0 and mine[-1][3] == c + last + 1
            assert all(a[3] == b[2] and a[3] % unit == 0 for a, b in zip(mine, mine[1:])) and all(x[2] < x[3] for x in mine)
            assert (mine[0][4] == -1) == (len(mine) == 1)
            taken += [int(x[4]) for x in mine if x[4] >= 0]
            rows = {p - c for x in mine for p in range(max(c, x[2]), x[3])}
            here = {t for t in range(n) if g * columns <= t * heads < (g + 1) * columns}
            assert here <= rows and not here & appended
            appended |= here
        assert appended == set(range(n))
    assert not by_group and sorted(taken) == list(range(slots))
    assert sum(int(j[3]) for j in jobs) == slots
