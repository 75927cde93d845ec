"""Attention over a ``LatentPagedKVCache``: the per-step context.

Head h's key of a token is ``[key_up[h] c, r]`` and its value ``value_up[h] c``,
with the token's latent c and rotated key r.  Multiplied out the other way
round, key_up^T into the query and value_up behind the softmax, every head
attends the rows of the cache themselves (the absorbed form): a row is read
once for all heads.
"""

from __future__ import annotations

import torch
from torch import Tensor

from light_vllm_amd import errors, native
from light_vllm_amd.latent_cache import LatentLayerSpec, aligned_rows, append_rows, check_rotary, check_rows
from light_vllm_amd.paged_cache import dtype_code
from light_vllm_amd.plan import DECODE_MERGE_PIECES, StepPlan, current_stream
from light_vllm_amd.quantized_cache import on_device

# Column tiles (of 16) per workgroup that the kernel is built for.
COL_TILES = (1, 2, 4)


class _Shape:
    """One layer shape's launch facts in a step plan."""

    __slots__ = ("work", "col_tiles", "acc_bytes", "workspace_bytes")

    def __init__(self, work, col_tiles: int, latent_size: int) -> None:
        self.work, self.col_tiles = work, col_tiles
        columns = work.num_partial_slots * 16 * col_tiles
        self.acc_bytes = columns * latent_size * 4
        self.workspace_bytes = self.acc_bytes + columns * 8


class _Work:
    """Work lists of one layer shape, in the form ``StepPlan`` uploads."""

    __slots__ = ("pieces_host", "first_host", "jobs_host", "pieces_ptr", "first_ptr", "jobs_ptr", "num_groups",
                 "num_partial_slots", "merge_columns", "num_jobs")

    def __init__(self, found) -> None:
        pieces, first, jobs, groups, _, slots, columns, _, _ = found
        self.pieces_host, self.first_host, self.jobs_host = (_i32(x) for x in (pieces, first, jobs))
        self.pieces_ptr = self.first_ptr = self.jobs_ptr = None
        self.num_groups, self.num_partial_slots, self.merge_columns = int(groups), int(slots), int(columns)
        self.num_jobs = self.jobs_host.size // native.MERGE_FIELDS

    def parts(self):
        found = [("pieces_ptr", self.pieces_host), ("first_ptr", self.first_host), ("jobs_ptr", self.jobs_host)]
        return [(name, array) for name, array in found if array.size]


def _i32(data):
    import numpy as np

    return np.frombuffer(data, dtype=np.int32)


def choose_col_tiles(q_lens, heads: int) -> int:
    """Column tiles per workgroup of a step: those of its widest request, as far
    as the kernel is built (a wider workgroup reads a row once for more
    columns)."""

    widest = -(-int(q_lens.max()) * heads // 16)
    return next((t for t in COL_TILES if t >= widest), COL_TILES[-1])


class LatentStepPlan(StepPlan):
    """A step plan with the latent kernels' work lists per (heads, sizes)."""

    def shape(self, spec: LatentLayerSpec, code: int) -> _Shape:
        key = (spec.num_query_heads, spec.latent_size, spec.rope_size, code)
        found = self.launches.get(key)
        if found is None:
            heads = spec.num_query_heads
            tiles = choose_col_tiles(self.facts.q_lens, heads)
            resident = native.latent_decode_resident_groups(code, spec.latent_size, spec.rope_size, tiles)
            work = _Work(native.host().latent_work(
                self._req_meta, self.facts.flat, heads, tiles, resident, self.block_size,
                int(native.load().lvamd_latent_decode_tile_tokens()), DECODE_MERGE_PIECES))
            self._register(key, work)
            found = self.launches[key] = _Shape(work, tiles, spec.latent_size)
        return found


class HipLatentPagedAttention:
    """Per-step context: writes each layer's rows, then attends them."""

    # forward takes rotary=(cosines, sines): the append turns keys and queries.
    supports_rotary = True

    def __init__(self, backend, cache, plan: LatentStepPlan) -> None:
        self._backend = backend
        self._cache = cache
        self._plan = plan
        self._layer_ids: set[str] = set()

    @property
    def layer_ids(self) -> frozenset[str]:
        return frozenset(self._layer_ids)

    @property
    def plan(self) -> LatentStepPlan:
        return self._plan

    def forward(self, layer_id: str, query: Tensor, latent: Tensor, rope_key: Tensor, *, scale: float,
                rotary: tuple[Tensor, Tensor] | None = None) -> Tensor:
        """Append this layer's rows, then attend what the cache holds.

        ``query`` ``[tokens, heads, latent_size + rope_size]``: the heads' queries
        multiplied by their key weights, then their rotated parts; returns
        ``[tokens, heads, latent_size]``, to be multiplied by the heads' value
        weights.  ``latent`` ``[tokens, latent_size]`` and ``rope_key`` ``[tokens,
        rope_size]`` are the step's rows.  With ``rotary=(cosines, sines)`` (fp32
        ``[tokens, rope_size / 2]``, ``RotaryEmbedding``) keys and queries come
        unrotated and the append's launch turns both."""

        cache, plan = self._cache, self._plan
        cfg = cache.config
        if layer_id in self._layer_ids:
            raise errors.KVCacheError(f"paged attention layer {layer_id!r} ran more than once")
        self._layer_ids.add(layer_id)
        spec = cache.layer_spec(layer_id)
        heads, size, rope = spec.num_query_heads, spec.latent_size, spec.rope_size
        for holds, message in (
            (lambda: query.ndim == 3, "paged attention query must have three dimensions"),
            (lambda: query.shape[0] == plan.num_query_tokens,
             "paged attention metadata token count does not match query"),
            (lambda: tuple(query.shape[1:]) == (heads, size + rope),
             "paged attention query shape does not match the layer spec"),
            (lambda: latent.ndim == 2 and latent.shape[0] == query.shape[0],
             "paged attention query and latent token dimensions must match"),
            (lambda: query.dtype == cfg.dtype and query.device == cfg.device,
             "HIP paged attention query dtype and device must match the KV cache"),
        ):
            if not holds():
                raise errors.KVCacheError(message)
        check_rows(cfg, spec, latent, rope_key)
        angles = check_rotary(spec, rotary, latent)
        query = aligned_rows(query)
        query_rope = query[..., size:]
        with on_device(cfg.device):
            code = dtype_code(cfg.dtype)
            shape = plan.shape(spec, code)
            turned = append_rows(cache, spec, latent, rope_key, angles, plan.slots_ptr, None, plan.num_tokens,
                                 None if angles is None else query_rope)
            query_rope = query_rope if turned is None else turned
            out = torch.empty((query.shape[0], heads, size), dtype=cfg.dtype, device=cfg.device)
            # (Of the call's own stream or graph: no two share one.)
            workspace = torch.empty(shape.workspace_bytes, dtype=torch.uint8, device=cfg.device)
            part_acc = workspace.data_ptr() if shape.workspace_bytes else None
            work = shape.work
            native.check(native.load().lvamd_latent_decode(
                query.data_ptr(), query.stride(0), query.stride(1), query_rope.data_ptr(), query_rope.stride(0),
                query_rope.stride(1), cache.layer(layer_id).rows.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1),
                work.pieces_ptr, work.first_ptr, work.num_groups, work.jobs_ptr, work.num_jobs, work.merge_columns,
                plan.tables_ptr, plan.vis_ptr, part_acc, None if part_acc is None else part_acc + shape.acc_bytes,
                work.num_partial_slots, heads, size, rope, shape.col_tiles, plan.block_size, float(scale), code,
                current_stream(cfg.device)), "lvamd_latent_decode")
        return out
