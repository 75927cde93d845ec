"""Attention over a ``LatentPagedKVCache``: the heads' weights and the per-step
context.

Head h's key of a token is ``[key_up[h] c, r]`` and its value ``value_up[h] c``,
with the token's latent c and rotated key r.  There are two ways to the same
result:

* absorbed: key_up^T is multiplied into the query and value_up behind the
  softmax, and every head attends the rows of the cache themselves: a row is
  read once for all heads, a (query, key) pair costs 2 L + P products;
* expanded: the request's keys and values are formed per head first, and a
  pair costs N + P + V.

Single tokens, short runs and draft trees take the first, long prompt chunks the
second (``_expanded``).
"""

from __future__ import annotations

import numpy as np
import torch
from torch import Tensor

from light_vllm_amd import errors, native
from light_vllm_amd.latent_cache import LatentLayerSpec, aligned_rows, append_rows, check_rotary, check_rows
from light_vllm_amd.paged_cache import dtype_code
from light_vllm_amd.plan import DECODE_MERGE_PIECES, PREFILL_MIN_TILES, StepPlan, current_stream
from light_vllm_amd.quantized_cache import _NOT_FAST, _raw_stream, on_device

# Column tiles (of 16) per workgroup that the latent-space kernel is built for.
COL_TILES = (1, 2, 4, 8)
# Rows of a 64-column workgroup's tile, and the tiles from which 128 columns pay.
TILE_ROWS, WIDE_TILES = 64, 24
# Widest workgroup whose launch appends the step's rows itself.
APPEND_TILES = 4
WEIGHT_SIZES = (64, 128)
# Queries per unit, keys per tile and rows per expanded block of the chunk kernels.
UNIT_QUERIES, UNIT_KEYS = 128, 64
# Most bytes of expanded keys and values at a time: heads go in groups beyond it.
EXPANDED_BYTES = 1 << 30


class LatentWeights:
    """The heads' weights of one layer, laid out once: ``key_up`` ``[heads,
    nope_size, latent_size]`` and ``value_up`` ``[heads, value_size, latent_size]``
    (rows as a linear layer's, per head)."""

    __slots__ = ("key_up", "value_up", "key_down", "heads", "latent_size", "nope_size", "value_size", "sizes", "fits",
                 "addresses")

    def __init__(self, key_up: Tensor, value_up: Tensor) -> None:
        for holds, message in (
            (lambda: key_up.ndim == 3 and value_up.ndim == 3, "latent weights must have three dimensions"),
            (lambda: key_up.shape[0] == value_up.shape[0] and key_up.shape[2] == value_up.shape[2],
             "latent weights must agree in heads and latent size"),
            (lambda: key_up.shape[1] in WEIGHT_SIZES and value_up.shape[1] in WEIGHT_SIZES,
             f"nope_size and value_size must be one of {WEIGHT_SIZES}"),
            (lambda: key_up.dtype == value_up.dtype and key_up.dtype in (torch.bfloat16, torch.float16),
             "latent weights must be bfloat16 or float16, both of one dtype"),
            (lambda: key_up.device == value_up.device and key_up.device.type == "cuda",
             "latent weights must be on one GPU (cuda) device"),
        ):
            if not holds():
                raise ValueError(message)
        # (Copies, so that the rows are 16-byte chunks wherever the weights lay.)
        self.key_up = key_up.detach().clone(memory_format=torch.contiguous_format)
        self.value_up = value_up.detach().clone(memory_format=torch.contiguous_format)
        self.key_down = self.key_up.transpose(1, 2).contiguous()  # into latent space
        self.heads, self.nope_size, self.latent_size = key_up.shape
        self.value_size = value_up.shape[1]
        self.sizes = (self.nope_size, self.value_size)
        # What a layer compares, and what a launch takes.
        self.fits = (self.heads, self.latent_size, self.key_up.dtype, self.key_up.device)
        self.addresses = (self.key_down.data_ptr(), self.value_up.data_ptr(), self.nope_size, self.value_size)


class _Lists:
    """int32 arrays of a layer shape's work, in the form ``StepPlan`` uploads:
    ``ptr[name]`` is an array's device address."""

    def __init__(self, **arrays: np.ndarray) -> None:
        self._arrays = {name: a for name, a in arrays.items() if a.size}
        for name in arrays:
            setattr(self, name, None)

    def parts(self):
        return list(self._arrays.items())


class _Shape:
    """One layer shape's launch facts in a step plan."""

    __slots__ = ("facts", "out_shape", "out_strides", "scratch_bytes", "lists", "col_tiles", "num_groups", "num_jobs",
                 "merge_columns", "num_slots", "acc_bytes", "latent_bytes", "num_rows", "row_base", "num_blocks",
                 "num_units", "num_unit_jobs", "unit_merge_columns", "num_unit_slots")


_NO_STEP = ((), (None, 0, None, 0, None, None, 0, 0))


def _step_args(spec: LatentLayerSpec, latent: Tensor, rope_key: Tensor, angles) -> tuple:
    """lvamd_latent_decode's arguments of the step's rows (behind the tensors that they
    name): the launch appends them."""

    cosines, sines = angles if angles is not None else (None, None)
    return (latent, rope_key), (
        latent.data_ptr(), latent.stride(0), rope_key.data_ptr(), rope_key.stride(0),
        None if cosines is None else cosines.data_ptr(), None if sines is None else sines.data_ptr(),
        0 if cosines is None else cosines.stride(0), int(spec.rotary_layout == "interleaved"))


def choose_col_tiles(q_lens, totals, heads: int, resident) -> int:
    """Column tiles per workgroup of a step: those of its widest request, as far
    as the kernel is built; 128 columns only where 64 would give each of the
    ``resident(4)`` workgroups at least ``WIDE_TILES`` tiles.

    A wider workgroup reads a row once for more columns; a narrower one writes fewer
    partials, up to 64 columns the launch appends, and of up to 32 columns two fit a CU.
    Measured (us, 16/32/64/128 columns): 16 heads, 64 requests x 2300 tokens 43 / 43 /
    49 / 67; 16 x 32767 tokens 114 / 119 / 146 / 178; 64 columns against 128: 128 heads,
    32 x 2300 (9 tiles per workgroup) 51 / 63, 64 x 2300 (18 tiles) 87 / 88, 256 x 1000 (32
    tiles) 152 / 113, 8 x 32767 (32 tiles) 128 / 119; 16 heads, 9 queries, 32 x 8000 (48
    tiles) 195 / 192, and some 5 more for the launches of 128 columns where the host
    sets the pace."""

    widest = -(-int(q_lens.max()) * heads // 16)
    fits = next((t for t in COL_TILES if t >= widest), COL_TILES[-1])
    if fits > APPEND_TILES:
        tiles = int((-(-totals // TILE_ROWS) * -(-q_lens * heads // (16 * APPEND_TILES))).sum())
        if tiles < WIDE_TILES * resident(APPEND_TILES):
            return APPEND_TILES
    return fits


def _expanded(facts, spec: LatentLayerSpec, nope: int, value: int) -> np.ndarray:
    """Which requests take the expanded form: linear ones where its products (with
    the expansion of every key) are fewer than 1.2 times the absorbed form's, which
    run at the lower rate.  Fewer than 64 queries cost as much as 64, keys count in
    32s.

    Measured (us, absorbed / expanded; one request, 16 heads, 512 + 64, 128 / 128):
    behind 1024 tokens 32 / 32 for 16 queries, 45 / 34 for 64, 65 / 38 for 256;
    behind 8192 44 / 80, 66 / 87, 150 / 108; behind 32768 60 / 259, 144 / 265, 379 / 319,
    with 512 queries 688 / 389; eight requests behind 8192 95 / 559, 242 / 565, 716 /
    601.  Over 111 steps of 16 to 128 heads the choice is 1.5 % off the better form's
    time, at most 1.4 times (32 queries of 128 heads, no history: 37 / 52)."""

    n, c = facts.q_lens.astype(np.float64), facts.computed.astype(np.float64)
    latent, rope = spec.latent_size, spec.rope_size
    keys, held = c + n / 2, -(-(c + n) // 32) * 32
    absorbed = n * keys * (2 * latent + rope) + n * latent * (nope + value)
    expanded = np.maximum(n, 64) * keys * (nope + rope + value) + held * latent * (nope + value)
    return (facts.vis_off < 0) & (expanded < 1.2 * absorbed)


class LatentStepPlan(StepPlan):
    """A step plan with the latent kernels' work lists per layer shape.

    It may be used on streams that run after the one it was made on (``reuse`` sees to
    that where a later step takes it), and dropped while their work is pending."""

    def __init__(self, *args, **kwargs) -> None:
        super().__init__(*args, **kwargs)
        self._stream = current_stream(self._staging.device)  # the allocator's, for the lists
        self._behind = {self._stream}  # streams that run after the lists' upload
        index = self._staging.device.index
        self._index = torch.cuda.current_device() if index is None else index

    def _made_on(self):
        device = self._staging.device
        return torch.cuda.ExternalStream(self._stream, device=device) if self._stream else torch.cuda.default_stream(device)

    def reuse(self) -> None:
        """Before another context of this plan: the current stream waits for the upload
        if that is another's.  (A stream that is captured can wait for nothing outside
        its graph: the capture began after the upload.)"""

        stream = _raw_stream(self._index)
        if stream not in self._behind and not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(self._staging.device).wait_stream(self._made_on())
            self._behind.add(stream)

    def use_on(self, stream: int) -> None:
        """Before a launch on ``stream``, the current one: the lists are that
        stream's until then, whoever drops the plan."""

        if stream != self._stream:
            for blob in (self._blob, *self._late_blobs):
                blob.record_stream(torch.cuda.current_stream(self._staging.device))

    def shape(self, spec: LatentLayerSpec, code: int, weights: tuple[int, int] | None) -> _Shape:
        """``weights``: (nope_size, value_size), or None where queries come
        absorbed."""

        key = (spec.num_query_heads, spec.latent_size, spec.rope_size, code, weights)
        found = self.launches.get(key)
        if found is None:
            if self._committed and torch.cuda.is_current_stream_capturing():
                raise errors.ExecutionError("a step of this form must run once before it is captured (its work lists are "
                                            "uploaded then)")
            found = self._plan_shape(spec, code, weights)
            late = self._committed
            self._register(key, found.lists)
            if late:
                # (The next launch may be on another stream than this one.)
                torch.cuda.current_stream(self._staging.device).synchronize()
                for blob in self._late_blobs:
                    blob.record_stream(self._made_on())
            self.launches[key] = found
        return found

    def bind(self, x: _Shape, spec: LatentLayerSpec, config, code: int, weights: tuple[int, int] | None) -> None:
        """What one native call takes of a step that needs no launch beside the
        latent-space kernel's (the lists are uploaded by now)."""

        index = config.device.index if config.device.index is not None else torch.cuda.current_device()
        heads, lists = spec.num_query_heads, x.lists
        x.facts = (
            config.dtype, torch.float32, _raw_stream, index, native.entry("lvamd_latent_decode"),
            native.entry("lvamd_latent_heads"), self.num_tokens, heads, spec.latent_size, spec.rope_size, code,
            int(spec.rotary_layout == "interleaved"), lists.pieces, x.num_groups, lists.jobs or 0, x.num_jobs,
            x.merge_columns, self.tables_ptr, self.vis_ptr, x.num_slots, x.col_tiles, self.block_size, x.acc_bytes,
            x.latent_bytes, lists.rows or 0, x.num_rows, x.row_base)
        x.scratch_bytes = x.latent_bytes + (0 if weights is None else 4 * x.num_rows * heads * spec.latent_size)
        width = spec.latent_size if weights is None else weights[1]
        x.out_shape, x.out_strides = (self.num_tokens, heads, width), (heads * width, width, 1)

    def _plan_shape(self, spec: LatentLayerSpec, code: int, weights: tuple[int, int] | None) -> _Shape:
        facts, heads, host = self.facts, spec.num_query_heads, native.host()
        if int(facts.q_lens.max()) * heads > 2**31 - 1:
            raise errors.KVCacheError("a request's queries times its heads must be below 2**31")
        none = np.zeros(0, np.int32)
        meta = self._req_meta.reshape(-1, native.REQ_FIELDS)
        long = np.zeros(self.batch_size, bool) if weights is None else _expanded(facts, spec, *weights)
        short = ~long
        x = _Shape()
        x.facts = None
        pieces = jobs = rows = blocks = units = unit_jobs = none
        x.num_groups = x.num_jobs = x.num_slots = x.merge_columns = x.num_rows = 0
        x.row_base, x.col_tiles = 0, COL_TILES[0]
        x.num_blocks = x.num_units = x.num_unit_jobs = x.unit_merge_columns = x.num_unit_slots = 0
        if short.any():
            def groups(col_tiles: int) -> int:
                return native.latent_decode_resident_groups(code, spec.latent_size, spec.rope_size, col_tiles)

            x.col_tiles = choose_col_tiles(facts.q_lens[short], (facts.computed + facts.q_lens)[short], heads, groups)
            resident = groups(x.col_tiles)
            mine = meta[short].copy()
            found = host.latent_work(mine, facts.flat, heads, x.col_tiles, resident, self.block_size,
                                     int(native.load().lvamd_latent_decode_tile_tokens(x.col_tiles)), DECODE_MERGE_PIECES,
                                     native.xcd_count())
            pieces, jobs = (np.frombuffer(a, dtype=np.int32) for a in found[:2])
            x.num_groups, x.num_slots, x.merge_columns = (int(v) for v in found[2:5])
            x.num_jobs = jobs.size // native.MERGE_FIELDS
            # Rows in latent space: the short requests' one after the other (without weights
            # the step's own).
            ends = np.cumsum(mine[:, 3], dtype=np.int32)
            first = mine[:, 4] if weights is None else ends - mine[:, 3]
            for records, fields in ((pieces, native.PIECE_FIELDS), (jobs, native.MERGE_FIELDS)):
                request = records.reshape(-1, fields)[:, 0]
                request[:] = first[request]
            x.num_rows, x.row_base = int(ends[-1]), int(mine[0, 4])
            if x.num_rows != int(mine[-1, 4] + mine[-1, 3]) - x.row_base:
                rows = np.concatenate([np.arange(s, s + n, dtype=np.int32) for s, n in zip(mine[:, 4], mine[:, 3])])
        if long.any():
            mine = meta[long].copy()
            total = (mine[:, 2] + mine[:, 3]).astype(np.int64)
            per = -(-total // UNIT_KEYS)
            base = np.cumsum(per) - per
            blocks = np.zeros((int(per.sum() + 1) // 2 * 2, 4), np.int32)
            blocks[:, 2] = 1  # (a padding block repeats the first table's first row)
            for b, k, off, t in zip(base, per, mine[:, 0], total):
                blocks[b:b + k, 0], blocks[b:b + k, 1], blocks[b:b + k, 2] = off, np.arange(k) * UNIT_KEYS, t
            mine[:, 0], mine[:, 1] = base, per
            resident = native.latent_prefill_resident_units(code, weights[0], spec.rope_size, weights[1])
            found = host.prefill_work(mine, np.zeros(blocks.shape[0], np.int32), 1, UNIT_QUERIES, UNIT_KEYS, resident // heads,
                                      PREFILL_MIN_TILES, 0, UNIT_KEYS, 0, heads, 0, 2)
            units, unit_jobs = (np.frombuffer(a, dtype=np.int32) for a in found[:2])
            x.num_blocks, x.num_units = blocks.shape[0], units.size // native.PREFILL_FIELDS
            x.num_unit_jobs, x.num_unit_slots = unit_jobs.size // native.MERGE_FIELDS, int(found[2])
            x.unit_merge_columns = int(found[4])
        columns = x.num_slots * 16 * x.col_tiles
        x.acc_bytes = columns * spec.latent_size * 4
        x.latent_bytes = x.acc_bytes + columns * 8
        x.lists = _Lists(pieces=pieces, jobs=jobs, rows=rows, blocks=blocks.reshape(-1), units=units,
                         unit_jobs=unit_jobs)
        return x


class HipLatentPagedAttention:
    """Per-step context: writes each layer's rows, then attends them."""

    # forward takes rotary=(cosines, sines): the append turns keys and queries.
    supports_rotary = True

    def __init__(self, cache, plan: LatentStepPlan, forms: dict) -> None:
        """``forms``: of the backend, what the cache's steps have taken."""

        self._cache = cache
        self._plan = plan
        self._layer_ids: set[str] = set()
        self._forms = forms
        self._attend = native.host().latent_attend

    @property
    def layer_ids(self) -> frozenset[str]:
        return frozenset(self._layer_ids)

    @property
    def plan(self) -> LatentStepPlan:
        return self._plan

    def forward(self, layer_id: str, query: Tensor, latent: Tensor, rope_key: Tensor, *, scale: float,
                rotary: tuple[Tensor, Tensor] | None = None, weights: LatentWeights | None = None) -> Tensor:
        """Append this layer's rows, then attend what the cache holds.

        With ``weights``: ``query`` ``[tokens, heads, nope_size + rope_size]``, returns
        ``[tokens, heads, value_size]``.  Without: ``query`` ``[tokens, heads,
        latent_size + rope_size]``, the heads' queries multiplied by their key weights
        already, and what returns, ``[tokens, heads, latent_size]``, has yet to be
        multiplied by their value weights.  ``latent`` ``[tokens, latent_size]`` and
        ``rope_key`` ``[tokens, rope_size]`` are the step's rows.  With
        ``rotary=(cosines, sines)`` (fp32 ``[tokens, rope_size / 2]``,
        ``RotaryEmbedding``) keys and queries come unrotated and the append's launch
        turns both.

        With weights, a query's part in latent space and what attention gives there
        are rounded to the cache's dtype, as are a long chunk's keys and values."""

        cache, plan = self._cache, self._plan
        cfg = cache.config
        if layer_id in self._layer_ids:
            raise errors.KVCacheError(f"paged attention layer {layer_id!r} ran more than once")
        self._layer_ids.add(layer_id)
        spec = cache.layer_spec(layer_id)
        # The common case in one native call: it reads the tensors itself and
        # launches when every rule holds; anything else takes the general path, which
        # raises the first broken rule's message.
        sizes = None if weights is None else weights.sizes
        code = dtype_code(cfg.dtype)
        form = (spec.num_query_heads, spec.latent_size, spec.rope_size, code, sizes)
        shape = plan.launches.get(form)
        if (shape is not None and shape.num_units == 0 and shape.col_tiles <= APPEND_TILES
                and (weights is None or weights.fits == (spec.num_query_heads, spec.latent_size, cfg.dtype, cfg.device))
                and (rotary is None or (type(rotary) is tuple and len(rotary) == 2 and rotary[0] is not None))):
            facts = shape.facts
            if facts is None or facts[11] != (spec.rotary_layout == "interleaved"):
                plan.bind(shape, spec, cfg, code, sizes)
                facts = shape.facts
            if torch.cuda.current_device() == facts[3]:
                plan.use_on(_raw_stream(facts[3]))
                out = torch.empty_strided(shape.out_shape, shape.out_strides, dtype=cfg.dtype, device=cfg.device)
                # (Of the call's own stream or graph: no two share one.)
                scratch = torch.empty_strided((shape.scratch_bytes,), (1,), dtype=torch.uint8,
                                              device=cfg.device) if shape.scratch_bytes else None
                cosines, sines = rotary if rotary is not None else (None, None)
                status = self._attend(facts, cache.pool_ptr(layer_id), query, latent, rope_key, cosines, sines, scale,
                                      out.data_ptr(), 0 if scratch is None else scratch.data_ptr(),
                                      None if weights is None else weights.addresses)
                if status == 0:
                    if form not in self._forms:
                        self._forms[form] = spec
                    return out
                if status != _NOT_FAST:
                    native.check(status, "lvamd_latent_decode")
        return self._forward_general(spec, query, latent, rope_key, scale, rotary, weights)

    def _forward_general(self, spec, query, latent, rope_key, scale, rotary, weights) -> Tensor:
        """Every rule, then the launches for any row strides and forms."""

        cache, plan = self._cache, self._plan
        cfg, layer_id = cache.config, spec.layer_id
        heads, rope = spec.num_query_heads, spec.rope_size
        size = spec.latent_size if weights is None else weights.nope_size
        for holds, message in (
            (lambda: query.ndim == 3, "paged attention query must have three dimensions"),
            (lambda: query.shape[0] == plan.num_query_tokens,
             "paged attention metadata token count does not match query"),
            (lambda: weights is None or (weights.heads, weights.latent_size) == (heads, spec.latent_size),
             "latent weights do not match the layer spec"),
            (lambda: weights is None or (weights.key_up.dtype == cfg.dtype and weights.key_up.device == cfg.device),
             "latent weights dtype and device must match the KV cache"),
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
        sizes = None if weights is None else (weights.nope_size, weights.value_size)
        with on_device(cfg.device):
            code, stream = dtype_code(cfg.dtype), current_stream(cfg.device)
            shape = plan.shape(spec, code, sizes)
            plan.use_on(stream)
            self._forms[(heads, spec.latent_size, rope, code, sizes)] = spec
            width = spec.latent_size if weights is None else weights.value_size
            out = torch.empty((query.shape[0], heads, width), dtype=cfg.dtype, device=cfg.device)
            rows = cache.layer(layer_id).rows
            if shape.num_units or shape.col_tiles > APPEND_TILES:
                # (The expansion reads the pool: the whole step is appended first.)
                turned = append_rows(cache, spec, latent, rope_key, angles, plan.slots_ptr, None, plan.num_tokens,
                                     None if angles is None else query_rope)
                query_rope = query_rope if turned is None else turned
                step = _NO_STEP
            else:
                step = _step_args(spec, aligned_rows(latent), aligned_rows(rope_key), angles)
            if weights is None:
                self._attend_latent(spec, shape, query, query_rope, step, rows, out, scale, code, stream)
            elif shape.num_rows:
                self._attend_short(spec, shape, weights, query, query_rope, step, rows, out, scale, code, stream)
            if shape.num_units:
                self._attend_long(spec, shape, weights, query, query_rope, rows, out, scale, code, stream)
        return out

    def _attend_latent(self, spec, shape, query, query_rope, step, rows, out, scale, code, stream) -> None:
        """The latent-space kernel and its merge."""

        plan, lists = self._plan, shape.lists
        # (Of the call's own stream or graph: no two share one.)
        workspace = torch.empty(shape.latent_bytes, dtype=torch.uint8, device=rows.device)
        acc = workspace.data_ptr() if shape.latent_bytes else None
        native.check(native.load().lvamd_latent_decode(
            query.data_ptr(), query.stride(0), query.stride(1), query_rope.data_ptr(),
            query_rope.stride(0), query_rope.stride(1), *step[1], rows.data_ptr(),
            out.data_ptr(), out.stride(0), out.stride(1), lists.pieces, shape.num_groups,
            lists.jobs, shape.num_jobs, shape.merge_columns, plan.tables_ptr, plan.vis_ptr, acc,
            None if acc is None else acc + shape.acc_bytes, shape.num_slots, spec.num_query_heads, spec.latent_size,
            spec.rope_size, shape.col_tiles, plan.block_size, float(scale), code, stream), "lvamd_latent_decode")

    def _attend_short(self, spec, shape, weights, query, query_rope, step, rows, out, scale, code, stream) -> None:
        """The absorbed form: into latent space, attention there, and out of it."""

        lib, heads, where = native.load(), spec.num_query_heads, shape.lists.rows
        base = shape.row_base if where is None else 0
        both = torch.empty((2, shape.num_rows, heads, spec.latent_size), dtype=query.dtype, device=query.device)
        absorbed, attended = both.unbind(0)
        es = query.element_size()
        native.check(lib.lvamd_latent_heads(
            query.data_ptr() + base * query.stride(0) * es, query.stride(0), query.stride(1), weights.key_down.data_ptr(),
            absorbed.data_ptr(), absorbed.stride(0), absorbed.stride(1), where, None, shape.num_rows, heads, weights.nope_size,
            spec.latent_size, code, stream), "lvamd_latent_heads")
        self._attend_latent(spec, shape, absorbed, query_rope, step, rows, attended, scale, code, stream)
        native.check(lib.lvamd_latent_heads(
            attended.data_ptr(), attended.stride(0), attended.stride(1), weights.value_up.data_ptr(),
            out.data_ptr() + base * out.stride(0) * es, out.stride(0), out.stride(1), None, where, shape.num_rows, heads,
            spec.latent_size, weights.value_size, code, stream), "lvamd_latent_heads")

    def _attend_long(self, spec, shape, weights, query, query_rope, rows, out, scale, code, stream) -> None:
        """The expanded form: per-head keys and values, then attention over them."""

        lib, plan, lists, heads = native.load(), self._plan, shape.lists, spec.num_query_heads
        keys, es = shape.num_blocks * UNIT_KEYS, query.element_size()
        nope, value, latent = weights.nope_size, weights.value_size, spec.latent_size
        per_head = keys * (nope + value) * es
        groups = min(heads, -(-heads * per_head // EXPANDED_BYTES))
        group = -(-heads // groups)
        columns = shape.num_unit_slots * UNIT_QUERIES * group
        sizes = (keys * nope * es * group, keys * value * es * group, keys * spec.rope_size * es, columns * value * 4,
                 columns * 8)
        workspace = torch.empty(sum(sizes), dtype=torch.uint8, device=rows.device)
        at = [workspace.data_ptr() + sum(sizes[:i]) for i in range(5)]
        for h in range(0, heads, group):
            n = min(group, heads - h)
            native.check(lib.lvamd_latent_expand(
                rows.data_ptr(), lists.blocks, shape.num_blocks, plan.tables_ptr,
                weights.key_up.data_ptr() + h * nope * latent * es, weights.value_up.data_ptr() + h * value * latent * es,
                at[0], at[1], at[2], n, latent, spec.rope_size, nope, value, plan.block_size, code, stream),
                "lvamd_latent_expand")
            native.check(lib.lvamd_latent_prefill(
                query.data_ptr() + h * query.stride(1) * es, query.stride(0), query.stride(1),
                query_rope.data_ptr() + h * query_rope.stride(1) * es, query_rope.stride(0), query_rope.stride(1),
                at[0], at[1], at[2], keys, out.data_ptr() + h * out.stride(1) * es, out.stride(0), out.stride(1),
                lists.units, shape.num_units, lists.unit_jobs, shape.num_unit_jobs, shape.unit_merge_columns,
                at[3] if columns else None, at[4] if columns else None, shape.num_unit_slots, n, nope, spec.rope_size, value,
                float(scale), code, stream), "lvamd_latent_prefill")
