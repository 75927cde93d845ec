"""Paged K/V pools in 8 bits on an MI355X: e4m3 codes with one power-of-two
scale per block and kv head.

``QuantizedPagedKVCache`` stands beside ``PagedKVCache`` with the same methods,
rules and messages, in about half the bytes of a 16-bit cache: the step's
tensors stay bf16 or fp16 (``config.dtype``), and ``HipPagedAttentionBackend``
attends it through the same ``create`` / ``forward``.  light-vllm has no
counterpart (its pools hold the model's dtype,
src/light_vllm/runtime/execution/paged_cache.py:328-338).

What a block holds: value = code * scale, scale = 2^e with e the smallest
exponent (at least -100) that brings the largest finite magnitude of the rows
within 448, e4m3's largest.  A block that is written at its offset 0 starts
anew; later rows can only raise its scale, and then the block's other rows are
re-scaled, which a power of two makes exact (unless a code becomes subnormal):
a token at a time gives the codes that a whole prompt gives.  Every row written
since offset 0 counts, a rejected draft's too: ``compact`` keeps the scale.
Non-finite values are stored as NaN and do not count for the scale.
"""

from __future__ import annotations

import functools
import weakref
from dataclasses import dataclass

import numpy as np
import torch
from torch import Tensor

from light_vllm_amd import errors, native
from light_vllm_amd.interfaces import AttentionLayerSpec, ModelKVCacheSpec
from light_vllm_amd.paged_cache import (
    PagedKVCacheConfig, PagedKVWriteMapping, _block_copy_pairs, _compact_bytes, _compact_request, _launch_block_copy,
    dtype_code,
)
from light_vllm_amd.plan import Staging, current_stream

CODE_DTYPE = torch.float8_e4m3fn
# Scale of a block that was never written.
LOWEST_SCALE = 2.0 ** -100
_HEAD_SIZES = range(32, 257, 16)
_NOT_FAST = 1 << 30  # append_tensors: a tensor rule of the fast path does not hold
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


@functools.lru_cache(maxsize=1)
def _append_tensors():
    return native.host().append_tensors


def quantized_kv_cache_bytes_per_block(model_spec: ModelKVCacheSpec, *, block_size: int) -> int:
    """Bytes of one physical block across all layers: K and V codes, and their scales."""

    return sum(2 * spec.num_kv_heads * (block_size * spec.head_size + 4) for spec in model_spec.layers)


@dataclass(frozen=True, slots=True)
class QuantizedPagedLayerCache:
    """One layer's codes ``[block, offset, kv_head, head_size]`` (e4m3) and
    scales ``[block, kv_head]`` (fp32, powers of two) of K and V."""

    keys: Tensor
    values: Tensor
    key_scales: Tensor
    value_scales: Tensor


@dataclass(frozen=True, slots=True)
class QuantizedKVWriteMapping(PagedKVWriteMapping):
    """Write slots of one step in which each block's slots are consecutive, for
    caches of this many blocks and block size
    (``QuantizedPagedKVCache.prepare_write``)."""

    geometry: tuple[int, int] = (0, 0)

    def __post_init__(self) -> None:
        # The launch reads them by address.
        slots, sources = self.slots, self.source_indices
        count = self.num_query_tokens if sources is None else sources.numel()
        if not (all(t.ndim == 1 and t.dtype == torch.long and t.is_contiguous() and t.device == slots.device
                    for t in (slots, sources) if t is not None)
                and slots.numel() == count <= self.num_query_tokens):
            raise errors.KVCacheError("slots and source indices of an 8-bit cache's mapping must be contiguous int64 "
                                      "vectors on one device, one entry per token written")


class _State:
    """Per-cache launch state: device tables of the layers' pool addresses by
    shape, of their scales' by kv heads, and a staging ring."""

    def __init__(self, cache: "QuantizedPagedKVCache") -> None:
        device = cache.config.device
        shapes: dict[tuple[int, int], list[tuple[int, int]]] = {}
        scales: dict[int, list[tuple[int, int]]] = {}
        for spec in cache.model_spec.layers:
            layer = cache.layer(spec.layer_id)
            shapes.setdefault((spec.num_kv_heads, spec.head_size), []).append(
                (layer.keys.data_ptr(), layer.values.data_ptr()))
            scales.setdefault(spec.num_kv_heads, []).append(
                (layer.key_scales.data_ptr(), layer.value_scales.data_ptr()))

        def table(ptrs):
            t = torch.tensor(ptrs, dtype=torch.int64).t().contiguous().to(device)
            return len(ptrs), t, t.data_ptr(), t.data_ptr() + 8 * len(ptrs)

        self.shapes = [(*shape, *table(ptrs)) for shape, ptrs in shapes.items()]
        bs = cache.config.block_size
        # (block bytes, layers, table, K and V addresses) of codes and scales.
        self.blocks = [(bs * heads * size, *rest) for heads, size, *rest in self.shapes]
        self.blocks += [(4 * heads, *table(ptrs)) for heads, ptrs in scales.items()]
        lib = native.load()
        self.small_copies = int(lib.lvamd_kv_block_copy_small_pairs())
        self.few_pairs = int(lib.lvamd_kv_compact_q8_few_pairs())
        self.call_pairs = int(lib.lvamd_kv_compact_q8_few_call_pairs())
        self.staging = Staging(device)


_STATES: "weakref.WeakKeyDictionary[QuantizedPagedKVCache, _State]" = weakref.WeakKeyDictionary()


class QuantizedPagedKVCache:
    """Per-layer 8-bit K/V pools shared by all requests, addressed by block id.

    ``config.dtype`` is that of the step's tensors, bfloat16 or float16."""

    quantized = True

    def __init__(self, model_spec: ModelKVCacheSpec, config: PagedKVCacheConfig) -> None:
        if config.device.type != "cuda":
            raise errors.KVCacheError("the HIP paged KV cache requires a GPU (cuda) device")
        if config.dtype not in (torch.bfloat16, torch.float16):
            raise errors.KVCacheError(f"the 8-bit KV cache takes bfloat16 or float16 tensors, not {config.dtype}")
        for spec in model_spec.layers:
            if spec.head_size not in _HEAD_SIZES:
                raise errors.KVCacheError(
                    f"the 8-bit KV cache supports head sizes {tuple(_HEAD_SIZES)}, not {spec.head_size} "
                    f"(layer {spec.layer_id!r})")
        if config.num_blocks * config.block_size > 2**31 - 1:
            raise errors.KVCacheError("the 8-bit KV cache holds at most 2**31 - 1 slots")
        self._model_spec = model_spec
        self._config = config
        self._layer_specs = {layer.layer_id: layer for layer in model_spec.layers}
        self._layers = {layer.layer_id: self._allocate_layer(layer) for layer in model_spec.layers}
        self._geometry = (config.num_blocks, config.block_size)
        # What append_tensors takes of a layer, made at its first write.
        self._append_facts: dict[str, tuple] = {}

    @property
    def config(self) -> PagedKVCacheConfig:
        return self._config

    @property
    def model_spec(self) -> ModelKVCacheSpec:
        return self._model_spec

    def layer_spec(self, layer_id: str) -> AttentionLayerSpec:
        try:
            return self._layer_specs[layer_id]
        except KeyError as exc:
            raise errors.KVCacheError(f"KV cache layer {layer_id!r} was not found") from exc

    def layer(self, layer_id: str) -> QuantizedPagedLayerCache:
        try:
            return self._layers[layer_id]
        except KeyError as exc:
            raise errors.KVCacheError(f"KV cache layer {layer_id!r} was not found") from exc

    def scale_offset(self, spec: AttentionLayerSpec) -> int:
        """Bytes from a pool's base to its scales, for layers of ``spec``'s shape."""

        return self._config.num_blocks * self._config.block_size * spec.num_kv_heads * spec.head_size

    @torch.inference_mode()
    def prepare_write(self, slot_mapping: Tensor, *, validate: bool = True) -> QuantizedKVWriteMapping:
        """One step's slot mapping for every layer's write, with
        ``PagedKVCache.prepare_write``'s rules.

        With ``validate`` the slots are checked from one host copy and put in
        order.  Without, the mapping stays on the device untouched: besides
        being in range and distinct, the slots that lie in one block must then
        be consecutive entries (as a step's ``slot_mapping`` has them)."""

        if slot_mapping.ndim != 1:
            raise errors.KVCacheError("slot mapping must have one entry per packed query token")
        if slot_mapping.device != self._config.device:
            raise errors.KVCacheError("slot mapping device must match the cache")
        num_tokens = slot_mapping.numel()
        if not validate:
            return QuantizedKVWriteMapping(slots=slot_mapping.to(torch.long).contiguous(), num_query_tokens=num_tokens,
                                           geometry=self._geometry)
        host = slot_mapping.to("cpu", torch.long).numpy()
        written = np.flatnonzero(host >= 0)
        written = written[np.argsort(host[written], kind="stable")]
        chosen = host[written]
        if chosen.size:
            if int(chosen[-1]) >= self._config.num_blocks * self._config.block_size:
                raise errors.KVCacheError("slot mapping contains an out-of-range physical slot")
            if np.any(chosen[1:] == chosen[:-1]):
                raise errors.KVCacheError("slot mapping must not write the same physical slot twice")
        device = self._config.device
        in_place = written.size == num_tokens and bool(np.all(written[1:] > written[:-1]))
        return QuantizedKVWriteMapping(
            slots=torch.from_numpy(chosen).to(device),
            num_query_tokens=num_tokens,
            source_indices=None if in_place else torch.from_numpy(written).to(device),
            geometry=self._geometry,
        )

    def write_prepared(self, layer_id: str, key: Tensor, value: Tensor, mapping: PagedKVWriteMapping) -> None:
        """Quantise one layer's K/V into the slots of a prepared mapping."""

        # The common case in one native call, as the backend's forward: it reads
        # the tensors itself and launches when every rule holds; anything else
        # takes the rules below.
        facts = self._append_facts.get(layer_id) or self._bind_append(layer_id)
        if (type(mapping) is QuantizedKVWriteMapping and mapping.geometry == self._geometry
                and mapping.slots.device == self._config.device and torch.cuda.current_device() == facts[2]):
            slots, sources = mapping.slots, mapping.source_indices
            status = _append_tensors()(facts, key, value, slots.data_ptr(), 0 if sources is None else sources.data_ptr(),
                                       slots.numel(), mapping.num_query_tokens)
            if status == 0:
                return
            if status != _NOT_FAST:
                native.check(status, "lvamd_kv_append_q8")
        layer = self.layer(layer_id)
        spec = self.layer_spec(layer_id)
        cfg = self._config
        tail = (spec.num_kv_heads, spec.head_size)
        rules = (
            (lambda: key.ndim == 3 and tuple(key.shape[1:]) == tail,
             "paged KV update must have shape [tokens, kv_heads, head_size]"),
            (lambda: value.shape == key.shape, "paged K/V updates must have the same shape"),
            (lambda: isinstance(mapping, QuantizedKVWriteMapping) and mapping.geometry == self._geometry,
             "an 8-bit KV cache takes a mapping of its own prepare_write"),
            (lambda: mapping.num_query_tokens == key.shape[0], "slot mapping must have one entry per query token"),
            (lambda: key.dtype == cfg.dtype and key.device == cfg.device,
             "paged KV update dtype and device must match the cache"),
            (lambda: value.dtype == key.dtype and value.device == key.device,
             "paged K/V updates must use the same dtype and device"),
            (lambda: mapping.slots.device == cfg.device
             and (mapping.source_indices is None or mapping.source_indices.device == cfg.device),
             "prepared slot mapping device must match the cache"),
        )
        for holds, message in rules:
            if not holds():
                raise errors.KVCacheError(message)
        slots, sources = mapping.slots, mapping.source_indices
        if slots.numel() == 0:
            return
        key, value = _aligned_rows(key), _aligned_rows(value)
        with on_device(cfg.device):
            native.check(native.load().lvamd_kv_append_q8(
                key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
                layer.keys.data_ptr(), layer.key_scales.data_ptr(), layer.values.data_ptr(),
                layer.value_scales.data_ptr(), slots.data_ptr(), sources.data_ptr() if sources is not None else None,
                slots.numel(), spec.num_kv_heads, spec.head_size, cfg.block_size, dtype_code(cfg.dtype),
                current_stream(cfg.device)), "lvamd_kv_append_q8")

    def _bind_append(self, layer_id: str) -> tuple:
        layer, spec, cfg = self.layer(layer_id), self.layer_spec(layer_id), self._config
        index = cfg.device.index if cfg.device.index is not None else torch.cuda.current_device()
        found = self._append_facts[layer_id] = (
            native.append_q8_entry(), cfg.dtype, index, cfg.dtype.itemsize, spec.num_kv_heads, spec.head_size,
            cfg.block_size, dtype_code(cfg.dtype), layer.keys.data_ptr(), layer.key_scales.data_ptr(),
            layer.values.data_ptr(), layer.value_scales.data_ptr(), _raw_stream,
        )
        return found

    def write(self, layer_id: str, key: Tensor, value: Tensor, slot_mapping: Tensor) -> None:
        """Quantise the active tokens' K/V into their physical slots."""

        self.write_prepared(layer_id, key, value, self.prepare_write(slot_mapping))

    def compact(
        self,
        block_ids: tuple[int, ...],
        *,
        num_computed_tokens: int,
        num_query_tokens: int,
        num_reserved_query_tokens: int,
        retained_query_indices: tuple[int, ...],
        num_readonly_prefix_blocks: int = 0,
    ) -> int:
        """Move the accepted path to the contiguous formal tail of every layer;
        returns how many tokens moved (``PagedKVCache.compact``)."""

        return self.compact_many((_compact_request(
            block_ids, num_computed_tokens=num_computed_tokens, num_query_tokens=num_query_tokens,
            num_reserved_query_tokens=num_reserved_query_tokens, retained_query_indices=retained_query_indices,
            num_readonly_prefix_blocks=num_readonly_prefix_blocks),))[0]

    def compact_many(self, requests) -> tuple[int, ...]:
        """``compact`` for every request of a step together.  Moved rows keep
        their values; a block that takes one from a block of a larger scale takes
        that scale (its other rows are re-scaled), so no two requests may move
        rows into one block."""

        if not isinstance(requests, (list, tuple)):
            requests = tuple(requests)
        cfg = self._config
        moved, src, dst = _compact_bytes(cfg, requests)
        if src:
            src, dst, counts = bytes(src), bytes(dst), bytes(moved)
            twice, starts = native.host().block_runs(counts, dst, cfg.block_size)
            if twice:
                raise errors.KVCacheError("compact requests of one step must not write the same block of an 8-bit cache")
            with on_device(cfg.device):
                self._launch_compact(counts, src, dst, starts)
        return tuple(np.frombuffer(moved, dtype=np.int64).tolist())

    def _launch_compact(self, counts: bytes, src: bytes, dst: bytes, starts: bytes) -> None:
        state = self._state()
        cfg = self._config
        n, groups = len(src) // 8, len(starts) // 8 - 1
        lib = native.load()
        slots = cfg.num_blocks * cfg.block_size
        stream = current_stream(cfg.device)
        # A step's accepted drafts ride in the kernel arguments: a few as one chunk
        # (int32 starts 0 and n), more in chunks that do not touch each other.
        if n <= state.few_pairs:
            chunks = (n << 32).to_bytes(8, "little")
        elif n <= state.call_pairs:
            chunks = native.host().compact_chunks(counts, src, dst, cfg.block_size, state.few_pairs)
        else:
            chunks = None
        if chunks is not None:
            for heads, size, layers, _, kptrs, vptrs in state.shapes:
                native.check(lib.lvamd_kv_compact_q8_few(kptrs, vptrs, layers, heads, size, cfg.block_size,
                                                         slots * heads * size, src, dst, n, chunks, len(chunks) // 4 - 1,
                                                         stream), "lvamd_kv_compact_q8_few")
            return
        buf = state.staging.buffer((len(src) + len(dst) + len(starts)) // 4)
        buf[:] = np.frombuffer(src + dst + starts, dtype=np.int32)
        blob = state.staging.upload(buf)
        at = blob.data_ptr()
        for heads, size, layers, _, kptrs, vptrs in state.shapes:
            # (Of the call's own stream: two streams' compacts do not share one.)
            nbytes = lib.lvamd_kv_compact_q8_workspace_size(n, layers, heads, size)
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=cfg.device)
            native.check(lib.lvamd_kv_compact_q8(
                kptrs, vptrs, layers, heads, size, cfg.block_size, slots * heads * size, at, at + 8 * n, n,
                at + 16 * n, groups, workspace.data_ptr(), nbytes, stream), "lvamd_kv_compact_q8")

    def copy_blocks(self, src_blocks, dst_blocks) -> None:
        """Copy-on-write of whole blocks, codes and scales, across every layer."""

        src, dst = _block_copy_pairs(self, src_blocks, dst_blocks)
        if src:
            state = self._state()
            with on_device(self._config.device):
                _launch_block_copy(self._config.device, src, dst, state.staging, state.small_copies, state.blocks)

    def _state(self) -> _State:
        found = _STATES.get(self)
        if found is None:
            found = _STATES[self] = _State(self)
        return found

    def _allocate_layer(self, spec: AttentionLayerSpec) -> QuantizedPagedLayerCache:
        cfg = self._config
        shape = (cfg.num_blocks, cfg.block_size, spec.num_kv_heads, spec.head_size)
        codes = self.scale_offset(spec)
        sides = []
        for _ in range(2):
            # One allocation per pool, the scales behind the codes: a layer's
            # launch then takes one address per pool.
            pool = torch.zeros(codes + 4 * cfg.num_blocks * spec.num_kv_heads, dtype=torch.uint8, device=cfg.device)
            scales = pool[codes:].view(torch.float32).view(cfg.num_blocks, spec.num_kv_heads)
            sides.append((pool[:codes].view(CODE_DTYPE).view(shape), scales.fill_(LOWEST_SCALE)))
        (keys, key_scales), (values, value_scales) = sides
        return QuantizedPagedLayerCache(keys, values, key_scales, value_scales)


def _aligned_rows(t: Tensor) -> Tensor:
    """``t``, or a copy whose rows are 16-byte chunks."""

    def fits(x: Tensor) -> bool:
        return x.stride(2) == 1 and x.data_ptr() % 16 == 0 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0

    # (contiguous() leaves the strides of single tokens and heads as they are.)
    return t if fits(t) else t.clone(memory_format=torch.contiguous_format)


class on_device:
    """Makes ``device`` the current one where it is not (a launch goes to the
    current device)."""

    __slots__ = ("_guard",)

    def __init__(self, device: torch.device) -> None:
        index = device.index
        self._guard = None
        if index is not None and index != torch.cuda.current_device():
            self._guard = torch.cuda.device(index)

    def __enter__(self) -> None:
        if self._guard is not None:
            self._guard.__enter__()

    def __exit__(self, *exc) -> None:
        if self._guard is not None:
            self._guard.__exit__(*exc)
