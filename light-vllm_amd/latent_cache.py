"""Paged pools of shared latent vectors on an MI355X.

``LatentPagedKVCache`` stands beside ``PagedKVCache`` for layers whose heads
share one latent vector a token: a row per token, ``[latent | rotated key]``, in
place of per-head keys and values.  It has the other caches' methods, rules and
messages, and ``HipPagedAttentionBackend`` attends it through the same
``create`` / ``forward`` (``latent_attention``).  light-vllm has no counterpart
(its layers cache per-head K and V,
src/light_vllm/modeling/attention/interfaces.py:9-36).
"""

from __future__ import annotations

import functools
import weakref
from dataclasses import dataclass

import numpy as np
import torch
from torch import Tensor

from light_vllm_amd import errors, native
from light_vllm_amd.interfaces import _is_int, _raise_first
from light_vllm_amd.paged_cache import (
    PagedKVCacheConfig, PagedKVWriteMapping, _block_copy_pairs, _compact_bytes, _compact_request, dtype_code,
)
from light_vllm_amd.plan import Staging, current_stream
from light_vllm_amd.quantized_cache import _NOT_FAST, _raw_stream, on_device

LATENT_SIZES = (128, 256, 384, 512)
ROPE_SIZES = (32, 64)
ROTARY_LAYOUTS = ("interleaved", "half")


@dataclass(frozen=True, slots=True)
class LatentLayerSpec:
    """Cache shape of one attention layer over latent vectors.

    ``rotary_layout`` says which values of a rotated part are a pair:
    ``"interleaved"`` (2i, 2i + 1) or ``"half"`` (i, i + rope_size / 2)."""

    layer_id: str
    num_query_heads: int
    latent_size: int
    rope_size: int
    rotary_layout: str = "interleaved"

    def __post_init__(self) -> None:
        _raise_first((
            (lambda: bool(self.layer_id), "layer_id must not be empty"),
            (lambda: _is_int(self.num_query_heads) and self.num_query_heads > 0,
             "num_query_heads must be a positive integer"),
            (lambda: _is_int(self.latent_size) and self.latent_size in LATENT_SIZES,
             f"latent_size must be one of {LATENT_SIZES}"),
            (lambda: _is_int(self.rope_size) and self.rope_size in ROPE_SIZES, f"rope_size must be one of {ROPE_SIZES}"),
            (lambda: self.rotary_layout in ROTARY_LAYOUTS, f"rotary_layout must be one of {ROTARY_LAYOUTS}"),
        ))

    @property
    def row_size(self) -> int:
        """Values of one token's row."""

        return self.latent_size + self.rope_size


@dataclass(frozen=True, slots=True)
class LatentKVCacheSpec:
    """Cache shapes of every latent attention layer of a model."""

    layers: tuple[LatentLayerSpec, ...]

    def __post_init__(self) -> None:
        layers = tuple(self.layers)
        ids = [layer.layer_id for layer in layers]
        _raise_first((
            (lambda: len(layers) > 0, "model KV cache spec must contain at least one layer"),
            (lambda: len(set(ids)) == len(ids), "attention layer IDs must be unique"),
        ))
        object.__setattr__(self, "layers", layers)


def latent_kv_cache_bytes_per_block(model_spec: LatentKVCacheSpec, *, block_size: int, dtype: torch.dtype) -> int:
    """Bytes of one physical block across all layers."""

    return sum(spec.row_size for spec in model_spec.layers) * block_size * dtype.itemsize


@dataclass(frozen=True, slots=True)
class LatentPagedLayerCache:
    """One layer's rows ``[block, offset, latent_size + rope_size]``; ``latents``
    and ``rope_keys`` are views of them."""

    rows: Tensor
    latents: Tensor
    rope_keys: Tensor


@functools.lru_cache(maxsize=1)
def _latent_write():
    return native.host().latent_write


class _State:
    """Per-cache launch state: device tables of the layers' pool addresses by row
    size, and a staging ring."""

    def __init__(self, cache: "LatentPagedKVCache") -> None:
        device = cache.config.device
        shapes: dict[int, list[int]] = {}
        for spec in cache.model_spec.layers:
            rows = cache.layer(spec.layer_id).rows
            shapes.setdefault(spec.row_size * rows.element_size(), []).append(rows.data_ptr())
        self.groups = []  # (row bytes, layers, device table)
        for row_bytes, ptrs in shapes.items():
            self.groups.append((row_bytes, len(ptrs), torch.tensor(ptrs, dtype=torch.int64).to(device)))
        self.few = int(native.load().lvamd_latent_move_few_pairs())
        self.staging = Staging(device)


_STATES: "weakref.WeakKeyDictionary[LatentPagedKVCache, _State]" = weakref.WeakKeyDictionary()


class LatentPagedKVCache:
    """Per-layer latent pools shared by all requests, addressed by block id."""

    latent = True

    def __init__(self, model_spec: LatentKVCacheSpec, config: PagedKVCacheConfig) -> None:
        if config.device.type != "cuda":
            raise errors.KVCacheError("the HIP paged KV cache requires a GPU (cuda) device")
        if config.dtype not in (torch.bfloat16, torch.float16):
            raise errors.KVCacheError(f"the latent KV cache takes bfloat16 or float16 tensors, not {config.dtype}")
        if config.num_blocks * config.block_size > 2**31 - 1:
            raise errors.KVCacheError("the latent KV cache holds at most 2**31 - 1 slots")
        if not isinstance(model_spec, LatentKVCacheSpec):
            raise errors.KVCacheError("the latent KV cache takes a LatentKVCacheSpec")
        self._model_spec = model_spec
        self._config = config
        self._layer_specs = {layer.layer_id: layer for layer in model_spec.layers}
        self._layers = {layer.layer_id: self._allocate_layer(layer) for layer in model_spec.layers}
        self._pool_ptrs = {layer_id: layer.rows.data_ptr() for layer_id, layer in self._layers.items()}
        # What latent_write takes of a layer, made at its first write.
        self._write_facts: dict[str, tuple] = {}
        self._slots = config.num_blocks * config.block_size

    @property
    def config(self) -> PagedKVCacheConfig:
        return self._config

    @property
    def model_spec(self) -> LatentKVCacheSpec:
        return self._model_spec

    def layer_spec(self, layer_id: str) -> LatentLayerSpec:
        try:
            return self._layer_specs[layer_id]
        except KeyError as exc:
            raise errors.KVCacheError(f"KV cache layer {layer_id!r} was not found") from exc

    def layer(self, layer_id: str) -> LatentPagedLayerCache:
        try:
            return self._layers[layer_id]
        except KeyError as exc:
            raise errors.KVCacheError(f"KV cache layer {layer_id!r} was not found") from exc

    def pool_ptr(self, layer_id: str) -> int:
        """Address of a layer's rows."""

        return self._pool_ptrs[layer_id]

    @torch.inference_mode()
    def prepare_write(self, slot_mapping: Tensor, *, validate: bool = True) -> PagedKVWriteMapping:
        """One step's slot mapping for every layer's write, with
        ``PagedKVCache.prepare_write``'s rules (without ``validate`` the slots stay
        on the device; those out of range are then not written)."""

        if slot_mapping.ndim != 1:
            raise errors.KVCacheError("slot mapping must have one entry per packed query token")
        if slot_mapping.device != self._config.device:
            raise errors.KVCacheError("slot mapping device must match the cache")
        num_tokens = slot_mapping.numel()
        if not validate:
            return PagedKVWriteMapping(slots=slot_mapping.to(torch.long).contiguous(), num_query_tokens=num_tokens)
        host = slot_mapping.to("cpu", torch.long).numpy()
        written = np.flatnonzero(host >= 0)
        chosen = host[written]
        if chosen.size:
            if int(chosen.max()) >= self._config.num_blocks * self._config.block_size:
                raise errors.KVCacheError("slot mapping contains an out-of-range physical slot")
            if np.unique(chosen).size != chosen.size:
                raise errors.KVCacheError("slot mapping must not write the same physical slot twice")
        device = self._config.device
        every = written.size == num_tokens
        return PagedKVWriteMapping(
            slots=torch.from_numpy(chosen).to(device),
            num_query_tokens=num_tokens,
            source_indices=None if every else torch.from_numpy(written).to(device),
        )

    def write_prepared(self, layer_id: str, latent: Tensor, rope_key: Tensor, mapping: PagedKVWriteMapping, *,
                       rotary: tuple[Tensor, Tensor] | None = None) -> None:
        """Write one layer's rows through a prepared mapping: ``latent``
        ``[tokens, latent_size]`` and ``rope_key`` ``[tokens, rope_size]``, turned by
        ``rotary=(cosines, sines)`` (fp32 ``[tokens, rope_size / 2]``) or as it is."""

        # The common case in one native call: it reads the tensors itself and launches
        # when every rule holds; anything else takes the rules below.
        cfg = self._config
        facts = self._write_facts.get(layer_id) or self._bind_write(layer_id)
        if (type(mapping) is PagedKVWriteMapping and torch.cuda.current_device() == facts[4]
                and (rotary is None or (type(rotary) is tuple and len(rotary) == 2 and rotary[0] is not None))):
            sources, tokens = mapping.source_indices, mapping.num_query_tokens
            cosines, sines = rotary if rotary is not None else (None, None)
            status = _latent_write()(facts, latent, rope_key, cosines, sines, mapping.slots, sources,
                                     tokens if sources is None else sources.numel(), tokens)
            if status == 0:
                return
            if status != _NOT_FAST:
                native.check(status, "lvamd_latent_append")
        spec = self.layer_spec(layer_id)
        check_rows(cfg, spec, latent, rope_key)
        slots, sources = mapping.slots, mapping.source_indices
        count = mapping.num_query_tokens if sources is None else sources.numel()
        for holds, message in (
            (lambda: mapping.num_query_tokens == latent.shape[0], "slot mapping must have one entry per query token"),
            (lambda: slots.device == cfg.device and (sources is None or sources.device == cfg.device),
             "prepared slot mapping device must match the cache"),
            (lambda: all(t.ndim == 1 and t.dtype == torch.long and t.is_contiguous()
                         for t in (slots, sources) if t is not None) and slots.numel() == count,
             "slots and source indices must be contiguous int64 vectors, one entry per token written"),
        ):
            if not holds():
                raise errors.KVCacheError(message)
        angles = check_rotary(spec, rotary, latent)
        append_rows(self, spec, latent, rope_key, angles, slots.data_ptr(), None if sources is None else sources.data_ptr(),
                    slots.numel())

    def _bind_write(self, layer_id: str) -> tuple:
        spec, cfg = self.layer_spec(layer_id), self._config
        index = cfg.device.index if cfg.device.index is not None else torch.cuda.current_device()
        found = self._write_facts[layer_id] = (
            torch.long, cfg.dtype, torch.float32, _raw_stream, index, native.entry("lvamd_latent_append"),
            self.layer(layer_id).rows.data_ptr(), self._slots, spec.latent_size, spec.rope_size, dtype_code(cfg.dtype),
            int(spec.rotary_layout == "interleaved"))
        return found

    def write(self, layer_id: str, latent: Tensor, rope_key: Tensor, slot_mapping: Tensor, *,
              rotary: tuple[Tensor, Tensor] | None = None) -> None:
        """Write the active tokens' rows to their physical slots."""

        self.write_prepared(layer_id, latent, rope_key, self.prepare_write(slot_mapping), rotary=rotary)

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
        """``compact`` for every request of a step together (one dict of
        ``compact``'s arguments, with ``block_ids``, per request)."""

        if not isinstance(requests, (list, tuple)):
            requests = tuple(requests)
        moved, src, dst = _compact_bytes(self._config, requests)
        if src:
            self._move(np.frombuffer(bytes(src), dtype=np.int64), np.frombuffer(bytes(dst), dtype=np.int64), rows=1,
                       apart=False)
        return tuple(np.frombuffer(moved, dtype=np.int64).tolist())

    def copy_blocks(self, src_blocks, dst_blocks) -> None:
        """Copy-on-write of whole blocks across every layer."""

        src, dst = _block_copy_pairs(self, src_blocks, dst_blocks)
        if src:
            self._move(np.asarray(src, dtype=np.int64), np.asarray(dst, dtype=np.int64), rows=self._config.block_size,
                       apart=True)

    def _move(self, src: np.ndarray, dst: np.ndarray, *, rows: int, apart: bool) -> None:
        """Runs of ``rows`` rows from places to places; ``apart``: no source is a
        destination."""

        state = _STATES.get(self)
        if state is None:
            state = _STATES[self] = _State(self)
        lib, n, device = native.load(), int(src.size), self._config.device
        with on_device(device):
            stream = current_stream(device)
            if n <= state.few:
                # A step's few pairs ride in the kernel arguments.
                for row_bytes, layers, table in state.groups:
                    native.check(lib.lvamd_latent_move_few(table.data_ptr(), layers, row_bytes * rows, src.ctypes.data,
                                                           dst.ctypes.data, n, stream), "lvamd_latent_move_few")
                return
            # (A replay would copy the places from a staging buffer that later calls reuse.)
            if torch.cuda.is_current_stream_capturing():
                raise errors.ExecutionError(f"a graph captures at most {state.few} moved tokens or copied blocks a call")
            blob, (at_src, at_dst) = state.staging.stage([src.view(np.int32), dst.view(np.int32)])
            at = blob.data_ptr()
            for row_bytes, layers, table in state.groups:
                workspace, nbytes = None, 0
                if not apart:
                    # (Of the call's own stream: two streams' compacts do not share one.)
                    nbytes = lib.lvamd_latent_move_workspace_size(n, layers, row_bytes * rows)
                    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
                native.check(lib.lvamd_latent_move(
                    table.data_ptr(), layers, row_bytes * rows, at + 4 * at_src, at + 4 * at_dst, n,
                    None if workspace is None else workspace.data_ptr(), nbytes, stream), "lvamd_latent_move")

    def _allocate_layer(self, spec: LatentLayerSpec) -> LatentPagedLayerCache:
        cfg = self._config
        # (Zeros: a request's last block is read to its end nowhere, but a model
        # that dumps its cache should not find another's data.)
        rows = torch.zeros((cfg.num_blocks, cfg.block_size, spec.row_size), dtype=cfg.dtype, device=cfg.device)
        return LatentPagedLayerCache(rows, rows[..., :spec.latent_size], rows[..., spec.latent_size:])


def is_latent(cache) -> bool:
    """Whether ``cache`` holds rows of latent vectors (``LatentPagedKVCache``)."""

    return getattr(cache, "latent", False) is True


def aligned_rows(t: Tensor) -> Tensor:
    """``t`` (two or three dimensions), or a copy whose rows are 16-byte chunks."""

    fits = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1])
    # (contiguous() leaves the strides of single tokens and heads as they are.)
    return t if fits else t.clone(memory_format=torch.contiguous_format)


def check_rows(cfg: PagedKVCacheConfig, spec: LatentLayerSpec, latent: Tensor, rope_key: Tensor) -> None:
    for holds, message in (
        (lambda: latent.ndim == 2 and latent.shape[1] == spec.latent_size,
         "latents must have shape [tokens, latent_size]"),
        (lambda: tuple(rope_key.shape) == (latent.shape[0], spec.rope_size),
         "rotated keys must have shape [tokens, rope_size]"),
        (lambda: all(t.dtype == cfg.dtype and t.device == cfg.device for t in (latent, rope_key)),
         "paged KV update dtype and device must match the cache"),
    ):
        if not holds():
            raise errors.KVCacheError(message)


def check_rotary(spec: LatentLayerSpec, rotary, like: Tensor) -> tuple[Tensor, Tensor] | None:
    """``rotary`` as two fp32 tensors of one row stride, or None."""

    if rotary is None:
        return None
    if not isinstance(rotary, (tuple, list)) or len(rotary) != 2:
        raise errors.KVCacheError("rotary must be a pair (cosines, sines)")
    shape = (like.shape[0], spec.rope_size // 2)
    for name, t in zip(("cosines", "sines"), rotary):
        if not isinstance(t, Tensor) or tuple(t.shape) != shape:
            raise errors.KVCacheError(f"rotary {name} must have shape [{shape[0]}, {shape[1]}]")
        if t.dtype != torch.float32 or t.device != like.device:
            raise errors.KVCacheError(f"rotary {name} must be float32 on the cache's device")
    cosines, sines = rotary
    if not (cosines.stride(0) == sines.stride(0) and all(
            t.stride(1) == 1 and t.stride(0) % 4 == 0 and t.data_ptr() % 16 == 0 for t in rotary)):
        cosines, sines = (t.clone(memory_format=torch.contiguous_format) for t in rotary)
    return cosines, sines


def append_rows(cache: LatentPagedKVCache, spec: LatentLayerSpec, latent: Tensor, rope_key: Tensor, angles, slots: int,
                sources: int | None, entries: int, query_rope: Tensor | None = None) -> Tensor | None:
    """The append's launch; with ``query_rope`` (aligned rows) the turned queries."""

    cfg = cache.config
    latent, rope_key = aligned_rows(latent), aligned_rows(rope_key)
    tokens = latent.shape[0]
    cosines, sines = angles if angles is not None else (None, None)
    with on_device(cfg.device):
        turned = None
        if query_rope is not None:
            turned = torch.empty((tokens, spec.num_query_heads, spec.rope_size), dtype=cfg.dtype, device=cfg.device)
        native.check(native.load().lvamd_latent_append(
            latent.data_ptr(), latent.stride(0), rope_key.data_ptr(), rope_key.stride(0),
            cache.layer(spec.layer_id).rows.data_ptr(), cfg.num_blocks * cfg.block_size, slots, sources, entries,
            None if cosines is None else cosines.data_ptr(), None if sines is None else sines.data_ptr(),
            0 if cosines is None else cosines.stride(0), int(spec.rotary_layout == "interleaved"),
            None if query_rope is None else query_rope.data_ptr(),
            0 if query_rope is None else query_rope.stride(0), 0 if query_rope is None else query_rope.stride(1),
            None if turned is None else turned.data_ptr(), tokens, spec.num_query_heads, spec.latent_size, spec.rope_size,
            dtype_code(cfg.dtype), current_stream(cfg.device)), "lvamd_latent_append")
    return turned
