"""Rotary angles of a step's positions, scaled for long contexts.

Pair i of a position p turns by p * frequency_i, frequency_i = base^(-2i / size).
light-vllm's Qwen2 forms its angles per model step in fp32
(``_rotary_embeddings``, src/light_vllm/modeling/models/qwen2.py), unscaled; here
the products are formed and reduced in fp64, by one launch per step whose rows
every layer uses: ``full=True`` gives the rows of the ``rotary=`` argument over a
``PagedKVCache``, the default those over a ``LatentPagedKVCache``.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor

from light_vllm_amd import errors, native
from light_vllm_amd.paged_cache import dtype_code
from light_vllm_amd.plan import current_stream
from light_vllm_amd.quantized_cache import _NOT_FAST, _raw_stream, on_device

_KINDS = ("linear", "base", "ramp", "smooth")


@dataclass(frozen=True, slots=True)
class RotaryScaling:
    """How the angles of a model trained on ``original_length`` positions are
    scaled for contexts ``factor`` times as long.

    * ``linear``: every frequency divided by ``factor`` (position interpolation);
    * ``base``: the base times factor^(size / (size - 2)) (the fastest pair keeps
      its frequency, the slowest is divided by ``factor``);
    * ``ramp``: by pair index: pairs that turn at least ``fast`` times over the
      original context keep their frequency, those that turn at most ``slow``
      times are divided by ``factor``, linearly blended in the index between
      (rounded outwards); cosines and sines are multiplied by ``magnitude``, by
      default 0.1 ln(factor) + 1 (YaRN, Peng et al. 2023);
    * ``smooth``: the same blend, linear in the number of turns between ``slow``
      and ``fast``, by default 1 and 4.
    """

    kind: str
    factor: float
    original_length: int = 4096
    slow: float = 1.0
    fast: float | None = None  # ramp: 32, smooth: 4
    magnitude: float | None = None

    def __post_init__(self) -> None:
        if self.kind not in _KINDS:
            raise ValueError(f"rotary scaling must be one of {_KINDS}")
        if self.fast is None:
            object.__setattr__(self, "fast", 32.0 if self.kind == "ramp" else 4.0)
        for holds, message in (
            (_finite(self.factor) and self.factor > 0, "rotary scaling factor must be a positive number"),
            (type(self.original_length) is int and self.original_length > 0,
             "original_length must be a positive integer"),
            (_finite(self.slow) and _finite(self.fast) and 0 < self.slow < self.fast,
             "rotary scaling needs 0 < slow < fast"),
            (self.magnitude is None or _finite(self.magnitude), "rotary magnitude must be a number"),
        ):
            if not holds:
                raise ValueError(message)


def _finite(x) -> bool:
    return type(x) in (int, float) and math.isfinite(x)


def rotary_frequencies(size: int, base: float, scaling: RotaryScaling | None = None) -> tuple[Tensor, float]:
    """fp64 frequencies of a rotated part of ``size`` values (radians per
    position), and the magnitude of its cosines and sines."""

    if type(size) is not int or size <= 0 or size % 2:
        raise ValueError("rotary size must be a positive even integer")
    if not _finite(base) or base <= 1:
        raise ValueError("rotary base must be a number above 1")
    magnitude = 1.0
    index = torch.arange(size // 2, dtype=torch.float64)
    freq = float(base) ** (-2.0 * index / size)
    if scaling is None:
        return freq, magnitude
    f = float(scaling.factor)
    if scaling.magnitude is not None:
        magnitude = float(scaling.magnitude)
    if scaling.kind == "linear":
        return freq / f, magnitude
    if scaling.kind == "base":
        if size == 2:
            raise ValueError("rotary scaling through the base needs more than one pair")
        return (float(base) * f ** (size / (size - 2))) ** (-2.0 * index / size), magnitude
    if scaling.kind == "ramp":
        if scaling.magnitude is None and f > 1:
            magnitude = 0.1 * math.log(f) + 1.0

        def pair(turns: float) -> float:  # the index that turns so often
            return size * math.log(scaling.original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair(scaling.fast)), 0)
        high = min(math.ceil(pair(scaling.slow)), size - 1)
        slowed = ((index - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    else:
        turns = scaling.original_length * freq / (2 * math.pi)
        slowed = 1.0 - ((turns - scaling.slow) / (scaling.fast - scaling.slow)).clamp(0.0, 1.0)
    return freq * (1.0 - slowed) + freq / f * slowed, magnitude


class RotaryEmbedding:
    """Angles of positions for a rotated part of ``size`` values, on the GPU.

    Made once per model; called once per step with the tokens' positions (an int32
    or int64 vector on the embedding's device),
    it returns ``(cosines, sines)``: ``[tokens, size / 2]``, one value per pair,
    or with ``full=True`` ``[tokens, size]``, each half the same (what the half
    layout multiplies a whole row with)."""

    def __init__(self, size: int, *, base: float = 10000.0, scaling: RotaryScaling | None = None,
                 device: str | torch.device = "cuda") -> None:
        freq, self.magnitude = rotary_frequencies(size, base, scaling)
        self.size, self.base, self.scaling = size, float(base), scaling
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise errors.ExecutionError("rotary embeddings require a GPU (cuda) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._turns = (freq / (2 * math.pi)).to(self.device)
        self._lib = native.load()
        self._facts = (torch.int64, torch.int32, _raw_stream, self.device.index, native.entry("lvamd_rotary_angles"),
                       self._turns.data_ptr(), size // 2)
        self._angles = native.host().rotary_angles

    def __call__(self, positions: Tensor, *, full: bool = False, dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor]:
        # The common case in one native call: it reads the positions and launches
        # when every rule holds; anything else takes the rules below.
        n, half = positions.shape[0] if isinstance(positions, Tensor) and positions.ndim == 1 else 0, self.size // 2
        if 0 < n <= (2**31 - 1) // half and torch.cuda.current_device() == self.device.index:
            code = dtype_code(dtype)
            width = self.size if full else half
            cosines = torch.empty_strided((n, width), (width, 1), dtype=dtype, device=self.device)
            sines = torch.empty_strided((n, width), (width, 1), dtype=dtype, device=self.device)
            status = self._angles(self._facts, positions, n, cosines.data_ptr(), sines.data_ptr(), 2 if full else 1, code,
                                  self.magnitude)
            if status == 0:
                return cosines, sines
            if status != _NOT_FAST:
                native.check(status, "lvamd_rotary_angles")
        if not isinstance(positions, Tensor) or positions.ndim != 1 or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("rotary positions must be an int32 or int64 vector")
        if positions.device != self.device:
            raise ValueError("rotary positions must be on the embedding's device")
        code = dtype_code(dtype)
        n = positions.shape[0]
        if n > (2**31 - 1) // half:
            raise ValueError("too many rotary positions for one call")
        positions = positions.contiguous()
        with on_device(self.device):
            both = torch.empty((2, n, self.size if full else half), dtype=dtype, device=self.device)
            cosines, sines = both.unbind(0)
            native.check(self._lib.lvamd_rotary_angles(
                positions.data_ptr(), positions.element_size(), n, self._turns.data_ptr(), half, self.magnitude,
                cosines.data_ptr(), sines.data_ptr(), 2 if full else 1, code, current_stream(self.device)),
                "lvamd_rotary_angles")
        return cosines, sines
