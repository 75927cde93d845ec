"""The 8-bit paged cache and the verification of drafts, restated in numpy fp64
from their definitions (no code shared with the kernels or the package).

Cache: value = code * scale per (block, kv head), code an e4m3 value, scale = 2^e
with e the smallest exponent, at least -100, with amax <= 448 * 2^e.
"""

from __future__ import annotations

import numpy as np

LOWEST = -100


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """The nearest e4m3 value (ties to even) of |x| <= 448; NaN stays."""

    size = np.abs(x)
    with np.errstate(divide="ignore", invalid="ignore"):
        exponent = np.maximum(np.floor(np.log2(np.where(size > 0, size, 1.0))), -6.0)
        step = np.exp2(exponent - 3.0)
        return np.where(np.isnan(x), np.nan, np.round(x / step) * step)


def scale_of(amax: np.ndarray) -> np.ndarray:
    amax = np.asarray(amax, dtype=np.float64)
    e = np.full(amax.shape, LOWEST)
    while np.any(amax > 448.0 * np.exp2(e)):
        e = np.where(amax > 448.0 * np.exp2(e), e + 1, e)
    return np.exp2(e.astype(np.float64))


def stored(rows: np.ndarray, scale: np.ndarray, largest: float) -> np.ndarray:
    """Codes of rows [..., heads, D] at scales [heads]."""

    clipped = np.where(np.isfinite(rows), np.clip(rows, -largest, largest), np.nan)
    return round_e4m3(clipped / scale[..., None])


def append(codes: np.ndarray, scales: np.ndarray, rows: np.ndarray, slots, largest: float) -> None:
    """codes [blocks, bs, heads, D] and scales [blocks, heads] (fp64, in place) take rows [n, heads, D] at slots."""

    bs = codes.shape[1]
    by_block: dict[int, list[int]] = {}
    for i, s in enumerate(slots):
        if s >= 0:
            by_block.setdefault(int(s) // bs, []).append(i)
    for block, members in by_block.items():
        new = rows[members].astype(np.float64)
        wanted = scale_of(np.where(np.isfinite(new), np.abs(new), 0.0).max(axis=(0, 2)))
        if any(int(slots[i]) % bs == 0 for i in members):
            scales[block] = wanted
        else:
            grown = np.maximum(scales[block], wanted)
            codes[block] = round_e4m3(codes[block] * (scales[block] / grown)[None, :, None])
            scales[block] = grown
        for i, row in zip(members, new):
            codes[block, int(slots[i]) % bs] = stored(row, scales[block], largest)


def compact(codes: np.ndarray, scales: np.ndarray, src, dst) -> None:
    """Rows move with their values; sources are read before any write."""

    bs = codes.shape[1]
    before, old = codes.copy(), scales.copy()
    for s, d in zip(src, dst):
        scales[d // bs] = np.maximum(scales[d // bs], old[s // bs])
    for block in {int(d) // bs for d in dst}:
        codes[block] = round_e4m3(before[block] * (old[block] / scales[block])[None, :, None])
    for s, d in zip(src, dst):
        codes[d // bs, d % bs] = round_e4m3(before[s // bs, s % bs] * (old[s // bs] / scales[d // bs])[:, None])


def verify(parents, tokens, target, node_uniforms, sample_uniform, draft_probs=None):
    """One request: parents and tokens of its drafts, target rows [1 + n, V], one
    uniform per row; (accepted drafts, token)."""

    def mass(p):
        p = np.asarray(p, dtype=np.float64)
        return np.where(np.isfinite(p) & (p > 0), p, 0.0)

    node, path = 0, []
    while True:
        p, u = mass(target[node]), float(node_uniforms[node])
        kids = [j for j, parent in enumerate(parents) if parent + 1 == node]
        taken, below = None, 0.0
        for j in kids:
            if draft_probs is not None:
                if u * float(mass(draft_probs[j])[tokens[j]]) < p[tokens[j]]:
                    taken = j
                break
            if below <= u < below + p[tokens[j]]:
                taken = j
                break
            below += p[tokens[j]]
        if taken is None:
            break
        path.append(taken)
        node = taken + 1
    rest = p.copy()
    if draft_probs is not None and kids:
        rest = np.maximum(p - mass(draft_probs[kids[0]]), 0.0)
    elif kids:
        rest[[tokens[j] for j in kids]] = 0.0
    if not rest.any():
        rest = p
    if not rest.any():
        return path, -1
    cdf = np.cumsum(rest)
    hits = np.flatnonzero((cdf > float(sample_uniform) * cdf[-1]) & (rest > 0))
    return path, int(hits[0]) if hits.size else int(np.flatnonzero(rest)[-1])
