"""Attention over a cache of shared latent vectors in fp64, from its definition:
head h's key of a row (c, r) is [key_up[h] c, r], its value value_up[h] c.
Without the weights the queries are the cache rows' own: key (c, r), value c."""

from __future__ import annotations

import numpy as np


def rotate(x, cosines, sines, interleaved: bool):
    """``x`` [tokens, ..., size] with its pairs turned by the tokens' angles."""

    x = np.asarray(x, dtype=np.float64)
    half = x.shape[-1] // 2
    shape = (x.shape[0],) + (1,) * (x.ndim - 2) + (half,)
    c, s = np.reshape(cosines, shape).astype(np.float64), np.reshape(sines, shape).astype(np.float64)
    out = np.empty_like(x)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        out[..., 0::2], out[..., 1::2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:]
        out[..., :half], out[..., half:] = a * c - b * s, b * c + a * s
    return out


def visible(parents, computed: int):
    """[queries, computed + queries]: what each query of one request sees."""

    n = len(parents)
    seen = np.zeros((n, computed + n), dtype=bool)
    seen[:, :computed] = True
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i, computed:] |= seen[p, computed:]
        seen[i, computed + i] = True
    return seen


def attention(query, rows, tables, computed, parents, block_size: int, latent: int, *, scale: float, key_up=None,
              value_up=None, per_key_error=None):
    """``query`` [tokens, heads, nope or latent + rope], ``rows`` [slots, latent + rope].
    Returns (out, attention of |value|, the largest score error): the last for
    per_key_error(|query row| of a head, |keys|) -> error of every score, before
    ``scale``; fp64, [tokens, heads, ...]."""

    query, rows = np.asarray(query, dtype=np.float64), np.asarray(rows, dtype=np.float64)
    rope = rows.shape[1] - latent
    heads = query.shape[1]
    outs, sizes, shifts, t0 = [], [], [], 0
    for table, c, par in zip(tables, computed, parents):
        n = len(par)
        at = np.arange(c + n)
        keys = rows[np.asarray(table, dtype=np.int64)[at // block_size] * block_size + at % block_size]
        seen = visible(par, c)
        for h in range(heads):
            q = query[t0:t0 + n, h]
            k, v = keys, keys[:, :latent]
            if key_up is not None:
                k = np.concatenate((v @ np.asarray(key_up[h], dtype=np.float64).T, keys[:, latent:]), axis=1)
                v = v @ np.asarray(value_up[h], dtype=np.float64).T
            with np.errstate(invalid="ignore", over="ignore"):
                s = np.where(seen, q @ k.T * scale, -np.inf)
                w = np.exp(s - s.max(axis=1, keepdims=True))
                total = w.sum(axis=1, keepdims=True)
                out, size = np.zeros((n, v.shape[1])), np.zeros((n, v.shape[1]))
                for i in range(n):  # (only what the query sees: 0 x NaN is none of its business)
                    out[i] = w[i, seen[i]] @ v[seen[i]] / total[i]
                    size[i] = w[i, seen[i]] @ np.abs(v[seen[i]]) / total[i]
                if per_key_error is not None:
                    shifts.append(np.where(seen, per_key_error(np.abs(q), np.abs(k)) * abs(scale), 0).max(axis=1))
            outs.append(out)
            sizes.append(size)
        t0 += n
    def stack(parts):
        at, rows_out = 0, []
        for par in parents:
            rows_out.append(np.stack(parts[at:at + heads], axis=1))
            at += heads
        return np.concatenate(rows_out)
    return stack(outs), stack(sizes), (stack(shifts) if shifts else None)
