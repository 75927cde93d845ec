"""Steps of a layer over the latent cache, with its heads' weights or (``nope`` None)
in latent space, their result in fp64, and how far a kernel's result may be from it.

The bound is on the norm of a (token, head)'s error.  What the kernels round on the way
(u = eps / 2 of the step's type): turned queries, softmax weights (the sum that divides
them counts them as rounded), the result; absorbed the query in latent space and the
attended latents, expanded every key and value.  Each rounding is off by at most u of
its value; ``draws`` computes the result with every one of them off by a random share of
u, uniform in [-1, 1].  The errors of the roundings are independent, so their sum's norm
is near the root of the draws' mean square; the bound is 6 times that (the draws' own
spread included), plus the fp32 sums' (keys / 16 + 64 + latent) 2^-24 times the attention
of |value|, and the result's smallest step, 2^-24, in every value."""

from __future__ import annotations

import numpy as np
import torch

import light_vllm_amd as lv
from oracle import latent_oracle as Z

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TREE = (-1, 0, 0, 1, 1, 2, 3, 0, 7)
ROUNDS, DRAWS = 6.0, 8

# heads, latent, rope, nope, value, block, computed, layouts
SHORT = [
    (16, 512, 64, 128, 128, 16, [0, 31, 700], [1, 1, 1]),
    (5, 128, 32, 64, 128, 12, [90, 0, 40], [TREE, 3, 1]),
    (40, 256, 32, 64, 64, 16, [300], [1]),
    (128, 384, 64, 128, 64, 1, [133, 70], [2, 1]),
    (16, 512, 64, 128, 128, 16, [2500, 90], [TREE, TREE]),
]
LONG = [
    (4, 512, 64, 128, 128, 16, [0], [700]),
    (3, 512, 64, 128, 128, 16, [1000, 0], [513, 400]),
    (8, 128, 32, 64, 128, 12, [64, 5, 333], [129, 300, 191]),
    (2, 256, 32, 64, 64, 16, [130], [1025]),
    (5, 384, 64, 128, 64, 64, [63], [640]),
    (2, 512, 64, 128, 128, 16, [9000], [300]),  # units in pieces, merged
]
MIXED = [
    (16, 256, 32, 64, 64, 16, [100, 70, 50, 3000, 20], [1, 500, TREE, 1, 400]),
    (4, 512, 64, 128, 128, 32, [0, 700, 1500], [600, 1, 450]),
]
EVERY_LENGTH = (3, 256, 64, 128, 64, 16, [0, 63, 64, 500, 0, 1, 127], [1, 1, 2, 65, 128, 129, 256])


def make(case, dtype, seed: int, layout: str = "interleaved") -> dict:
    """A step on the CPU: the pool (NaN wherever no token is), the step's tensors, angles
    and weights."""

    heads, latent, rope, nope, value, bs, computed, layouts = case
    rng = np.random.default_rng(seed)
    layouts = [p if isinstance(p, tuple) else tuple(range(-1, p - 1)) for p in layouts]
    need = [-(-(c + len(p)) // bs) for c, p in zip(computed, layouts)]
    free = [int(b) for b in rng.permutation(sum(need) + 3)]
    tables = []
    for n in need:
        tables.append(tuple(free[:n]))
        free = free[n:]
    gen = torch.Generator().manual_seed(seed)
    rows = torch.full(((sum(need) + 3) * bs, latent + rope), torch.nan, dtype=dtype)
    for table, c in zip(tables, computed):
        at = torch.arange(c)
        rows[torch.tensor(table)[at // bs] * bs + at % bs] = torch.randn((c, latent + rope), generator=gen).to(dtype)
    t = sum(map(len, layouts))
    size = latent if nope is None else nope
    query = (1.5 * torch.randn((t, heads, size + rope), generator=gen)).to(dtype)
    both = torch.randn((t, latent + rope), generator=gen).to(dtype)
    up = None if nope is None else [(torch.randn((heads, n, latent), generator=gen) * latent**-0.5).to(dtype)
                                    for n in (nope, value)]
    angle = 100000.0 * torch.rand((t, rope // 2), generator=gen, dtype=torch.float64)
    md = lv.PagedAttentionMetadata(block_tables=tuple(tables), num_computed_tokens=tuple(computed),
                                   query_layouts=tuple(lv.QueryLayout(p) for p in layouts))
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec("layer0", heads, latent, rope, layout),))
    return dict(spec=spec, block=bs, num_blocks=sum(need) + 3, rows=rows, query=query, latent=both[:, :latent],
                rope_key=both[:, latent:], up=up, rotary=(angle.cos().float(), angle.sin().float()), metadata=md,
                slots=md.slot_mapping(block_size=bs, device=torch.device("cpu")), dtype=dtype)


def append(step: dict, rotary: bool = True) -> torch.Tensor:
    """The pool with the step's rows, as the type holds them."""

    layer = step["spec"].layers[0]
    key = step["rope_key"].double().numpy()
    if rotary:
        key = Z.rotate(key, *(a.double().numpy() for a in step["rotary"]), layer.rotary_layout == "interleaved")
    rows = step["rows"].clone()
    rows[step["slots"]] = torch.cat((step["latent"].double(), torch.from_numpy(key)), dim=1).to(step["dtype"])
    return rows


def attend(step: dict, rows: torch.Tensor, expanded, *, scale: float, rotary: bool = True, heads=None, gen=None, seen=None,
           shift: int = 0):
    """fp64 [tokens, heads, value] over the pool ``rows`` and the attention of |value|, on
    the device of ``rows``.  ``expanded``: of each request, its form (for the roundings).
    ``gen``: each rounding off by a random share of u.  ``seen(request, mask)`` and
    ``shift`` (heads by which the result is off) plant mistakes."""

    layer, bs, device = step["spec"].layers[0], step["block"], rows.device
    latent, rope = layer.latent_size, layer.rope_size
    u = torch.finfo(step["dtype"]).eps / 2
    q = step["query"].double().numpy().copy()
    if rotary:
        q[..., -rope:] = Z.rotate(q[..., -rope:], *(a.double().numpy() for a in step["rotary"]),
                                  layer.rotary_layout == "interleaved")
    q = torch.from_numpy(q).to(device)
    up = None if step["up"] is None else [w.to(device).double() for w in step["up"]]
    heads = range(q.shape[1]) if heads is None else heads

    def rounded(x):
        return x if gen is None else x * (1 + u * (2 * torch.rand(x.shape, generator=gen, dtype=x.dtype, device=x.device) - 1))

    md, outs, sizes, t0 = step["metadata"], [], [], 0
    for r, (table, c, tokens) in enumerate(zip(md.block_tables, md.num_computed_tokens, md.query_layouts)):
        n = len(tokens)
        at = torch.arange(c + n)
        keys = rows[(torch.tensor(table)[at // bs] * bs + at % bs).to(device)].double()
        mask = torch.from_numpy(Z.visible(tokens.parent_indices, c)).to(device)
        mask = mask if seen is None else seen(r, mask)
        c_, r_ = keys[:, :latent], keys[:, latent:]
        out, size = [], []
        for h in heads:
            h = (h + shift) % q.shape[1]
            qn, qr = q[t0:t0 + n, h, :-rope], q[t0:t0 + n, h, -rope:]
            s = (rounded(qr) if rotary else qr) @ r_.T
            if up is None:
                s = s + qn @ c_.T
            elif expanded[r]:
                s = s + qn @ rounded(c_ @ up[0][h].T).T
            else:
                s = s + rounded(qn @ up[0][h]) @ c_.T
            s = (s * scale).masked_fill(~mask, -torch.inf)
            w = rounded(torch.exp(s - s.amax(dim=1, keepdim=True)))
            w = w / w.sum(dim=1, keepdim=True)
            if up is None:
                v = c_
                o = w @ v
            elif expanded[r]:
                v = c_ @ up[1][h].T
                o = w @ rounded(v)
            else:
                v = c_ @ up[1][h].T
                o = rounded(w @ c_) @ up[1][h].T
            out.append(rounded(o))
            size.append(w @ v.abs())
        outs.append(torch.stack(out, dim=1))
        sizes.append(torch.stack(size, dim=1))
        t0 += n
    return torch.cat(outs), torch.cat(sizes)


def bound(step: dict, rows: torch.Tensor, expanded, want, size, **kw):
    """[tokens, heads]: what the norm of an error may be."""

    gen = torch.Generator(device=rows.device).manual_seed(1)
    square = sum((attend(step, rows, expanded, gen=gen, **kw)[0] - want).square().sum(dim=-1) for _ in range(DRAWS)) / DRAWS
    md = step["metadata"]
    keys = torch.cat([torch.full((len(p),), c + len(p)) for c, p in zip(md.num_computed_tokens, md.query_layouts)])
    sums = (keys / 16 + 64 + step["spec"].layers[0].latent_size).double().to(rows.device)[:, None] * 2.0**-24
    return ROUNDS * square.sqrt() + sums * size.norm(dim=-1) + 2.0**-24 * want.shape[-1] ** 0.5


def scale_of(case) -> float:
    return ((case[3] or 128) + case[2]) ** -0.5
