"""Attention over a paged cache of shared latent vectors, as cases that can be timed and compared.

Every token leaves one latent vector (``latent`` values, shared by all heads) and
one rotated key (``rope`` values, shared too) in the cache.  Head h's key is
[key_up[h] c, r] and its value value_up[h] c for a token's latent c and rotated key r.

* ``angles``: cosines and sines of a step's positions, scaled for long contexts.
* ``write``: a step's latents and keys into the cache, the keys rotated.
* ``attend``: one layer of a step whose queries were multiplied by key_up already:
  the write, the queries' rotation, attention over the latents (what comes out has
  yet to be multiplied by value_up).
* ``layer``: the same with key_up and value_up, from per-head queries to per-head values.

A case's lengths come from the case alone (``lens_seed``); values and the
blocks' places in the pool come from the seed.  ``own`` says which side runs:
the plain torch forms below, or the package's calls.
"""

from __future__ import annotations

import importlib
import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

_CACHE = dict(heads=16, latent=512, rope=64, interleaved=True, dtype="bf16", block=16, lens_seed=1)


def _angles(**kw) -> dict:
    """``tokens`` positions below ``farthest``."""
    return {"op": "angles", "tokens": 1, "size": 64, "base": 10000.0, "scaling": "ramp", "factor": 32.0,
            "original": 4096, "farthest": 131072, **kw}


def _write(**kw) -> dict:
    """``tokens`` in ``requests`` runs, each after up to ``hist`` tokens of its own."""
    return {**_CACHE, "op": "write", "requests": 1, "tokens": 1, "hist": 64, **kw}


def _attend(**kw) -> dict:
    """``requests`` of ``q_lo``..``q_hi`` queries after ``ctx_lo``..``ctx_hi`` tokens, and ``chunk`` more queries of one
    request after ``chunk_ctx`` (0: none); ``tree``: the queries are draft trees."""
    return {**_CACHE, "op": "attend", "requests": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 1, "ctx_hi": 1, "tree": False,
            "chunk": 0, "chunk_ctx": 0, **kw}


def _layer(**kw) -> dict:
    return _attend(**{"nope": 128, "value": 128, **kw, "op": "layer"})


def listed() -> list[dict]:
    return [
        # Every decode step: one position of each of 64 sequences.
        _angles(name="angles_64", tokens=64),
        # A long prompt's positions, another scaling and base.
        _angles(name="angles_32760", tokens=32760, scaling="smooth", factor=8.0, original=8192, base=500000.0),
        # Every layer of a decode step: one token of each of 64 sequences.
        _write(name="write_64_tokens", requests=64, tokens=64, hist=4096),
        # Prompts of ragged lengths that continue partial blocks, narrow latents, blocks of 12, the half layout.
        _write(name="write_prompts_8190", latent=256, rope=32, interleaved=False, dtype="fp16", block=12, requests=16,
               tokens=8190, hist=50),
        # One chat of a few hundred tokens on one of eight ranks (16 heads each): latency.
        _attend(name="attend_1_short", ctx_lo=301, ctx_hi=301),
        # The batch of a serving rank: 64 sequences of 512 to 4096 tokens.
        _attend(name="attend_64", requests=64, ctx_lo=512, ctx_hi=4095),
        # Every head on one GPU (data-parallel attention): as much arithmetic as memory traffic.
        _attend(name="attend_32_128heads", heads=128, requests=32, ctx_lo=512, ctx_hi=4095),
        # Long documents in fp16, 32 heads.
        _attend(name="attend_16x32k_fp16", heads=32, dtype="fp16", requests=16, ctx_lo=32767, ctx_hi=32767),
        # Speculative decoding: 32 trees of a pending token and 8 drafts.
        _attend(name="attend_trees_32", requests=32, q_lo=9, q_hi=9, ctx_lo=500, ctx_hi=2560, tree=True),
        # A decode step from per-head queries to per-head values.
        _layer(name="layer_decode_48", requests=48, ctx_lo=256, ctx_hi=3000),
        # A chunk of a long document's prompt over the 14K tokens before it.
        _layer(name="layer_chunk_2048_of_16k", q_lo=2048, q_hi=2048, ctx_lo=14336, ctx_hi=14336),
        # A mixed step of a narrow fp16 model: 21 decoding sequences and one prompt, the half layout.
        _layer(name="layer_mixed_narrow", heads=40, latent=256, rope=32, nope=64, value=64, interleaved=False,
               dtype="fp16", requests=21, ctx_lo=100, ctx_hi=1900, chunk=1000),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    """Sequences of 1 to 32K tokens, batches of 1 to 128, 5 to 128 heads, latents of 128 to 512, blocks of 1 to 64."""
    op = rng.choice(("angles",) + ("write",) * 2 + ("decode",) * 4 + ("tree",) + ("layer",) * 4)
    if op == "angles":
        return _angles(tokens=_log_int(rng, 1, 32760), size=rng.choice((32, 64, 64, 128, 96)),
                       base=rng.choice((10000.0, 500000.0)), scaling=rng.choice(("none", "linear", "base", "ramp", "smooth")),
                       factor=rng.choice((2.0, 8.0, 32.0, 40.0)), original=rng.choice((4096, 8192)),
                       farthest=_log_int(rng, 64, 1 << 20))
    common = dict(latent=rng.choice((512, 512, 512, 256, 384, 128)), rope=rng.choice((64, 64, 32)),
                  interleaved=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "fp16")),
                  block=rng.choice((16, 16, 16, 32, 64, 12, 1)), lens_seed=rng.randrange(1 << 30),
                  heads=rng.choice((16, 16, 8, 32, 64, 128, 5, 20, 40)))
    if op == "write":
        tokens = _log_int(rng, 1, 8190)
        return _write(**common, tokens=tokens, requests=min(tokens, _log_int(rng, 1, 64)), hist=_log_int(rng, 1, 1024))
    if op == "layer":
        common.update(nope=rng.choice((128, 64)), value=rng.choice((128, 64)))
    make = _layer if op == "layer" else _attend
    shape = op if op != "layer" else rng.choice(("decode", "chunk", "chunk", "mixed", "tree"))
    if shape == "decode":
        hi = _log_int(rng, 2, 32767)
        case = make(**common, requests=_log_int(rng, 1, 128), ctx_lo=int(hi * rng.random()), ctx_hi=hi)
    elif shape == "tree":
        nodes, hi = rng.randint(3, 16), _log_int(rng, 16, 8192)
        case = make(**common, requests=_log_int(rng, 1, 64), q_lo=nodes, q_hi=nodes, ctx_lo=int(hi * rng.random()),
                    ctx_hi=hi, tree=True)
    elif shape == "mixed":
        hi = _log_int(rng, 2, 4096)
        case = make(**common, requests=_log_int(rng, 1, 32), ctx_lo=int(hi * rng.random()), ctx_hi=hi,
                    chunk=_log_int(rng, 2, 1024), chunk_ctx=rng.choice((0, 0, 700, 5001)))
    else:
        q, hi = _log_int(rng, 2, 2048), _log_int(rng, 16, 14336)
        case = make(**common, requests=_log_int(rng, 1, 8), q_lo=max(1, int(q * rng.random())), q_hi=q,
                    ctx_lo=0, ctx_hi=hi if rng.random() < 0.7 else 0)
    while _too_much(case):
        key = "requests" if case["requests"] > 1 else "chunk_ctx" if case["chunk_ctx"] > 1 else "ctx_hi"
        case[key] = max(1, case[key] // 2)
        case["ctx_lo"] = min(case["ctx_lo"], case["ctx_hi"])
    return case


def _too_much(case: dict) -> bool:
    w = work(case)
    reqs = _requests(case)
    longest, most = max(r["computed"] + r["n"] for r in reqs), max(r["n"] for r in reqs)
    scores = len(reqs) * case["heads"] * most * longest  # of the plain form
    rows = len(reqs) * longest * (case["latent"] + case["rope"])
    return w["bytes"] > 6.5e8 or w["flops"] > 4.5e11 or scores > 1.2e9 or rows > 4.0e8


# ---- a case's requests -------------------------------------------------------

def _requests(case: dict) -> list[dict]:
    """Per request: tokens already in the cache, new tokens, their parents (-1: none)."""
    rng = random.Random(case["lens_seed"])
    if case["op"] == "write":
        cuts = sorted(rng.sample(range(1, case["tokens"]), case["requests"] - 1)) if case["requests"] > 1 else []
        runs = [b - a for a, b in zip([0, *cuts], [*cuts, case["tokens"]])]
        return [dict(computed=rng.randint(0, case["hist"]), n=n, parents=tuple(range(-1, n - 1))) for n in runs]
    reqs = []
    for _ in range(case["requests"]):
        n = rng.randint(case["q_lo"], case["q_hi"])
        parents = tuple([-1] + [rng.randint(0, i - 1) for i in range(1, n)] if case["tree"] else range(-1, n - 1))
        reqs.append(dict(computed=rng.randint(case["ctx_lo"], case["ctx_hi"]), n=n, parents=parents))
    if case["chunk"]:
        reqs.append(dict(computed=case["chunk_ctx"], n=case["chunk"], parents=tuple(range(-1, case["chunk"] - 1))))
    return reqs


def _place(case: dict, seed: int) -> dict:
    """The requests with their block tables (disjoint, in random places) and their tokens' slots and positions."""
    reqs, bs = _requests(case), case["block"]
    need = [-(-(r["computed"] + r["n"]) // bs) for r in reqs]
    num_blocks = sum(need) + 7
    ids = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, at, slots, positions = [], 0, [], []
    for r, n in zip(reqs, need):
        table = ids[at:at + n]
        tables.append(tuple(table))
        at += n
        new = torch.arange(r["computed"], r["computed"] + r["n"])
        slots.append(torch.tensor(table)[new // bs] * bs + new % bs)
        depth: list[int] = []
        for p in r["parents"]:
            depth.append(0 if p < 0 else depth[p] + 1)
        positions.append(torch.tensor(depth) + r["computed"])
    return dict(requests=reqs, tables=tables, num_blocks=num_blocks, slots=torch.cat(slots).to(DEVICE),
                positions=torch.cat(positions).to(DEVICE))


def _step(case: dict, seed: int, place: dict) -> dict:
    """The cache's rows so far and the step's tensors, all from the seed."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, latent, rope = DTYPES[case["dtype"]], case["latent"], case["rope"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, device=DEVICE).normal_(std=std, generator=gen).to(dtype)

    tokens = len(place["slots"])
    both = normal(tokens, latent + rope)  # what the model's down projection gives, in one row
    out = dict(rows=normal(place["num_blocks"] * case["block"], latent + rope), slots=place["slots"],
               latent=both[:, :latent], rope_key=both[:, latent:])
    angle = place["positions"].double()[:, None] * _frequencies(rope, 10000.0)
    out["rotary"] = (angle.cos().float(), angle.sin().float())
    if case["op"] == "attend":
        out["query"] = normal(tokens, case["heads"], latent + rope)
        out["scale"] = 1.0 / math.sqrt(128 + rope)
    elif case["op"] == "layer":
        out["query"] = normal(tokens, case["heads"], case["nope"] + rope, std=1.5)
        out["key_up"] = normal(case["heads"], case["nope"], latent, std=latent ** -0.5)
        out["value_up"] = normal(case["heads"], case["value"], latent, std=latent ** -0.5)
        out["scale"] = 1.0 / math.sqrt(case["nope"] + rope)
    return out


def _gather_plans(case: dict, place: dict) -> list[dict]:
    """The plain attention's indices: of the requests alike, and of the one whose chunk is longer than theirs."""
    alike = case["requests"]
    before = sum(r["n"] for r in place["requests"][:alike])
    return [_gather_plan(case, place["requests"][:alike], place["tables"][:alike], 0)] + (
        [_gather_plan(case, place["requests"][alike:], place["tables"][alike:], before)] if case["chunk"] else [])


def _gather_plan(case: dict, reqs: list[dict], tables: list, first: int) -> dict:
    """Padded [requests, tokens] indices of requests whose first token is ``first``."""
    bs = case["block"]
    longest, queries = max(r["computed"] + r["n"] for r in reqs), max(r["n"] for r in reqs)
    at = torch.zeros((len(reqs), longest), dtype=torch.int64)
    rows = torch.zeros((len(reqs), queries), dtype=torch.int64)
    seen = torch.zeros((len(reqs), queries, queries), dtype=torch.bool)  # of the step's own tokens
    kept, start = [], first
    for b, (r, table) in enumerate(zip(reqs, tables)):
        n, pos = r["n"], torch.arange(r["computed"] + r["n"])
        at[b, :len(pos)] = torch.tensor(table)[pos // bs] * bs + pos % bs
        rows[b, :n] = torch.arange(start, start + n)
        seen[b, :n, :n] = _seen(r["parents"])
        kept += range(b * queries, b * queries + n)
        start += n
    computed = torch.tensor([r["computed"] for r in reqs])
    return {k: t.to(DEVICE) for k, t in dict(at=at, rows=rows, seen=seen, kept=torch.tensor(kept), computed=computed).items()}


def _seen(parents: tuple[int, ...]) -> torch.Tensor:
    n = len(parents)
    if parents == tuple(range(-1, n - 1)):
        return torch.ones((n, n), dtype=torch.bool).tril()
    seen = torch.zeros((n, n), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def _positions(case: dict, seed: int) -> torch.Tensor:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return torch.randint(0, case["farthest"], (case["tokens"],), generator=gen, device=DEVICE)


def prepare(case: dict, seed: int) -> dict:
    """Inputs, and what a serving program keeps: the cache, the step's metadata, the layer's weights laid out."""
    if case["op"] == "angles":
        state = dict(case=case, positions=_positions(case, seed))
        if own:
            lv = importlib.import_module("light-vllm_amd")
            scaling = None if case["scaling"] == "none" else lv.RotaryScaling(
                case["scaling"], factor=case["factor"], original_length=case["original"])
            state["embedding"] = lv.RotaryEmbedding(case["size"], base=case["base"], scaling=scaling, device=DEVICE)
        return state
    place = _place(case, seed)
    state = dict(case=case, **_step(case, seed, place))
    if case["op"] != "write":
        state["plans"] = _gather_plans(case, place)
    if own:
        _keep(state, place)
    return state


def _keep(state: dict, place: dict) -> None:
    """The package's cache with the same history, and the handles beside it."""
    lv = importlib.import_module("light-vllm_amd")
    case = state["case"]
    spec = lv.LatentKVCacheSpec((lv.LatentLayerSpec(
        "layer0", num_query_heads=case["heads"], latent_size=case["latent"], rope_size=case["rope"],
        rotary_layout="interleaved" if case["interleaved"] else "half"),))
    cache = lv.LatentPagedKVCache(spec, lv.PagedKVCacheConfig(
        num_blocks=place["num_blocks"], block_size=case["block"], dtype=DTYPES[case["dtype"]], device=DEVICE))
    rows = cache.layer("layer0").rows
    rows.view(-1, rows.shape[-1]).copy_(state["rows"])
    state.update(cache=cache, rows=rows.view(-1, rows.shape[-1]))
    if case["op"] == "write":
        state["mapping"] = cache.prepare_write(state["slots"])
        return
    state["backend"] = lv.HipPagedAttentionBackend()
    state["metadata"] = lv.PagedAttentionMetadata(
        block_tables=tuple(place["tables"]), num_computed_tokens=tuple(r["computed"] for r in place["requests"]),
        query_layouts=tuple(lv.QueryLayout(r["parents"]) for r in place["requests"]))
    state["weights"] = lv.LatentWeights(state["key_up"], state["value_up"]) if case["op"] == "layer" else None


# ---- one pass ------------------------------------------------------------------

def run(state: dict) -> dict:
    op = state["case"]["op"]
    if op == "angles":
        cosines, sines = state["embedding"](state["positions"]) if own else _plain_angles(state["case"], state["positions"])
        return dict(cosines=cosines, sines=sines)
    if own:
        if op == "write":
            state["cache"].write_prepared("layer0", state["latent"], state["rope_key"], state["mapping"],
                                          rotary=state["rotary"])
            return dict(rows=state["rows"])
        context = state["backend"].create(state["cache"], state["metadata"])
        attention = context.forward("layer0", state["query"], state["latent"], state["rope_key"], scale=state["scale"],
                                    rotary=state["rotary"], weights=state["weights"])
        return dict(attention=attention, rows=state["rows"])
    rows, latent = state["rows"], state["case"]["latent"]
    rows[state["slots"], :latent] = state["latent"]
    rows[state["slots"], latent:] = _plain_rotate(state["rope_key"].float(), state["rotary"], state["case"]).to(rows.dtype)
    if op == "write":
        return dict(rows=rows)
    return dict(attention=_plain_attend(state), rows=rows)


def _frequencies(size: int, base: float) -> torch.Tensor:
    return base ** (torch.arange(0, size, 2, dtype=torch.float64, device=DEVICE) / -size)


def _plain_angles(case: dict, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Angle i of a position is position * frequency i.  Scaled by a factor f for contexts f times the original: every
    frequency by it ("linear"), through the base ("base"), or those that turn little over the original context
    ("ramp": between the indices that turn 32 times and once; "smooth": between 4 turns and 1)."""
    size, base, f, turn = case["size"], case["base"], case["factor"], 2 * math.pi
    freq, kind = _frequencies(size, base), case["scaling"]
    magnitude = 1.0
    if kind == "linear":
        freq = freq / f
    elif kind == "base":
        freq = _frequencies(size, base * f ** (size / (size - 2)))
    elif kind == "ramp":
        low, high = (size * math.log(case["original"] / (turns * turn)) / (2 * math.log(base)) for turns in (32, 1))
        low, high = max(math.floor(low), 0), min(math.ceil(high), size - 1)
        index = torch.arange(size // 2, dtype=torch.float64, device=DEVICE)
        share = ((index - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq * (1 - share) + freq / f * share
        magnitude = 0.1 * math.log(f) + 1.0
    elif kind == "smooth":
        share = ((case["original"] * freq / turn - 1) / (4 - 1)).clamp(0, 1)
        freq = freq * share + freq / f * (1 - share)
    angle = positions.double()[:, None] * freq
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()


def _plain_rotate(x: torch.Tensor, rotary, case: dict) -> torch.Tensor:
    """The last dimension's pairs (2i, 2i + 1), or (i, i + half), turned by the token's angles."""
    cosines, sines = (t.to(x.dtype).view(t.shape[0], *[1] * (x.ndim - 2), t.shape[1]) for t in rotary)
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if case["interleaved"] else (x[..., :half], x[..., half:])
    a, b = a * cosines - b * sines, b * cosines + a * sines
    return torch.stack((a, b), dim=-1).flatten(-2) if case["interleaved"] else torch.cat((a, b), dim=-1)


def _plain_attend(state: dict) -> torch.Tensor:
    case, q = state["case"], state["query"].float()
    turned = _plain_rotate(q[..., -case["rope"]:], state["rotary"], case)
    q = q[..., :-case["rope"]]
    if case["op"] == "layer":
        q = torch.matmul(q.transpose(0, 1), state["key_up"].float()).transpose(0, 1)
    q = torch.cat((q, turned), dim=-1)
    out = torch.cat([_plain_step(state, plan, q[plan["rows"]]) for plan in state["plans"]])
    if case["op"] == "layer":
        out = torch.matmul(out.transpose(0, 1), state["value_up"].float().transpose(1, 2)).transpose(0, 1)
    return out.to(state["rows"].dtype).contiguous()


def _plain_step(state: dict, plan: dict, q: torch.Tensor) -> torch.Tensor:
    latent = state["case"]["latent"]
    keys = state["rows"].float()[plan["at"]]                               # [requests, tokens, latent + rope]
    (b, n, heads, _), t = q.shape, keys.shape[1]                           # q: [requests, queries, heads, latent + rope]
    scores = torch.matmul(q.flatten(1, 2), keys.transpose(1, 2)).view(b, n, heads, t) * state["scale"]
    own_at = torch.arange(t, device=DEVICE) - plan["computed"][:, None]    # [requests, tokens]: of the step's tokens
    index = own_at.clamp(0, n - 1)[:, None, :].expand(b, n, t)
    visible = (own_at < 0)[:, None] | ((own_at < n)[:, None] & plan["seen"].gather(2, index))
    scores = scores.masked_fill_(~visible[:, :, None], float("-inf"))
    # (Queries that pad a request see its prefix or nothing; they are left out below.)
    weights = (scores - scores.amax(dim=-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = weights.sum(dim=-1, keepdim=True)
    out = torch.matmul(weights.flatten(1, 2), keys[..., :latent]).view(b, n, heads, latent) / total
    return out.flatten(0, 1)[plan["kept"]]


# ---- what a pass cannot do without ---------------------------------------------

def work(case: dict) -> dict:
    if case["op"] == "angles":
        values = case["tokens"] * case["size"]
        return {"bytes": 8 * case["tokens"] + 4 * values, "flops": 20 * values}
    reqs, row, heads = _requests(case), case["latent"] + case["rope"], case["heads"]
    tokens, half = sum(r["n"] for r in reqs), case["rope"] // 2
    flops = 6 * tokens * half
    nbytes = 2 * 2 * tokens * row + 8 * tokens * half + 8 * tokens
    if case["op"] == "write":
        return {"bytes": nbytes, "flops": flops}
    flops += 6 * tokens * heads * half
    nbytes += 2 * row * sum(r["computed"] for r in reqs)  # (the step's own rows are read as inputs)
    shared = 2 * (row + case["latent"])                   # of a query and key, over the latents
    if case["op"] == "attend":
        nbytes += 2 * tokens * heads * (row + case["latent"])
        return {"bytes": nbytes, "flops": flops + sum(_pairs(r) * heads * shared for r in reqs)}
    nope, value = case["nope"], case["value"]
    nbytes += 2 * tokens * heads * (nope + case["rope"] + value) + 2 * heads * (nope + value) * case["latent"]
    up = 2 * case["latent"] * (nope + value)              # per head: of a query through the weights, or of a token
    apart = 2 * (nope + case["rope"] + value)             # of a query and key, over per-head keys and values
    return {"bytes": nbytes, "flops": flops + sum(
        heads * min(_pairs(r) * shared + r["n"] * up, _pairs(r) * apart + (r["computed"] + r["n"]) * up) for r in reqs)}


def _pairs(r: dict) -> int:
    """Query-key pairs of a request that some mask leaves (a tree's queries: all of the step's tokens at most)."""
    return r["n"] * r["computed"] + r["n"] * (r["n"] + 1) // 2


# ---- the definitions in 64 bits ------------------------------------------------

def _exact_angles(case: dict, positions: torch.Tensor) -> dict:
    size, base, f = case["size"], case["base"], case["factor"]
    freqs, magnitude = [], 1.0
    if case["scaling"] == "ramp":
        magnitude = 1.0 + math.log(f) / 10.0
        first = max(0, math.floor(size / 2 * math.log(case["original"] / (64 * math.pi), base)))
        last = min(size - 1, math.ceil(size / 2 * math.log(case["original"] / (2 * math.pi), base)))
    for i in range(size // 2):
        w = math.exp(-2 * i / size * math.log(base))
        if case["scaling"] == "linear":
            w /= f
        elif case["scaling"] == "base":
            w = math.exp(-2 * i / size * (math.log(base) + math.log(f) * size / (size - 2)))
        elif case["scaling"] == "ramp":
            slow = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            w = slow * (w / f) + (1 - slow) * w
        elif case["scaling"] == "smooth":
            turns = case["original"] * w / (2 * math.pi)
            w = w if turns > 4 else w / f if turns < 1 else w * ((turns - 1) / 3 + (4 - turns) / 3 / f)
        freqs.append(w)
    angle = positions.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device=DEVICE)
    return dict(cosines=magnitude * torch.cos(angle), sines=magnitude * torch.sin(angle))


def _exact_turned(x: torch.Tensor, rotary, interleaved: bool) -> torch.Tensor:
    """Each pair as a complex number times e^(i angle)."""
    wheel = torch.complex(rotary[0].double(), rotary[1].double()).view(x.shape[0], *[1] * (x.ndim - 2), -1)
    half = x.shape[-1] // 2
    pairs = x.double().unflatten(-1, (half, 2) if interleaved else (2, half))
    pairs = pairs if interleaved else pairs.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * wheel)
    return (turned if interleaved else turned.transpose(-1, -2)).flatten(-2)


def exact(case: dict, seed: int):
    if case["op"] == "angles":
        return _exact_angles(case, _positions(case, seed))
    place = _place(case, seed)
    step = _step(case, seed, place)
    latent, rope, dtype = case["latent"], case["rope"], DTYPES[case["dtype"]]
    rows = step["rows"].double()
    new = torch.cat((step["latent"].double(), _exact_turned(step["rope_key"], step["rotary"], case["interleaved"])), dim=1)
    rows[place["slots"]] = new
    if case["op"] == "write":
        return dict(rows=rows)
    held = rows.to(dtype).double()  # what the cache holds of them
    query = step["query"].double()
    turned = _exact_turned(step["query"][..., -rope:], step["rotary"], case["interleaved"])
    out, t0 = [], 0
    for r, table in zip(place["requests"], place["tables"]):
        n, total = r["n"], r["computed"] + r["n"]
        at = torch.arange(total)
        keys = held[(torch.tensor(table)[at // case["block"]] * case["block"] + at % case["block"]).to(DEVICE)]
        visible = torch.ones((n, total), dtype=torch.bool, device=DEVICE)
        visible[:, r["computed"]:] = _seen(r["parents"]).to(DEVICE)
        heads = []
        for h in range(case["heads"]):
            q, v = query[t0:t0 + n, h], keys[:, :latent]
            if case["op"] == "layer":  # through per-head keys and values
                k = torch.cat((keys[:, :latent] @ step["key_up"][h].double().T, keys[:, latent:]), dim=1)
                v = keys[:, :latent] @ step["value_up"][h].double().T
            else:
                k = keys
            s = torch.cat((q[:, :-rope], turned[t0:t0 + n, h]), dim=1) @ k.T * step["scale"]
            heads.append(torch.softmax(s.masked_fill(~visible, float("-inf")), dim=-1) @ v)
        out.append(torch.stack(heads, dim=1))
        t0 += n
    return dict(attention=torch.cat(out), rows=rows)
