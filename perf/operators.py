"""The operators of speculative serving over an 8-bit paged cache, as cases that can be timed and compared.

* ``append``: keys and values of a step's tokens into the 8-bit cache (e4m3
  codes, one power-of-two scale per block and kv head).
* ``attend``: one layer of a step over that cache: the append, then attention
  (single tokens, prompt chunks over their history, draft trees).
* ``compact``: the accepted rows of verified drafts to the contiguous tail.
* ``verify``: drafted tokens against the target's probabilities.

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
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn
LARGEST = 448.0   # of e4m3
LOWEST = -100     # smallest scale exponent

_CACHE = dict(hq=28, hkv=4, d=128, dtype="bf16", block=16, layers=1, lens_seed=1)


def _append(**kw) -> dict:
    """``tokens`` in ``requests`` runs, each after up to ``hist`` tokens of its own."""
    return {**_CACHE, "op": "append", "requests": 1, "tokens": 1, "hist": 64, **kw}


def _attend(**kw) -> dict:
    """``requests`` of ``q_lo``..``q_hi`` queries after ``ctx_lo``..``ctx_hi`` tokens; ``tree``: the queries are draft trees."""
    return {**_CACHE, "op": "attend", "requests": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 1, "ctx_hi": 1, "tree": False, **kw}


def _compact(**kw) -> dict:
    return {**_CACHE, "op": "compact", "requests": 1, "nodes": 8, "ctx_lo": 16, "ctx_hi": 64, **kw}


def _verify(**kw) -> dict:
    """``requests`` with ``lo``..``hi`` drafts each; ``chain``: drafted one after the other from known probabilities."""
    return {"op": "verify", "requests": 1, "lo": 4, "hi": 4, "vocab": 32000, "dtype": "fp32", "chain": True,
            "lens_seed": 1, **kw}


def listed() -> list[dict]:
    return [
        # Every layer of a decode step: one token of each of 64 sequences, 7B heads.
        _append(name="append_64_tokens", requests=64, tokens=64, hist=4096),
        # Prompts of ragged lengths that continue partial blocks: the bandwidth of the append.
        _append(name="append_prompts_8190", requests=16, tokens=8190, hist=50),
        # A narrow fp16 model with an odd block size.
        _append(name="append_d80_blocks_of_12", hq=16, hkv=2, d=80, dtype="fp16", block=12, requests=5, tokens=1023, hist=100),
        # The smallest step: four short chats of a 0.5B model.
        _attend(name="decode_4_d64", hq=14, hkv=2, d=64, requests=4, ctx_lo=37, ctx_hi=511),
        # The headline decode: 64 sequences of 512 to 4096 tokens, 7B heads.
        _attend(name="decode_64_7b", requests=64, ctx_lo=512, ctx_hi=4095),
        # Long contexts in fp16: 16 documents of 32K tokens.
        _attend(name="decode_16x32k_fp16", dtype="fp16", requests=16, ctx_lo=32767, ctx_hi=32767),
        # A chunk of a long document's prompt over the 14K tokens before it.
        _attend(name="chunk_2048_of_16k", q_lo=2048, q_hi=2048, ctx_lo=14336, ctx_hi=14336),
        # Speculative decoding: 32 trees of a pending token and 8 drafts, 1.5B heads.
        _attend(name="trees_32", hq=12, hkv=2, requests=32, q_lo=9, q_hi=9, ctx_lo=500, ctx_hi=2560, tree=True),
        # One chat's accepted drafts, through 12 layers.
        _compact(name="compact_1", hq=12, hkv=2, layers=12, ctx_lo=800, ctx_hi=800),
        # A large batch's accepted drafts.
        _compact(name="compact_128", hq=12, hkv=2, layers=12, requests=128, ctx_lo=16, ctx_hi=600),
        # One chat, a chain of four drafts from a draft model: latency.
        _verify(name="verify_chain_1", vocab=151936),
        # A batch of draft trees without probabilities (lookup drafts), odd vocabulary, 16-bit probabilities.
        _verify(name="verify_trees_128", requests=128, lo=3, hi=12, vocab=100003, dtype="bf16", chain=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(28, 4, 128)] * 4 + [(12, 2, 128)] * 3 + [(14, 2, 64)] * 3 + [(32, 8, 128), (8, 8, 64), (16, 2, 80), (16, 4, 96),
                                                                    (8, 2, 256), (32, 4, 32), (16, 2, 112), (16, 4, 192)]


def draw(rng: random.Random) -> dict:
    """Sequences of 1 to 32K tokens, batches of 1 to 128, head sizes 32 to 256, groups of 1 to 8, blocks of 4 to 64."""
    op = rng.choice(("append",) * 2 + ("decode",) * 4 + ("chunk",) * 2 + ("tree",) * 2 + ("compact",) * 2 + ("verify",) * 3)
    if op == "verify":
        chain, hi = rng.random() < 0.5, rng.randint(1, 12)
        return _verify(requests=_log_int(rng, 1, 128), lo=rng.randint(0, hi), hi=hi, vocab=_log_int(rng, 1000, 160000),
                       dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), chain=chain, lens_seed=rng.randrange(1 << 30))
    hq, hkv, d = rng.choice(_HEADS)
    common = dict(hq=hq, hkv=hkv, d=d, dtype=rng.choice(("bf16", "bf16", "fp16")),
                  block=rng.choice((16, 16, 16, 32, 64, 12, 4)), lens_seed=rng.randrange(1 << 30))
    if op == "append":
        tokens = _log_int(rng, 1, 8190)
        return _append(**common, tokens=tokens, requests=min(tokens, _log_int(rng, 1, 64)), hist=_log_int(rng, 1, 1024))
    if op == "compact":
        return _compact(**common, layers=rng.randint(1, 12), requests=_log_int(rng, 1, 128), nodes=rng.randint(2, 12),
                        ctx_hi=_log_int(rng, 64, 600))
    if op == "decode":
        hi = _log_int(rng, 2, 32767)
        case = _attend(**common, requests=_log_int(rng, 1, 128), ctx_lo=int(hi * rng.random()), ctx_hi=hi)
    elif op == "tree":
        nodes, hi = rng.randint(3, 16), _log_int(rng, 16, 8192)
        case = _attend(**common, requests=_log_int(rng, 1, 64), q_lo=nodes, q_hi=nodes, ctx_lo=int(hi * rng.random()),
                       ctx_hi=hi, tree=True)
    else:
        q, hi = _log_int(rng, 2, 2048), _log_int(rng, 16, 14336)
        case = _attend(**common, requests=_log_int(rng, 1, 8), q_lo=max(1, int(q * rng.random())), q_hi=q,
                       ctx_lo=0, ctx_hi=hi if rng.random() < 0.7 else 0)
    while _too_much(case):
        key = "requests" if case["requests"] > 1 else "ctx_hi"
        case[key] = max(1, case[key] // 2)
        case["ctx_lo"] = min(case["ctx_lo"], case["ctx_hi"])
    return case


def _too_much(case: dict) -> bool:
    w = work(case)
    scores = case["requests"] * case["hq"] * case["q_hi"] * (case["ctx_hi"] + case["q_hi"])  # of the plain form
    rows = case["requests"] * (case["ctx_hi"] + case["q_hi"]) * case["hkv"] * case["d"]
    return w["bytes"] > 5.4e8 or w["flops"] > 4.5e11 or scores > 1.0e9 or rows > 2.7e8


# ---- a case's requests -------------------------------------------------------

def _tree(rng: random.Random, drafts: int, chain: bool = False) -> tuple[tuple[int, ...], tuple[int, ...]]:
    """(parents of a pending token and a draft tree under it, an accepted root-to-leaf path)."""
    parents = [-1] + [i - 1 if chain else rng.randint(0, i - 1) for i in range(1, drafts + 1)]
    path, node = [], rng.randint(0, drafts)
    while node != -1:
        path.append(node)
        node = parents[node]
    return tuple(parents), tuple(sorted(path))


def _requests(case: dict) -> list[dict]:
    """Each request's computed tokens, parents of its queries and, for a tree, its accepted path."""
    rng = random.Random(case["lens_seed"])
    n = case["requests"]
    if case["op"] == "append":
        cuts = sorted(rng.sample(range(1, case["tokens"]), n - 1)) if n > 1 else []
        return [dict(computed=rng.randint(0, case["hist"]), n=b - a) for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    if case["op"] == "verify":
        return [dict(parents=_tree(rng, rng.randint(case["lo"], case["hi"]), case["chain"])[0]) for _ in range(n)]
    out = []
    for _ in range(n):
        computed = rng.randint(case["ctx_lo"], case["ctx_hi"])
        if case["op"] == "compact" or case["tree"]:
            parents, path = _tree(rng, case["nodes"] if case["op"] == "compact" else case["q_lo"] - 1)
            out.append(dict(computed=computed, n=len(parents), parents=parents, path=path))
        else:
            q = rng.randint(case["q_lo"], case["q_hi"])
            out.append(dict(computed=computed, n=q, parents=tuple(range(-1, q - 1))))
    return out


def _place(case: dict, seed: int) -> dict:
    """Block tables over a shuffled pool, and the slots of the step's tokens."""
    rng = random.Random(seed)
    bs, reqs = case["block"], _requests(case)
    need = [-(-(r["computed"] + r["n"]) // bs) for r in reqs]
    free = list(range(sum(need) + 5))
    rng.shuffle(free)
    count, tables = len(free), []
    for n in need:
        tables.append(tuple(free[:n]))
        free = free[n:]
    slots = [t[p // bs] * bs + p % bs for r, t in zip(reqs, tables) for p in range(r["computed"], r["computed"] + r["n"])]
    return dict(requests=reqs, tables=tables, slots=slots, num_blocks=count)


# ---- inputs ------------------------------------------------------------------

def _scale_of(amax: torch.Tensor) -> torch.Tensor:
    """2^e, e the smallest exponent (at least LOWEST) with amax <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(amax)
    e = torch.where(mantissa > LARGEST / 512, exponent - 8, exponent - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, LOWEST)).clamp(min=LOWEST)
    return torch.ldexp(torch.ones_like(amax), e)


def _values(case: dict, gen: torch.Generator, *shape: int) -> torch.Tensor:
    """Rows with channels of different sizes, as projections give them."""
    x = torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(generator=gen)
    return x * torch.empty(shape[-2:], device=DEVICE).normal_(std=0.5, generator=gen).exp()


def _pools(case: dict, num_blocks: int, gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """The cache's history: codes [layers, 2, blocks, block size, kv heads, head size], scales [layers, 2, blocks, kv heads]."""
    hkv, d, bs = case["hkv"], case["d"], case["block"]
    codes = torch.empty((case["layers"], 2, num_blocks, bs, hkv, d), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((case["layers"], 2, num_blocks, hkv), dtype=torch.float32, device=DEVICE)
    for layer in range(case["layers"]):
        for side in range(2):
            x = _values(case, gen, num_blocks, bs, hkv, d)
            s = scales[layer, side] = _scale_of(x.abs().amax(dim=(1, 3)))
            codes[layer, side] = (x / s[:, None, :, None]).to(F8).view(torch.uint8)
    return codes, scales


def _step(case: dict, place: dict, gen: torch.Generator) -> dict:
    t, dtype = len(place["slots"]), DTYPES[case["dtype"]]
    k, v = (_values(case, gen, t, case["hkv"], case["d"]).to(dtype) for _ in range(2))
    out = dict(key=k, value=v, slots=torch.tensor(place["slots"], dtype=torch.int64, device=DEVICE))
    if case["op"] == "attend":
        out["query"] = _values(case, gen, t, case["hq"], case["d"]).to(dtype)
    return out


def _gather_plan(case: dict, place: dict) -> dict:
    """Padded index tensors for the plain attention: keys' slots, queries' rows and who sees whom."""
    bs, reqs = case["block"], place["requests"]
    keys, queries = max(r["computed"] + r["n"] for r in reqs), max(r["n"] for r in reqs)
    at = torch.zeros((len(reqs), keys), dtype=torch.int64)
    rows = torch.zeros((len(reqs), queries), dtype=torch.int64)
    seen = torch.zeros((len(reqs), queries, queries), dtype=torch.bool)
    kept, start = [], 0
    for b, (r, table) in enumerate(zip(reqs, place["tables"])):
        n, pos = r["n"], torch.arange(r["computed"] + r["n"])
        at[b, :len(pos)] = torch.tensor(table)[pos // bs] * bs + pos % bs
        rows[b, :n] = torch.arange(start, start + n)
        if r["parents"] == tuple(range(-1, n - 1)):
            seen[b, :n, :n] = torch.ones((n, n), dtype=torch.bool).tril()
        else:
            for i, p in enumerate(r["parents"]):
                if p >= 0:
                    seen[b, i] = seen[b, p]
                seen[b, i, i] = True
        kept += range(b * queries, b * queries + n)
        start += n
    computed = torch.tensor([r["computed"] for r in reqs])
    return {k: t.to(DEVICE) for k, t in dict(at=at, rows=rows, seen=seen, kept=torch.tensor(kept), computed=computed).items()}


def _drafts(case: dict, seed: int) -> dict:
    """Target rows (a request's root, then its drafts), the drafts' tokens and, for chains, what they were drawn from."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    reqs, vocab, dtype = _requests(case), case["vocab"], DTYPES[case["dtype"]]
    rows = sum(len(r["parents"]) for r in reqs)
    logits = torch.empty((rows, vocab), device=DEVICE).normal_(std=3.0, generator=gen)
    target = logits.softmax(dim=-1).to(dtype)
    noisy = logits.add_(torch.empty((rows, vocab), device=DEVICE).normal_(std=0.7, generator=gen))
    root, drafted, parent_row, kth = [], [], [], []
    start = 0
    for r in reqs:
        root.append(start)
        born = [0] * len(r["parents"])
        for i, p in enumerate(r["parents"]):
            if i:
                drafted.append(start + i)
                parent_row.append(start + p)
                kth.append(born[p])
                born[p] += 1
        start += len(r["parents"])
    parent_row = torch.tensor(parent_row, dtype=torch.int64, device=DEVICE)
    out = dict(target=target, requests=reqs, draft_probs=None)
    if case["chain"]:
        q = noisy[parent_row].softmax(dim=-1)
        u = torch.rand((len(drafted), 1), device=DEVICE, dtype=torch.float64, generator=gen)
        cdf = q.double().cumsum(dim=-1)
        tokens = torch.searchsorted(cdf, u * cdf[:, -1:]).clamp(max=vocab - 1).flatten() if drafted else parent_row
        out["draft_probs"] = q.to(dtype)
    elif drafted:
        top = noisy.topk(min(vocab, max(kth) + 1), dim=-1).indices
        tokens = top[parent_row, torch.tensor(kth, device=DEVICE)]
    else:
        tokens = parent_row
    out["tokens"] = tokens
    out["node_uniforms"] = torch.rand(rows, device=DEVICE, generator=gen)
    out["sample_uniforms"] = torch.rand(len(reqs), device=DEVICE, generator=gen)
    return out


def _draft_plan(case: dict, drafts: dict) -> dict:
    """Padded [requests, drafts] indices for the plain verification."""
    reqs = drafts["requests"]
    b, most = len(reqs), max(1, max(len(r["parents"]) - 1 for r in reqs))
    draft = torch.zeros((b, most), dtype=torch.int64)
    valid = torch.zeros((b, most), dtype=torch.bool)
    prow = torch.zeros((b, most), dtype=torch.int64)
    row = torch.zeros((b, most), dtype=torch.int64)
    before = torch.zeros((b, most, most), dtype=torch.bool)   # earlier siblings and itself
    above = torch.zeros((b, most, most), dtype=torch.bool)    # ancestors and itself
    root, start, first = torch.zeros(b, dtype=torch.int64), 0, 0
    for i, r in enumerate(reqs):
        n = len(r["parents"]) - 1
        root[i] = start
        for j in range(n):
            p = r["parents"][j + 1]
            draft[i, j], valid[i, j], prow[i, j], row[i, j] = first + j, True, start + p, start + j + 1
            for s in range(j + 1):
                before[i, j, s] = r["parents"][s + 1] == p
            if p > 0:
                above[i, j] = above[i, p - 1]
            above[i, j, j] = True
        start += n + 1
        first += n
    plan = dict(draft=draft, valid=valid, prow=prow, row=row, before=before, above=above, root=root)
    return {k: t.to(DEVICE) for k, t in plan.items()}


def prepare(case: dict, seed: int) -> dict:
    """Inputs, and what a serving program keeps: the cache and its step plan, the drafts' plan."""
    if case["op"] == "verify":
        drafts = _drafts(case, seed)
        state = dict(case=case, drafts=drafts, plan=_draft_plan(case, drafts))
        if own:
            lv = importlib.import_module("light-vllm_amd")
            tokens, trees, at = drafts["tokens"].tolist(), [], 0
            for r in drafts["requests"]:
                n = len(r["parents"]) - 1
                trees.append(lv.DraftTree(tuple(tokens[at:at + n]), tuple(p - 1 for p in r["parents"][1:])))
                at += n
            state["batch"] = lv.DraftBatch(trees, device=DEVICE)
        return state
    place = _place(case, seed)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    codes, scales = _pools(case, place["num_blocks"], gen)
    state = dict(case=case, place=place, codes=codes, scales=scales, scale=1.0 / math.sqrt(case["d"]))
    pairs = [(r["computed"] + q, r["computed"] + i, t) for r, t in zip(place["requests"], place["tables"])
             for i, q in enumerate(r.get("path", ())) if i != q]
    if case["op"] == "compact":
        bs = case["block"]
        state["src"] = torch.tensor([t[a // bs] * bs + a % bs for a, _, t in pairs], dtype=torch.int64, device=DEVICE)
        state["dst"] = torch.tensor([t[z // bs] * bs + z % bs for _, z, t in pairs], dtype=torch.int64, device=DEVICE)
    else:
        state.update(_step(case, place, gen))
    if case["op"] == "attend":
        state["plan"] = _gather_plan(case, place)
    if own:
        _keep(state)
    return state


def _keep(state: dict) -> None:
    """The package's cache with the same history, and the handles beside it."""
    lv = importlib.import_module("light-vllm_amd")
    case, place = state["case"], state["place"]
    layers = tuple(f"layer{i}" for i in range(case["layers"]))
    spec = lv.ModelKVCacheSpec(tuple(lv.AttentionLayerSpec(i, case["hq"], case["hkv"], case["d"]) for i in layers))
    cache = lv.QuantizedPagedKVCache(spec, lv.PagedKVCacheConfig(
        num_blocks=place["num_blocks"], block_size=case["block"], dtype=DTYPES[case["dtype"]], device=DEVICE))
    for i, name in enumerate(layers):
        layer = cache.layer(name)
        for side, (pool, scales) in enumerate(((layer.keys, layer.key_scales), (layer.values, layer.value_scales))):
            pool.view(torch.uint8).copy_(state["codes"][i, side])
            scales.copy_(state["scales"][i, side])
    del state["codes"], state["scales"]
    state.update(cache=cache, pools=[cache.layer(i) for i in layers])
    reqs, tables = place["requests"], place["tables"]
    if case["op"] == "append":
        state["mapping"] = cache.prepare_write(state["slots"])
    elif case["op"] == "attend":
        state["backend"] = lv.HipPagedAttentionBackend()
        state["metadata"] = lv.PagedAttentionMetadata(
            block_tables=tuple(tables), num_computed_tokens=tuple(r["computed"] for r in reqs),
            query_layouts=tuple(lv.QueryLayout(r["parents"]) for r in reqs))
    else:
        state["compacts"] = [
            dict(block_ids=t, num_computed_tokens=r["computed"], num_query_tokens=r["n"], num_reserved_query_tokens=r["n"],
                 retained_query_indices=r["path"], num_readonly_prefix_blocks=0) for r, t in zip(reqs, tables)]


# ---- one pass ------------------------------------------------------------------

def run(state: dict) -> dict:
    op = state["case"]["op"]
    if op == "verify":
        d = state["drafts"]
        if own:
            lv = importlib.import_module("light-vllm_amd")
            v = lv.verify_drafts(state["batch"], d["target"], d["node_uniforms"], d["sample_uniforms"],
                                 draft_probs=d["draft_probs"])
            return dict(counts=v.counts, paths=v.paths, tokens=v.tokens)
        return _plain_verify(d, state["plan"])
    if own:
        cache, out = state["cache"], {}
        if op == "append":
            cache.write_prepared("layer0", state["key"], state["value"], state["mapping"])
        elif op == "attend":
            context = state["backend"].create(cache, state["metadata"])
            out["attention"] = context.forward("layer0", state["query"], state["key"], state["value"], scale=state["scale"])
        else:
            cache.compact_many(state["compacts"])
        return dict(out, pools=[(p.keys, p.values, p.key_scales, p.value_scales) for p in state["pools"]])
    codes, scales = state["codes"], state["scales"]
    out = {}
    if op == "compact":
        _plain_compact(codes, scales, state["src"], state["dst"])
    else:
        _plain_append(codes[0], scales[0], state["key"], state["value"], state["slots"])
    if op == "attend":
        out["attention"] = _plain_attend(codes[0], scales[0], state["query"], state["plan"], state["scale"])
    values = codes.view(F8)
    return dict(out, pools=[(k, v, ks, vs) for (k, v), (ks, vs) in zip(values.unbind(0), scales.unbind(0))])


def _plain_append(codes, scales, key, value, slots) -> None:
    """codes [2, blocks, block size, kv heads, head size], scales [2, blocks, kv heads], K and V at once."""
    bs = codes.shape[2]
    blocks, offset = slots // bs, slots % bs
    new = torch.stack((key, value)).float()
    largest = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0 ** 127}[key.dtype]
    size = torch.where(new.isfinite(), new.abs(), 0.0).amax(dim=-1)
    amax = torch.zeros_like(scales).index_reduce_(1, blocks, size, "amax")
    fresh = torch.zeros(scales.shape[1], dtype=torch.bool, device=slots.device)
    fresh[blocks[offset == 0]] = True
    at = blocks.unique()
    old, fresh = scales[:, at], fresh[at]
    grown = torch.where(fresh[None, :, None], _scale_of(amax[:, at]), torch.maximum(old, _scale_of(amax[:, at])))
    kept = codes[:, at].view(F8).float() * (old / grown)[:, :, None, :, None]
    kept = torch.where(fresh[None, :, None, None, None], codes[:, at], kept.to(F8).view(torch.uint8))
    codes[:, at] = kept
    scales[:, at] = grown
    x = torch.where(new.isfinite(), new.clamp(-largest, largest) / scales[:, blocks][..., None], math.nan)
    codes.flatten(1, 2)[:, slots] = x.to(F8).view(torch.uint8)


def _plain_attend(codes, scales, query, plan, scale):
    at, bs = plan["at"], codes.shape[2]
    rows = codes.flatten(1, 2)[:, at].view(F8).float() * scales[:, at // bs][..., None]  # [2, B, keys, Hkv, D]
    k, v = rows.permute(0, 1, 3, 2, 4).contiguous().unbind(0)
    b, hkv, keys, d = k.shape
    nq, hq = plan["rows"].shape[1], query.shape[1]
    q = query.float()[plan["rows"]].view(b, nq, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).view(b, hkv, nq, hq // hkv, keys)
    new = torch.arange(keys, device=at.device)[None] - plan["computed"][:, None]  # which of the step's tokens a key is
    inside = (new < nq)[:, None] & plan["seen"].gather(2, new.clamp(0, nq - 1)[:, None].expand(b, nq, keys))
    visible = (new < 0)[:, None] | inside
    scores = scores.masked_fill_(~visible[:, None, :, None], -math.inf)
    out = torch.matmul(scores.softmax(dim=-1).view(b, hkv, -1, keys), v)
    out = out.view(b, hkv, nq, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b * nq, hq, d)
    return out[plan["kept"]].to(query.dtype)


def _plain_compact(codes, scales, src, dst) -> None:
    codes, scales = codes.flatten(0, 1), scales.flatten(0, 1)
    bs = codes.shape[2]
    to = dst // bs
    rows = codes.flatten(1, 2)[:, src].view(F8).float() * scales[:, src // bs][..., None]
    grown = scales.clone().index_reduce_(1, to, scales[:, src // bs], "amax")
    at = to.unique()
    kept = codes[:, at].view(F8).float() * (scales[:, at] / grown[:, at])[:, :, None, :, None]
    codes[:, at] = kept.to(F8).view(torch.uint8)
    codes.flatten(1, 2)[:, dst] = (rows / grown[:, to][..., None]).to(F8).view(torch.uint8)
    scales.copy_(grown)


def _plain_verify(d: dict, plan: dict) -> dict:
    target, tokens, q = d["target"], d["tokens"], d["draft_probs"]
    vocab, most = target.shape[1], plan["draft"].shape[1]
    u, valid = d["node_uniforms"].double(), plan["valid"]
    positive = lambda p: torch.where(p.isfinite() & (p > 0), p, 0.0).double()  # noqa: E731
    if tokens.numel() == 0:
        tokens = torch.zeros(1, dtype=torch.int64, device=u.device)
    tok = tokens[plan["draft"]]
    p = torch.where(valid, positive(target[plan["prow"], tok]), 0.0)
    if q is None:
        upto = torch.where(plan["before"], p[:, None, :], 0.0).cumsum(dim=-1)[..., -1]
        chosen = (u[plan["prow"]] < upto) & (u[plan["prow"]] >= upto - p)
    else:
        drawn = positive(q[plan["draft"], tok]) if q.shape[0] else p
        chosen = u[plan["prow"]] * drawn < p
    chosen &= valid
    accepted = valid & (chosen[:, None, :] | ~plan["above"]).all(dim=-1)
    counts = accepted.sum(dim=-1)
    places = torch.arange(most, device=u.device)
    paths = torch.where(accepted, places, most).sort(dim=-1).values
    paths = torch.where(paths < most, paths, -1)
    last = paths.max(dim=-1).values
    stop = torch.where(last >= 0, plan["row"].gather(1, last.clamp(min=0)[:, None])[:, 0], plan["root"])
    rest = full = positive(target[stop])
    children = valid & (plan["prow"] == stop[:, None])
    if q is None:
        gone = torch.zeros((rest.shape[0], vocab + 1), dtype=torch.bool, device=u.device)
        gone = gone.scatter_(1, torch.where(children, tok, vocab), True)[:, :vocab]
        rest = torch.where(gone, 0.0, rest)
    elif q.shape[0]:
        rejected = torch.where(children, plan["draft"], 0).sum(dim=-1)
        less = torch.where(children.any(dim=-1)[:, None], positive(q[rejected]), 0.0)
        rest = (rest - less).clamp(min=0.0)
    rest = torch.where((rest > 0).any(dim=-1, keepdim=True), rest, full)
    cdf = rest.cumsum(dim=-1)
    beyond = cdf > (d["sample_uniforms"].double() * cdf[:, -1])[:, None]
    first = beyond.to(torch.int8).argmax(dim=-1)
    ids = torch.arange(vocab, device=u.device)
    final = torch.where(rest > 0, ids, -1).max(dim=-1).values  # the last that can be drawn; -1: none
    token = torch.where(beyond.any(dim=-1), first, final)
    return dict(counts=counts.to(torch.int32), paths=paths.to(torch.int32), tokens=token)


# ---- what a pass cannot do without ---------------------------------------------

def work(case: dict) -> dict:
    reqs = _requests(case)
    if case["op"] == "verify":
        # One row of the target's per request, and for a chain the row that its first rejected draft was drawn from.
        es, n = DTYPES[case["dtype"]].itemsize, sum(len(r["parents"]) for r in reqs)
        rows = len(reqs) * (2 if case["chain"] else 1)
        return dict(bytes=rows * case["vocab"] * es + n * (8 + 4 + 2 * es) + len(reqs) * 16, flops=rows * case["vocab"])
    row, bs = case["hkv"] * case["d"], case["block"]
    if case["op"] == "compact":
        moved = sum(1 for r in reqs for i, q in enumerate(r["path"]) if i != q)
        return dict(bytes=max(1, case["layers"] * 2 * moved * (2 * row + 12 * case["hkv"])), flops=0)
    written = sum(r["n"] for r in reqs)
    touched = sum(-(-(r["computed"] + r["n"]) // bs) - r["computed"] // bs for r in reqs)
    nbytes = 2 * (written * row * 3 + touched * 8 * case["hkv"]) + 8 * written
    if case["op"] == "append":
        return dict(bytes=nbytes, flops=2 * written * row)
    pairs = 0
    for r in reqs:
        depth = [0] * r["n"]
        for i, p in enumerate(r["parents"]):
            depth[i] = 1 + (depth[p] if p >= 0 else 0)
        pairs += r["computed"] * r["n"] + sum(depth)
        nbytes += 2 * r["computed"] * row + 2 * 2 * r["n"] * case["hq"] * case["d"] + 8 * -(-r["computed"] // bs) * case["hkv"]
    return dict(bytes=nbytes, flops=4 * case["hq"] * case["d"] * pairs)


# ---- the same in 64 bits, from the definitions -----------------------------------

def _rounded(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value (ties to even), in 64 bits; |x| at most 448."""
    size = x.abs()
    step = torch.exp2(torch.floor(torch.log2(torch.where(size > 0, size, 1.0))).clamp(min=-6.0) - 3.0)
    return torch.round(x / step) * step


def _exact_scale(largest: torch.Tensor) -> torch.Tensor:
    e = torch.full_like(largest, float(LOWEST))
    for k in range(LOWEST, 121):  # the smallest that holds it
        e = torch.where(largest > LARGEST * 2.0 ** k, float(k + 1), e)
    return torch.exp2(e)


def _exact_append(pool, scale, x, slots, bs) -> None:
    """One side: pool [blocks, bs, Hkv, D] of code values and scale [blocks, Hkv], 64 bits, in place."""
    by_block: dict[int, list[tuple[int, int]]] = {}
    for t, s in enumerate(slots):
        by_block.setdefault(s // bs, []).append((s % bs, t))
    names = list(by_block)
    index = torch.zeros(x.shape[0], dtype=torch.int64)
    for i, b in enumerate(names):
        index[[t for _, t in by_block[b]]] = i
    largest = torch.zeros((len(names),) + x.shape[1:2], dtype=torch.float64, device=x.device)
    largest = largest.scatter_reduce(0, index.to(x.device)[:, None].expand(-1, x.shape[1]), x.abs().amax(dim=-1), "amax")
    wanted = _exact_scale(largest)
    for i, b in enumerate(names):
        offs, toks = zip(*by_block[b])
        if 0 in offs:
            scale[b] = wanted[i]
        else:
            grown = torch.maximum(scale[b], wanted[i])
            pool[b] = _rounded(pool[b] * (scale[b] / grown)[None, :, None])
            scale[b] = grown
        pool[b, list(offs)] = _rounded(x[list(toks)] / scale[b][None, :, None])


def _attend_one(q, k, v, computed, parents, scale):
    """One request: q [n, Hq, D], k and v [computed + n, Hkv, D]."""
    n, hq, d = q.shape
    hkv, keys = k.shape[1], k.shape[0]
    seen = None
    if parents != tuple(range(-1, n - 1)):
        seen = torch.eye(n, dtype=torch.bool)
        for i, p in enumerate(parents):
            if p >= 0:
                seen[i] |= seen[p]
        seen = torch.cat((torch.ones((n, computed), dtype=torch.bool), seen), dim=1).to(q.device)
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    out = torch.empty_like(q)
    where = torch.arange(keys, device=q.device)
    for i in range(0, n, 256):
        part = q[i:i + 256]
        m = part.shape[0]
        see = seen[i:i + m] if seen is not None else where[None] <= (computed + i + torch.arange(m, device=q.device))[:, None]
        heads = part.reshape(m, hkv, hq // hkv, d).permute(1, 0, 2, 3).reshape(hkv, -1, d).contiguous()
        s = (torch.matmul(heads, kt) * scale).view(hkv, m, hq // hkv, keys).masked_fill_(~see[None, :, None], -math.inf)
        p = torch.softmax(s, dim=-1).view(hkv, -1, keys)
        out[i:i + m] = torch.matmul(p, vt).view(hkv, m, hq // hkv, d).permute(1, 0, 2, 3).reshape(m, hq, d)
    return out


def _exact_verify(case: dict, d: dict) -> dict:
    counts, paths, tokens = [], [], []
    all_tokens = d["tokens"].tolist()
    most = max(1, max(len(r["parents"]) - 1 for r in d["requests"]))
    row0 = first = 0
    for b, r in enumerate(d["requests"]):
        n, node, path = len(r["parents"]) - 1, 0, []
        mine = all_tokens[first:first + n]
        while True:
            p = d["target"][row0 + node].double()
            u = float(d["node_uniforms"][row0 + node])
            kids = [j for j in range(n) if r["parents"][j + 1] == node]
            taken, below = None, 0.0
            for j in kids:
                if case["chain"]:
                    taken = j if u * float(d["draft_probs"][first + j, mine[j]]) < float(p[mine[j]]) else taken
                else:
                    below += float(p[mine[j]])
                    if u < below:
                        taken = j
                        break
            if taken is None:
                break
            path.append(taken)
            node = taken + 1
        rest = p.clone()
        if case["chain"] and kids:
            rest = (rest - d["draft_probs"][first + kids[0]].double()).clamp(min=0.0)
        elif kids:
            rest[[mine[j] for j in kids]] = 0.0
        if not bool((rest > 0).any()):
            rest = p
        cdf = rest.cumsum(dim=0)
        hit = torch.nonzero(cdf > float(d["sample_uniforms"][b]) * cdf[-1])
        tokens.append(int(hit[0]) if len(hit) else int(torch.nonzero(rest > 0).max()))
        counts.append(len(path))
        paths.append(path + [-1] * (most - len(path)))
        row0 += n + 1
        first += n
    return dict(counts=torch.tensor(counts, dtype=torch.int32), paths=torch.tensor(paths, dtype=torch.int32),
                tokens=torch.tensor(tokens))


def exact(case: dict, seed: int):
    if case["op"] == "verify":
        return _exact_verify(case, _drafts(case, seed))
    place = _place(case, seed)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    codes, scales = _pools(case, place["num_blocks"], gen)
    bs, out = case["block"], {}
    if case["op"] == "compact":
        pools = codes.view(F8).double()
        sizes = scales.double()
        before, old = pools.clone(), sizes.clone()
        moves = [(t[(c + q) // bs], (c + q) % bs, t[(c + i) // bs], (c + i) % bs)
                 for r, t in zip(place["requests"], place["tables"]) for c in [r["computed"]]
                 for i, q in enumerate(r["path"]) if i != q]
        for a, _, z, _ in moves:
            sizes[:, :, z] = torch.maximum(sizes[:, :, z], old[:, :, a])
        for z in {m[2] for m in moves}:
            pools[:, :, z] = _rounded(before[:, :, z] * (old[:, :, z] / sizes[:, :, z])[:, :, None, :, None])
        for a, i, z, j in moves:
            pools[:, :, z, j] = _rounded(before[:, :, a, i] * (old[:, :, a] / sizes[:, :, z])[..., None])
        return dict(pools=[(p[0], p[1], s[0], s[1]) for p, s in zip(pools, sizes)])
    step = _step(case, place, gen)
    pools, sizes = codes[0].view(F8).double(), scales[0].double()
    for side, x in enumerate((step["key"], step["value"])):
        _exact_append(pools[side], sizes[side], x.double(), place["slots"], bs)
    if case["op"] == "attend":
        rows, t0 = [], 0
        for r, table in zip(place["requests"], place["tables"]):
            n = r["n"]
            at = torch.arange(r["computed"] + n)
            block, off = torch.tensor(table)[at // bs].to(DEVICE), (at % bs).to(DEVICE)
            k, v = (pools[s][block, off] * sizes[s][block][..., None] for s in range(2))
            rows.append(_attend_one(step["query"][t0:t0 + n].double(), k, v, r["computed"], r["parents"],
                                    1.0 / math.sqrt(case["d"])))
            t0 += n
        out["attention"] = torch.cat(rows)
    return dict(out, pools=[(pools[0], pools[1], sizes[0], sizes[1])])
