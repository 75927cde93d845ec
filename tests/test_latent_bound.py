"""The bound that tests of latent steps hold kernels to (``latent_cases``), on the CPU:
results with a mistake in them pass it by far."""

from __future__ import annotations

import pytest
import torch

import latent_cases as L

LATENT_SPACE = (16, 512, 64, None, None, 16, [0, 431, 700], [1, L.TREE, 40])
CASES = [(c, False) for c in L.SHORT] + [(c, True) for c in L.LONG] + [
    (L.EVERY_LENGTH, True), (L.EVERY_LENGTH, False), (LATENT_SPACE, False)]


def _heads(case):
    return sorted({0, case[0] // 2, case[0] - 1})


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("case, expanded", CASES)
def test_mistakes_pass_the_bound(case, expanded, dtype) -> None:
    step = L.make(case, L.DTYPES[dtype], seed=3)
    rows, forms, kw = L.append(step), [expanded] * len(case[6]), dict(scale=L.scale_of(case), heads=_heads(case))
    want, size = L.attend(step, rows, forms, **kw)
    assert want.isfinite().all()
    most = L.bound(step, rows, forms, want, size, **kw)

    def beyond(got):
        """Share of the (token, head) pairs that ``got`` differs in whose error passes the bound."""
        off = (got - want).norm(dim=-1)
        changed = off > 0
        assert changed.any()
        return float((off > most)[changed].double().mean())

    assert beyond(torch.zeros_like(want)) == 1.0
    if case[0] > 1:  # (of one key the heads differ too: in their values)
        assert beyond(L.attend(step, rows, forms, shift=1, **kw)[0]) == 1.0
    # A tile of 64 keys that every later query should see; one piece of the keys.
    for first, last in ((0, 64), (128, 192), (0, 4096)):
        def without(r, mask, first=first, last=last):
            mask = mask.clone()
            if mask.shape[1] - len(mask) > last or mask.shape[1] > last + 64:
                mask[last:, first:last] = False  # (of queries that see others)
            return mask

        got = L.attend(step, rows, forms, seen=without, **kw)[0]
        if (got != want).any():
            assert beyond(got) > 0.5
    # Every query sees the step's next token too, or not its own.
    def next_token(r, mask):
        out, c = mask.clone(), mask.shape[1] - len(mask)
        for i in range(len(mask) - 1):
            out[i, c + i + 1] = True
        return out

    def not_its_own(r, mask):
        out, c = mask.clone(), mask.shape[1] - len(mask)
        for i in range(len(mask)):
            if out[i].sum() > 1:
                out[i, c + i] = False
        return out

    for wrong in (next_token, not_its_own):
        got = L.attend(step, rows, forms, seen=wrong, **kw)[0]
        # (One key of hundreds weighs less than bf16's roundings.)
        if (got != want).any() and dtype == "fp16":
            assert beyond(got) > 0.1
    # Queries that were not turned.
    assert beyond(L.attend(step, rows, forms, rotary=False, **kw)[0]) > 0.5


@pytest.mark.parametrize("scale", (1.0, -0.5))
def test_mistakes_pass_the_bound_at_other_scales(scale) -> None:
    case = (4, 128, 32, 64, 64, 16, [200, 30], [300, 2])
    step = L.make(case, torch.bfloat16, seed=4)
    rows, forms, kw = L.append(step), [True, False], dict(scale=scale)
    want, size = L.attend(step, rows, forms, **kw)
    most = L.bound(step, rows, forms, want, size, **kw)
    for got in (torch.zeros_like(want), L.attend(step, rows, forms, shift=1, **kw)[0],
                L.attend(step, rows, forms, scale=-scale)[0]):
        assert float(((got - want).norm(dim=-1) > most).double().mean()) > 0.98
