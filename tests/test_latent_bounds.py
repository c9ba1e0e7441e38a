"""CPU tests of the error bounds that the latent attention tests use: they let a
result through that is rounded as the kernels round, and stop one with a row that is
missing, masked at another token, or held in fewer bits."""
from __future__ import annotations

import pytest
import torch

from latent_util import assert_attention_rows, attention, attention_rows

WIDTHS = {"wide": (512, 64, 128, 128), "small": (256, 32, 64, 64)}


def case(widths, rows, H, cached, std=1.5):
    rank, rope, nope, v = WIDTHS[widths]
    g = torch.Generator()
    g.manual_seed(rows + H)
    randn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q = (randn(rows, H, nope + rope) * std).to(torch.bfloat16)
    kv_b = (randn(H, nope + v, rank) * rank ** -0.5).to(torch.bfloat16)
    latent, key = randn(cached + rows, rank).double(), randn(cached + rows, rope).double()
    return q, latent, key, kv_b, nope, (nope + rope) ** -0.5, cached


def stopped(got, ref, bound):
    with pytest.raises(AssertionError):
        assert_attention_rows(got, ref, bound)


SIZES = [("wide", 300, 8, 0), ("wide", 40, 6, 500), ("small", 130, 5, 31), ("small", 7, 3, 2000)]


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
@pytest.mark.parametrize("size", SIZES)
def test_a_rounded_result_passes_and_a_missing_row_does_not(form, size):
    args = case(*size)
    ref, bound = attention_rows(*args, form)
    rounded = ref.to(torch.bfloat16)
    assert_attention_rows(rounded, ref, bound)
    for row in range(0, ref.shape[0], 6):
        for head in range(ref.shape[1]):
            broken = rounded.clone()
            broken[row, head] = 0
            stopped(broken, ref, bound)


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
@pytest.mark.parametrize("size", SIZES)
def test_a_mask_one_token_off_does_not_pass(form, size):
    """Sixteen rows that miss their last token, or see the next one."""
    args = case(*size)
    ref, bound = attention_rows(*args, form)
    start = args[-1]
    off = [attention(*args[:-1], start + d)[0] for d in (-1, 1)]
    for row in range(1, ref.shape[0] - 1, 16):
        rows = slice(row, min(row + 16, ref.shape[0] - 1))
        for other in off:
            broken = ref.to(torch.bfloat16)
            broken[rows] = other[rows].to(torch.bfloat16)
            stopped(broken, ref, bound)


@pytest.mark.parametrize("part", ["nothing", "keys", "values", "weights"])
def test_parts_held_in_bf16_do_not_pass(part):
    """Keys, values or softmax weights rounded to bf16 instead of fp16: seen in the sum of
    many rows."""
    args = q, latent, key, kv_b, nope, scale, start = case("wide", 300, 16, 0, std=4.0 if part == "keys" else 1.5)
    ref, bound = attention_rows(*args, "expanded")
    w, x = kv_b.double(), q.double().transpose(0, 1)
    rounded = lambda y, *parts: y.to(torch.bfloat16 if part in parts else torch.float16).double()  # noqa: E731
    k = rounded(latent @ w[:, :nope].transpose(1, 2), "keys")
    v = rounded(latent @ w[:, nope:].transpose(1, 2), "values")
    score = (x[..., :nope] @ k.transpose(1, 2) + x[..., nope:] @ key.T) * scale
    score = torch.where(torch.ones(300, 300, dtype=torch.bool).tril(), score, -torch.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True)) * 64
    got = (rounded(p, "weights") @ v / p.sum(-1, keepdim=True)).transpose(0, 1).to(torch.bfloat16)
    if part == "nothing":
        assert_attention_rows(got, ref, bound)
    else:
        stopped(got, ref, bound)
