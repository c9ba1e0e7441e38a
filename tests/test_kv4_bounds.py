"""CPU test of the bound that holds decode over 4-bit caches to its weights of 17 bits: a
simulation of the kernel's roundings keeps it, one with weights of a single bf16 product
does not."""
from __future__ import annotations

import math

import pytest
import torch

from kv4_tight import beyond, decode_bound
from kv4_util import held, quantised, spread


def case(D, n, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (quantised(torch.randn(n, 2, D, generator=g)) for _ in range(2))
    return (0.01 * torch.randn(1, 8, D, generator=g)).to(torch.bfloat16), k, v


def simulated(q, kparts, vparts, weight):
    """Attention with weights p s rounded by `weight`, the rest in 64 bits."""
    k, D = held(*kparts), q.shape[-1]
    out = []
    for h in range(8):
        g = h // 4
        score = q[0, h].double() @ k[:, g].T / math.sqrt(D)
        p = torch.exp(score - score.max())
        ps = weight((p[:, None] * spread(vparts[1][:, g].double(), D)).float()).double()
        out.append(((ps * vparts[0][:, g].double()).sum(0) + p @ spread(vparts[2][:, g].double(), D)) / p.sum())
    return torch.stack(out)[None].to(torch.bfloat16)


def high_and_low(x):
    high = x.to(torch.bfloat16).float()
    return high.double() + (x - high).to(torch.bfloat16).double()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [2, 5, 17, 32])
def test_bound_tells_weights_apart(D, n):
    wrong = 0
    for seed in range(4):
        q, k, v = case(D, n, seed)
        want, bound = decode_bound(q, k, v, n - 1)
        assert beyond(simulated(q, k, v, high_and_low), want, bound) == 0
        wrong += beyond(simulated(q, k, v, lambda x: x.to(torch.bfloat16).float()), want, bound)
    assert wrong
