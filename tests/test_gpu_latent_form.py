"""GPU tests of which form a prompt of latent attention takes: the outputs of the two
differ in their last bits, so that equal ones tell the form."""
from __future__ import annotations

import pytest
import torch

from gpu_util import tuned
from test_gpu_latent import SMALL, WIDE, bf16, generator, make_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("widths,H,cached,rows,form", [
    # Keys and values of all heads pass the workspace, and every pass of a few heads
    # walks the tokens: 29.0 ms expanded against 10.0 absorbed; 12.4 against 6.6.
    (WIDE, 128, 131072, 256, "absorbed"),
    (SMALL, 128, 131072, 256, "absorbed"),
    # More rows: 8.9 ms against 18.8; in one pass 0.67 against 1.6, 0.13 against 0.62.
    (WIDE, 128, 60000, 1024, "expanded"),
    (WIDE, 128, 8000, 512, "expanded"),
    (WIDE, 64, 1000, 1024, "expanded"),
    (WIDE, 128, 8000, 4, "absorbed"),
])
def test_form_of_a_prompt(torch_dev, widths, H, cached, rows, form):
    rank, rope, nope, v = widths
    g = generator(61)
    with tuned() as rt, tuned(QM38_LATENT_FORM=1) as one, tuned(QM38_LATENT_FORM=2) as two:
        _, _, weights = make_weights(rt, g, H, widths)
        cache = rt.create_latent_kv(rank, rope)
        cache.append(bf16(g, cached, rank + rope), None, 0.0, cached)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        outs = []
        for r in (rt, one, two):
            outs.append(torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev))
            r.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, outs[-1])
            torch.cuda.synchronize()
            cache.truncate(cached)
        taken, absorbed, expanded = outs
        assert not torch.equal(absorbed, expanded)
        assert torch.equal(taken, absorbed if form == "absorbed" else expanded)
        weights.close()
        cache.close()


def test_prompt_whose_workspace_does_not_fit(torch_dev):
    """Keys and values of all heads at once (a workspace of 400 GB allowed) pass the
    device's memory: the call takes the other form instead of failing, and later calls
    go on."""
    rank, rope, nope, v = SMALL
    g = generator(62)
    H, cached, rows = 256, 6_000_000, 256
    if torch.cuda.mem_get_info()[1] > (cached * H * 256 * 9) // 10:
        pytest.skip("the device holds them")
    with tuned(QM38_LATENT_MB=400_000) as rt, tuned(QM38_LATENT_FORM=1) as one:
        _, _, weights = make_weights(rt, g, H, SMALL)
        cache = rt.create_latent_kv(rank, rope)
        cache.reserve(cached + rows)
        many = bf16(g, 500_000, rank + rope)
        for _ in range(cached // len(many)):
            cache.append(many, None, 0.0, len(many))
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        outs = []
        for r in (rt, one):
            outs.append(torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev))
            r.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, outs[-1])
            torch.cuda.synchronize()
            assert cache.sequence_length == cached + rows
            cache.truncate(cached)
        assert torch.isfinite(outs[0]).all() and torch.equal(*outs)
        cache.truncate(1000)  # a prompt whose workspace is there again
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, outs[0])
        torch.cuda.synchronize()
        assert cache.sequence_length == 1000 + rows and torch.isfinite(outs[0]).all()
        weights.close()
        cache.close()
