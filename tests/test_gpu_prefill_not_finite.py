"""Prefill over a bf16 cache when a score is not finite: the rows that see it are NaN wherever the key stands, as the reference's
arithmetic makes them, and the others are as they were."""
import math

import pytest
import torch

import gguf_runner_b200 as g
from gguf_runner_b200.binding import AttnConfig, KV_BF16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("prefix,m", [(0, 300), (1700, 333)])
def test_a_key_that_is_not_finite_counts_wherever_it_stands(prefix, m, d, bad):
    """At every residue of 8, in one launch and (behind a prefix) with split keys. One element, which RoPE makes two."""
    ctx = g.AttnContext(AttnConfig(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=d, seq_len=2100, rope_theta=1e6, kv_format=KV_BF16))
    gen = torch.Generator(device="cuda").manual_seed(d)
    q, k, v = (torch.randn(prefix + m, h, d, generator=gen, device="cuda").bfloat16() for h in (4, 2, 2))

    def run(keys):
        rows = [x.view(prefix + m, -1) for x in (q, keys, v)]
        if prefix:
            ctx.prefill(0, 0, *(x[:prefix] for x in rows))
        return ctx.prefill(0, prefix, *(x[prefix:] for x in rows)).view(m, 4, d)

    want = run(k).clone()
    assert bool(torch.isfinite(want).all())
    for r in range(8):
        at = (prefix or 192) - 96 + r
        spoilt = k.clone()
        spoilt[at, 1, 5] = bad
        got = run(spoilt)
        first = max(0, at - prefix)
        assert torch.equal(got[:, :2], want[:, :2]) and torch.equal(got[:first], want[:first])
        seen = got[first:, 2:]
        if math.isnan(bad):
            assert bool(seen.isnan().all()), (r, float(seen.isnan().double().mean()))
        else:  # +inf in one rotated element and +inf or -inf in the other: a score of +inf, NaN or -inf by the signs of q
            assert bool((seen.isnan().all(-1) | torch.isfinite(seen).all(-1)).all()), r
            assert bool(seen.isnan().any())
