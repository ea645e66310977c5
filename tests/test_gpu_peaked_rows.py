"""Log-probabilities near 0: rows in which one token has nearly all of the mass, under a wide softcap."""

from __future__ import annotations

import pytest
import torch

from tests.dist_reference import Reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,k", [(200, 5), (3000, 7), (40000, 3)])
@pytest.mark.parametrize("softcap", [50.0, 300.0, None])
def test_selected_tokens_of_peaked_rows(cuda_device, V, k, softcap):
    """The best token's logit leaves its own log-probability: what is left is the error of the sum of the
    others' probabilities, and of the sums' and the result's roundings."""
    from gemma4_posttrain_jax_b200 import sample_top_k, top_token_logps

    T, d = 400, 64
    gen = torch.Generator(device=cuda_device).manual_seed(V)
    W = torch.randn((V, d), generator=gen, device=cuda_device) / 8
    likely = torch.randint(V, (T,), generator=gen, device=cuda_device)
    gap = 9 + 30 * torch.rand((T, 1), generator=gen, device=cuda_device)
    H = (torch.randn((T, d), generator=gen, device=cuda_device) / 2 + gap * W[likely]).to(torch.bfloat16)
    W = W.to(torch.bfloat16)
    ref = Reference(W, H, softcap)
    got = top_token_logps(W, H, softcap, k, tokens=likely)
    order = ref.order(k)
    assert torch.equal(got.ids.long(), order)
    # The others' probabilities are off by 2 delta of themselves, in all 2 delta (1 - p). The f32 sum of
    # terms that add up to 1 and little more: the 128 columns of a warp in pieces of 16, some 24 additions, and
    # their partials' (two per 256 columns, 16 to a thread and 12 steps over threads), 2^-24 each.
    rest = 1 - ref.p.gather(1, order[:, :1])
    sums = (24 + 16 + 12) * 2**-24
    for what, value, want in (
        ("logps", got.logps, ref.logp.gather(1, order)),
        ("token logps", got.token_logps[:, None], ref.logp.gather(1, likely[:, None])),
    ):
        off = (value.double() - want).abs()
        bound = 2 * ref.delta[:, None] * rest + sums + 2**-23 * want.abs()
        print(what, float((off / bound).max()))
        assert (off <= bound).all()
    u = torch.zeros((T,), device=cuda_device)  # draws the best
    token, logp = sample_top_k(W, H, softcap, u, temperature=1.0, top_k=k)
    assert torch.equal(token.long(), order[:, 0]) and torch.equal(logp, got.logps[:, 0])
