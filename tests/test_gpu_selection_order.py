"""The order that ``top_token_logps`` and ``sample_top_k`` promise -- exact dot products, the lowest id first
among equals -- where f32 sums cannot tell the tokens apart: cancelling terms, thousands of neighbours within
a rounding, rows of the embedding of very different lengths."""

from __future__ import annotations

import pytest
import torch

from tests.dist_reference import Reference, within

pytestmark = pytest.mark.gpu

# columns per selection key at k <= 20: the f32 sums themselves, groups of 8, groups of 32
VOCABS = [1200, 9001, 60000]

def _cancelling(V, d=1024, seed=5):
    """Seven rows whose dot product with a row of ones is exactly 0, the sum of terms from 2^-16 to 2^6 that
    f32 rounds differently in each; -1 for every other row."""
    gen = torch.Generator().manual_seed(seed)
    W = torch.zeros((V, d))
    part = torch.randn((256,), generator=gen) * 2.0 ** torch.randint(-16, 6, (256,), generator=gen)
    part = part.to(torch.bfloat16).float()
    W[:, :256] = part
    some = [5, 9, 17, 33, 40, 51, 60]
    for i in some:
        W[i, :256] = part[torch.randperm(256, generator=gen)]
    W[:, 256:512] = -part
    W[:, 512] = -1.0
    W[some, 512] = 0.0
    return W.to(torch.bfloat16), torch.ones((1, d), dtype=torch.bfloat16), some


@pytest.mark.parametrize("V", [64, 4099, 60000])
@pytest.mark.parametrize("k", [1, 4, 7])
def test_equal_sums_of_cancelling_terms(cuda_device, V, k):
    from gemma4_posttrain_jax_b200 import sample_top_k, top_token_logps

    W, H, some = _cancelling(V)
    W, H = W.to(cuda_device), H.to(cuda_device)
    got = top_token_logps(W, H, None, k)
    assert got.ids[0].tolist() == some[:k]
    # k equal weights: the numbers (j + 1/2) / k draw token j
    u = (torch.arange(k, device=cuda_device) + 0.5) / k
    token, _ = sample_top_k(W, H.expand(k, -1), None, u, temperature=1.0, top_k=k)
    assert token.tolist() == some[:k]


@pytest.mark.parametrize("d", [16, 136, 2048, 8192])
def test_what_an_accumulator_may_be_off_by(cuda_device, d):
    """The bound that the selection counts on, (17/4 + 1) 2^-23 of |h| |w| for every 16 terms, against sums
    that lose the most: one large term with many that lie just below its last bits, on either side of it."""
    from gemma4_posttrain_jax_b200 import _lib, ops

    lib = _lib.load()
    gen = torch.Generator(device=cuda_device).manual_seed(d)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=cuda_device)

    small = 2.0 ** -torch.arange(10, 42, device=cuda_device).float()[:, None]
    rows = []
    for sign in (1.0, -1.0):
        for size in (1.0, 1.9921875):
            for every in (d, 64, 16):
                w = (size * sign * small).expand(-1, d).clone()
                w[:, ::every] = 1.0
                rows.append(w)
    rows += [normal(64, d), normal(64, d).abs(), normal(64, d) * 2.0 ** torch.randint(-12, 12, (64, d), generator=gen, device=cuda_device)]
    W = torch.cat(rows).to(torch.bfloat16)
    H = torch.cat([torch.ones((1, d), device=cuda_device), normal(63, d), normal(64, d).abs()]).to(torch.bfloat16)
    D = torch.empty((H.shape[0], W.shape[0]), device=cuda_device)
    rc = lib.lp_gemm_bf16(ops._stream(cuda_device), ops._ptr(H), H.shape[0], d, d, 0, ops._ptr(W), W.shape[0], d, 0,
                          ops._ptr(D), W.shape[0])
    _lib.check(rc, "lp_gemm_bf16")
    off = (D.double() - H.double() @ W.double().T).abs()
    lengths = H.double().norm(dim=1)[:, None] * W.double().norm(dim=1)
    within(off, torch.zeros_like(off), -(-d // 16) * 5.25 * 2**-23 * lengths, "accumulators")


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("order", [[0, 1], [1, 0]])
def test_thousands_of_neighbours_within_a_rounding(cuda_device, V, order):
    """Logits 1 + u 2^-12 for 256 values of u between 0 and 1: far more of them lie within a rounding of the
    k-th than are looked at first, and those that differ are told apart."""
    from gemma4_posttrain_jax_b200 import top_token_logps

    k, d = 20, 64
    gen = torch.Generator(device=cuda_device).manual_seed(V)
    W = torch.zeros((V, d), device=cuda_device)
    W[:, order[0]] = 1.0
    W[:, order[1]] = torch.rand((V,), generator=gen, device=cuda_device)
    H = torch.zeros((3, d), device=cuda_device)
    H[:, order[0]] = torch.tensor([1.0, 2.0, -4.0], device=cuda_device)
    H[:, order[1]] = torch.tensor([2.0**-12, -(2.0**-13), 2.0**-12], device=cuda_device)
    W, H = W.to(torch.bfloat16), H.to(torch.bfloat16)
    ref = Reference(W, H, None)
    got = top_token_logps(W, H, None, k)
    assert torch.equal(got.ids.long(), ref.order(k))
    best = ref.logp.gather(1, ref.order(k))
    within(got.logps, best, ref.logp_bound(best), "logps")


@pytest.mark.parametrize("V", VOCABS)
def test_draw_among_neighbours_within_a_rounding(cuda_device, V):
    from gemma4_posttrain_jax_b200 import sample_top_k

    k, d, B = 20, 64, 16
    gen = torch.Generator(device=cuda_device).manual_seed(V + 1)
    W = torch.zeros((V, d), device=cuda_device)
    W[:, 0] = 1.0
    W[:, 1] = torch.rand((V,), generator=gen, device=cuda_device)
    H = torch.zeros((B, d), device=cuda_device)
    H[:, 0], H[:, 1] = 1.0, 2.0**-12
    W, H = W.to(torch.bfloat16), H.to(torch.bfloat16)
    u = (torch.arange(B, device=cuda_device) + 0.5) / B
    token, _ = sample_top_k(W, H, None, u, temperature=1.0, top_k=k, top_p=0.9)
    assert torch.equal(token.long(), Reference(W, H, None).draw(u, k, 1.0, 0.9))


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("k", [1, 20])
def test_every_token_the_same(cuda_device, V, k):
    from gemma4_posttrain_jax_b200 import top_token_logps

    gen = torch.Generator(device=cuda_device).manual_seed(3)
    row = torch.randn((1, 72), generator=gen, device=cuda_device).to(torch.bfloat16)
    W = row.expand(V, 72).contiguous()
    H = torch.randn((4, 72), generator=gen, device=cuda_device).to(torch.bfloat16)
    got = top_token_logps(W, H, None, k)
    assert torch.equal(got.ids.long(), torch.arange(k, device=cuda_device).expand(4, k))


@pytest.mark.parametrize("V", VOCABS)
def test_long_rows_that_cancel(cuda_device, V):
    """A few rows of the embedding a thousand times longer than the others, whose f32 sums are off by more
    than the others' whole spread, and whose exact ones are among the largest."""
    from gemma4_posttrain_jax_b200 import top_token_logps

    k, d = 12, 512
    gen = torch.Generator(device=cuda_device).manual_seed(V + 2)
    W = torch.randn((V, d), generator=gen, device=cuda_device) * 2.0**-8
    big = torch.randn((d // 2,), generator=gen, device=cuda_device).to(torch.bfloat16).float() * 16
    for i in (3, 30, 31, 700, 701, 1100):
        W[i, : d // 2] = big[torch.randperm(d // 2, generator=gen, device=cuda_device)]
        W[i, d // 2 :] = -big[torch.randperm(d // 2, generator=gen, device=cuda_device)]
        W[i, 0] += 1.0  # about 1 where the others are within +-0.5
    H = torch.ones((2, d), device=cuda_device)
    H[1] = -1.0
    W, H = W.to(torch.bfloat16), H.to(torch.bfloat16)
    got = top_token_logps(W, H, None, k)
    assert torch.equal(got.ids.long(), Reference(W, H, None).order(k))


@pytest.mark.parametrize("V", VOCABS)
def test_an_infinite_logit_is_not_left_out(cuda_device, V):
    """Under a softcap the row's other log-probabilities stay finite; the infinite score answers NaN."""
    from gemma4_posttrain_jax_b200 import top_token_logps

    k, at = 5, 1037
    gen = torch.Generator(device=cuda_device).manual_seed(V + 4)
    W = torch.randn((V, 64), generator=gen, device=cuda_device).to(torch.bfloat16)
    H = torch.randn((3, 64), generator=gen, device=cuda_device).to(torch.bfloat16)
    H[:, 9] = 1.0
    want = Reference(W, H, 30.0).order(k)
    W[at, 9] = float("inf")
    got = top_token_logps(W, H, 30.0, k)
    assert (got.ids[:, 0] == at).all() and got.logps[:, 0].isnan().all()
    for t in range(3):
        rest = [i for i in want[t].tolist() if i != at][: k - 1]
        assert got.ids[t, 1:].tolist() == rest
    assert got.logps[:, 1:].isfinite().all()
