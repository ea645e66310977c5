"""The given tokens' entries of the gradient with respect to the logits reach dH, and dW of few rows, without
a rounding of their own: what is left is the result's."""

from __future__ import annotations

import pytest
import torch

from tests.dist_reference import Reference, within

pytestmark = pytest.mark.gpu

# bf16 rounds 1 + 2^-8 by its largest step, 2^-8
STEP = 2.0**-8


def _grads(W, H, y, g, **options):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    W, H = W.clone().requires_grad_(True), H.clone().requires_grad_(True)
    logps, _ = token_logps_and_entropy(W, H, y, **options)
    return torch.autograd.grad([logps], [H, W], [g])


@pytest.mark.parametrize("T,V,d,token_chunk", [
    (1, 300, 64, None),
    (3, 1036, 160, None),
    (37, 70001, 72, None),
    (150, 1036, 136, None),
    (600, 4099, 64, None),  # more rows than dW is summed again for
    (200, 517, 64, 64),  # chunks of rows
])  # fmt: skip
@pytest.mark.parametrize("repeat", [False, True])
@pytest.mark.parametrize("keep", [True, False])
def test_gradients_that_only_given_tokens_have(cuda_device, T, V, d, token_chunk, repeat, keep):
    """Two tokens with opposite gradients a and -a: no other entry of the row has any, whatever its
    probabilities, so dH = a (W_1 - W_2), and dW the sum of the rows' a h in either token's row."""
    gen = torch.Generator(device=cuda_device).manual_seed(T + V)
    W = torch.randn((V, d), generator=gen, device=cuda_device).to(torch.bfloat16)
    H = (torch.randn((T, d), generator=gen, device=cuda_device) / d**0.5).to(torch.bfloat16)
    first = torch.randint(V, (T,), generator=gen, device=cuda_device)
    if T > 2:
        first[1::3] = first[0]  # a token that several rows share
    second = (first + 1 + torch.randint(V - 1, (T,), generator=gen, device=cuda_device)) % V
    a = (1 + STEP) * (1 + 2.0**-13 * (torch.rand((T,), generator=gen, device=cuda_device) - 0.5))
    none = torch.full_like(first, -1)
    y = torch.stack([first, none, second], 1)
    g = torch.stack([a, a, -a], 1)
    if repeat:  # one of them in two slots, with half of its gradient each
        y = torch.stack([first, second, first, none], 1)
        g = torch.stack([a / 2, -a, a / 2, a], 1)
    dH, dW = _grads(W, H, y, g, softcap=None, keep_logits=keep, token_chunk=token_chunk)
    w, h, a = W.double(), H.double(), a.double()
    want_H = a[:, None] * (w[first] - w[second])
    size_H = a[:, None] * (w[first].abs() + w[second].abs())
    # one rounding to bf16; f32 sums of two terms and of the product's zeros
    within(dH, want_H, 1.01 * STEP * want_H.abs() + 2**-22 * size_H, "d hidden")
    want_W = torch.zeros((V, d), dtype=torch.float64, device=cuda_device)
    want_W.index_add_(0, first, a[:, None] * h).index_add_(0, second, -a[:, None] * h)
    size_W = torch.zeros_like(want_W).index_add_(0, first, a[:, None] * h.abs()).index_add_(0, second, a[:, None] * h.abs())
    # where dW is not summed again its entries keep their rounding to bf16
    again = token_chunk is None and T * T * y.shape[1] <= 65536
    off = (T + 2) * 2**-24 * size_W if again else 1.01 * STEP * size_W
    within(dW, want_W, 1.01 * STEP * want_W.abs() + off + 1e-30, "d embedding")  # (rows of no token are exactly 0)
    assert (dW[(want_W == 0).all(1)] == 0).all()


@pytest.mark.parametrize("T", [1, 3, 11])
@pytest.mark.parametrize("keep", [True, False])
def test_one_token_per_row_beside_a_saturated_one(cuda_device, T, keep):
    """One given token of small probability beside one that has nearly all of it, far beyond the softcap, where
    its slope leaves it no gradient: dH = a (1 - p) slope W_y."""
    c, d, V = 30.0, 16 * T, 700
    gen = torch.Generator(device=cuda_device).manual_seed(T)
    H = torch.zeros((T, T, 16), device=cuda_device)
    rows = torch.arange(T, device=cuda_device)
    H[rows, rows] = torch.randint(1, 4, (T, 16), generator=gen, device=cuda_device).float()  # a block of its own each
    W = torch.randn((V, T, 16), generator=gen, device=cuda_device) / 16
    W[300 : 300 + T] = 0.0
    W[300 + rows, rows] = 64.0  # a logit of a thousand and more for its row
    W, H = W.reshape(V, d).to(torch.bfloat16), H.reshape(T, d).to(torch.bfloat16)
    y = torch.randint(0, 300, (T,), generator=gen, device=cuda_device)
    a = torch.full((T,), 1 + STEP - 2.0**-16, device=cuda_device)
    dH, dW = _grads(W, H, y, a, softcap=c, keep_logits=keep)
    ref = Reference(W, H, c)
    slope = 1 - (ref.z / c) ** 2
    at = y[:, None]
    dz = (slope * (torch.zeros_like(ref.p).scatter_(1, at, a.double()[:, None]) - ref.p * a.double()[:, None]))
    own = torch.zeros_like(dz).scatter_(1, at, 1.0)
    # the given entry in f32 (2^-18 covers its slope and probability); the others, whose probabilities are below
    # e^-20 but for the saturated one's, whose slope is below 2^-23, as they may be
    off = own * 2**-18 * dz.abs() + (1 - own) * (2 * dz.abs() + 2.0**-23 * ref.p * 1.01 * a.double()[:, None])
    want_H, want_W = dz @ W.double(), dz.T @ H.double()
    within(dH, want_H, 1.01 * STEP * want_H.abs() + off @ W.double().abs(), "d hidden")
    within(dW, want_W, 1.01 * STEP * want_W.abs() + off.T @ H.double().abs() + 1e-30, "d embedding")
