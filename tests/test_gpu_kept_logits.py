"""Gradients from logits kept in 16 bits, entry by entry, where a group of 32 neighbours holds logits of
every size: one far beyond the softcap on either side beside ordinary ones."""

from __future__ import annotations

import pytest
import torch

from tests.dist_reference import Reference, within

pytestmark = pytest.mark.gpu

LEAD = 4.0


def _one_position(dev, logits):
    """A head whose raw logits are ``logits``, each one exact product: the hidden state's only number that is
    not zero is LEAD, so that row v of dW is dZ_v times LEAD."""
    W = torch.zeros((len(logits), 8), device=dev)
    W[:, 3] = logits / LEAD
    H = torch.zeros((1, 8), dtype=torch.bfloat16, device=dev)
    H[0, 3] = LEAD
    return W.to(torch.bfloat16), H


def _dz_of(W, H, y, g, ge, softcap, keep):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    leaf = W.clone().requires_grad_(True)
    logps, entropy = token_logps_and_entropy(leaf, H, y, softcap=softcap, keep_logits=keep)
    (got,) = torch.autograd.grad([logps, entropy], [leaf], [g, ge])
    return got[:, 3].double() / LEAD


@pytest.mark.parametrize("softcap", [30.0, 100.0])
@pytest.mark.parametrize("far", [-8.5, -2.2, 2.2, None])  # of the softcap; 2.2: the target's neighbour saturates
@pytest.mark.parametrize("K", [1, 2])
@pytest.mark.parametrize("keep", [True, False])
def test_given_token_that_is_nearly_certain(cuda_device, softcap, far, K, keep):
    """g (1 - p) of a target with p near 1: what its logit is off by, 1 - p is off by the p / (1 - p) fold of."""
    V, target = 320, 37
    gen = torch.Generator(device=cuda_device).manual_seed(int(softcap) + K)
    logits = torch.randn((V,), generator=gen, device=cuda_device)
    logits[target] = 9.0 + 5.0
    if far is not None:
        logits[50] = far * softcap
    if far == 2.2:
        logits[target] = 3.0 * softcap  # and its neighbour less, both beyond the cap
    W, H = _one_position(cuda_device, logits)
    y = torch.tensor([[target, -1][:K]], device=cuda_device)
    g, ge = torch.tensor([[1.0, 1.0][:K]], device=cuda_device), torch.zeros((1,), device=cuda_device)
    got = _dz_of(W, H, y, g, ge, softcap, keep)[target]
    ref = Reference(W, H, softcap)
    p, z = ref.p[0, target], ref.z[0, target]
    slope = 1 - (z / softcap) ** 2
    want = slope * (1 - p)
    # two roundings to bf16; log p in f32, off by 2^-22 of z and of the cap (the softcap's two functions), moves
    # 1 - p by that times p; the slope, 1 - (z / c)^2 in f32, is off by 2^-21
    off = 2.02 * 2**-8 * want + slope * p * 2**-21 * (z.abs() + softcap + 1) + 2**-21 * (1 - p)
    within(got.reshape(1), want.reshape(1), off.reshape(1), "d logit of the target")


@pytest.mark.parametrize("softcap", [5.0, 30.0, 300.0])
@pytest.mark.parametrize("far", [-9.0, -2.5, 2.5])
@pytest.mark.parametrize("K", [1, 2])
@pytest.mark.parametrize("keep", [True, False])
def test_ordinary_logits_beside_a_saturated_one(cuda_device, softcap, far, K, keep):
    """One of every 32 neighbours is far beyond the softcap; the other 31 keep their accuracy."""
    V = 640
    gen = torch.Generator(device=cuda_device).manual_seed(int(softcap) + 11)
    logits = torch.randn((V,), generator=gen, device=cuda_device) * min(3.0, softcap / 4)
    logits[::32] = far * softcap
    ordinary = torch.arange(V, device=cuda_device) % 32 != 0
    W, H = _one_position(cuda_device, logits)
    y = torch.tensor([[70, -1][:K]], device=cuda_device)
    g, ge = torch.tensor([[1.5, 1.0][:K]], device=cuda_device), torch.tensor([0.5], device=cuda_device)
    got = _dz_of(W, H, y, g, ge, softcap, keep)
    ref = Reference(W, H, softcap)
    slope = 1 - (ref.z[0] / softcap) ** 2
    E, lp, p = ref.entropy[0], ref.logp[0], ref.p[0]
    hot = torch.zeros_like(p)
    hot[70] = 1.5
    want = slope * (hot - p * (1.5 + 0.5 * (lp + E)))
    # Two roundings to bf16. A logit kept in 15 bits over a range of 48 ln2 at most is off by half a step, 5.1e-4:
    # p by that of itself, log p by that, the slope, 1 - (z / c)^2, by 2 |z| / c^2 times that. f32's share: 2^-18.
    # What lies further below the group's largest than the range is at 2^-48 of it.
    half = 5.1e-4
    raw = hot + p * (1.5 + 0.5 * (lp.abs() + E))
    off = 2.02 * 2**-8 * want.abs() + slope * p * half * (1.5 + 0.5 * (lp.abs() + E) + 0.5)
    off = off + 2 * ref.z[0].abs() / softcap**2 * half * p * (1.5 + 0.5 * (lp.abs() + E)) + 2**-18 * raw
    off = off + 2**-47 * (1.5 + 0.5 * (40 + E)) + 1e-30
    within(got[ordinary], want[ordinary], off[ordinary], "d logits")
