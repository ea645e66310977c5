"""Several given tokens' log-probabilities with the entropy, the most likely tokens, and the top-k draw,
against the same in 64 bits (``dist_reference``)."""

from __future__ import annotations

import pytest
import torch

from tests.dist_reference import Reference, within

pytestmark = pytest.mark.gpu


def _inputs(dev, T, V, d, scale=1.0, seed=0, lift=6.0):
    gen = torch.Generator(device=dev).manual_seed(seed + 1000 * T + V)
    W = (torch.randn((V, d), generator=gen, device=dev) * (scale / d**0.5)).to(torch.bfloat16)
    H = torch.randn((T, d), generator=gen, device=dev)
    likely = torch.randint(V, (T,), generator=gen, device=dev)
    strength = torch.rand((T, 1), generator=gen, device=dev) * lift / scale**2
    return W, (H + strength * W[likely].float()).to(torch.bfloat16), gen


def _tokens(gen, dev, T, V, K, pad=True):
    y = torch.randint(V, (T, K), generator=gen, device=dev)
    if pad and K > 1:
        y[torch.rand((T, K), generator=gen, device=dev) < 0.3] = -1
        y[0] = V  # a row without any token
        y[-1, : K // 2 + 1] = y[-1, 0].clamp(0, V - 1)  # a token named several times
    return y


SHAPES = [
    (1, 1, 8, None),  # a vocabulary of one token: logp 0, entropy 0
    (1, 5, 8, 30.0),
    (3, 97, 64, None),  # less than one tile each way
    (37, 1036, 160, 30.0),
    (128, 256, 72, 3.0),  # exactly one tile, a narrow cap
    (129, 257, 64, None),  # one past the tile both ways: CTA pairs, a vocabulary tail of one column
    (513, 4099, 136, 30.0),
    (300, 70001, 64, 50.0),
]


@pytest.mark.parametrize("T,V,d,softcap", SHAPES)
@pytest.mark.parametrize("K", [None, 0, 1, 5])
def test_logps_and_entropy(cuda_device, T, V, d, softcap, K):
    from gemma4_posttrain_jax_b200 import _lib, token_logps_and_entropy

    W, H, gen = _inputs(cuda_device, T, V, d)
    y = _tokens(gen, cuda_device, T, V, 1 if K is None else K)
    logps, entropy = token_logps_and_entropy(W, H, y[:, 0] if K is None else y, softcap=softcap)
    assert logps.dtype == entropy.dtype == torch.float32
    assert logps.shape == ((T,) if K is None else (T, K)) and entropy.shape == (T,)
    ref = Reference(W, H, softcap)
    picked = ref.picked(y)
    within(logps.reshape(picked.shape), picked, ref.logp_bound(picked), "logps")
    within(entropy, ref.entropy, ref.entropy_bound(), "entropy")
    assert (logps <= 0).all() and (entropy >= 0).all()
    assert _lib.device_error(0) == 0


@pytest.mark.parametrize("T,V,d,softcap", SHAPES)
@pytest.mark.parametrize("K,send", [(1, "both"), (1, "logps"), (1, "entropy"), (5, "both"), (4, "logps"), (2, "entropy")])
@pytest.mark.parametrize("keep", [True, False])
def test_gradients(cuda_device, T, V, d, softcap, K, send, keep):
    from gemma4_posttrain_jax_b200 import _lib, token_logps_and_entropy

    W, H, gen = _inputs(cuda_device, T, V, d)
    y = _tokens(gen, cuda_device, T, V, K)
    g = torch.randn((T, K), generator=gen, device=cuda_device) if send != "entropy" else None
    ge = torch.randn((T,), generator=gen, device=cuda_device) if send != "logps" else None
    W.requires_grad_(True)
    H.requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, H, y, softcap=softcap, keep_logits=keep)
    loss = 0.0 if g is None else (logps * g).sum()
    loss = loss if ge is None else loss + (entropy * ge).sum()
    loss.backward()
    dH, dW, bH, bW = Reference(W.detach(), H.detach(), softcap, kept=keep).grads(y, g, ge)
    within(H.grad, dH, bH, "d hidden")
    within(W.grad, dW, bW, "d embedding")
    assert _lib.device_error(0) == 0


@pytest.mark.parametrize("softcap", [1.0, 5.0, 30.0, 100.0])
@pytest.mark.parametrize("K", [1, 2])
@pytest.mark.parametrize("keep", [True, False])
def test_gradients_of_saturated_logits(cuda_device, softcap, K, keep):
    """Logits far beyond the softcap, where its slope is small, one entry of dZ at a time: one position,
    whose hidden state has one number that is not zero, so that every logit is one exact product and
    row v of dW is dZ_v times that number."""
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    V, d, lead = 1037, 8, 4.0
    gen = torch.Generator(device=cuda_device).manual_seed(17)
    span = torch.rand((V,), generator=gen, device=cuda_device) * 2 - 1
    span[:256] = span[:256] * 0.4  # slopes that are not small
    span[256:320] = span[256:320].abs() * 0.3 + 0.7  # every one of 64 neighbours near the cap
    W = torch.zeros((V, d), device=cuda_device)
    W[:, 3] = span * 5 * softcap / lead
    W = W.to(torch.bfloat16).requires_grad_(True)
    H = torch.zeros((1, d), dtype=torch.bfloat16, device=cuda_device)
    H[0, 3] = lead
    z = Reference(W.detach(), H, softcap).z[0]
    for first in (int(z.argmax()), int(z.argmin()), 300, 7):
        y = torch.tensor([[first, 260][:K]], device=cuda_device)
        g = torch.tensor([[1.5, -0.75][:K]], device=cuda_device)
        ge = torch.tensor([0.25], device=cuda_device)
        logps, entropy = token_logps_and_entropy(W, H, y, softcap=softcap, keep_logits=keep)
        (got,) = torch.autograd.grad([logps, entropy], [W], [g, ge])
        ref = Reference(W.detach(), H, softcap)
        _, dW, _, _ = ref.grads(y, g, ge)
        slope = 1 - (ref.z[0] / softcap) ** 2
        hot = torch.zeros(V, dtype=torch.float64, device=cuda_device).index_add_(0, y[0], g[0].abs().double())
        raw = hot + ref.p[0] * (g.abs().sum() + ge.abs() * (ref.logp[0].abs() + ref.entropy))
        # Two roundings to bf16 (dZ and dW). A logit kept by its distance below the largest is off by
        # 24 ln2 / 65535 = 2.6e-4 at most, and p and log p by that; its slope is above 0.06 and off by
        # 2 / c of half a step, which is at most 2 * 1.53e-5 / 0.06 of it. Kept by y = 2 x / c in base 2,
        # in 65535 steps of at most 52.1, it is off by 4e-4 of y: the slope by ln2 * 4e-4, z by
        # c / 2 * ln2 * 4e-4 of the slope. f32's share is that of z / c, 2^-19 of 1.
        rel = 2.6e-4 * 2 + 5.1e-4 + 2.8e-4 + 2 * 1.4e-4 * softcap * slope + 2**-18
        far = 2**-47 * (g.abs().sum() + ge.abs() * (40 + ref.entropy))
        off = 2.02 * 2**-8 * dW[:, 3].abs() + lead * ((slope * rel + 2**-19) * raw + far) + 1e-30
        within(got[:, 3], dW[:, 3], off, f"d embedding, token {first}")


@pytest.mark.parametrize("frozen", ["embed", "hidden"])
@pytest.mark.parametrize("K", [1, 3])
@pytest.mark.parametrize("keep", [True, False])
def test_one_gradient_alone_and_row_chunks(cuda_device, frozen, K, keep):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    T, V, d = 700, 1036, 128
    W, H, gen = _inputs(cuda_device, T, V, d)
    y = _tokens(gen, cuda_device, T, V, K)
    g, ge = torch.randn((T, K), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
    leaf = (H if frozen == "embed" else W).requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0, token_chunk=256, keep_logits=keep)
    (got,) = torch.autograd.grad([logps, entropy], [leaf], [g, ge])
    dH, dW, bH, bW = Reference(W.detach(), H.detach(), 30.0, kept=keep).grads(y, g, ge)
    within(got, dH if frozen == "embed" else dW, bH if frozen == "embed" else bW, "gradient")


def test_many_tokens_per_position(cuda_device):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    T, V, d, K = 9, 300, 64, 256
    W, H, gen = _inputs(cuda_device, T, V, d)
    y = torch.randint(-40, V + 40, (T, K), generator=gen, device=cuda_device)  # many of them several times
    g, ge = torch.randn((T, K), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
    W.requires_grad_(True), H.requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0)
    ref = Reference(W.detach(), H.detach(), 30.0, kept=True)
    picked = ref.picked(y)
    within(logps, picked, ref.logp_bound(picked), "logps")
    dH, dW, bH, bW = ref.grads(y, g, ge)
    got = torch.autograd.grad([logps, entropy], [H, W], [g, ge])
    within(got[0], dH, bH, "d hidden")
    within(got[1], dW, bW, "d embedding")


def test_entropy_alone_and_a_graph_used_twice(cuda_device):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    T, V, d = 45, 1036, 64
    W, H, gen = _inputs(cuda_device, T, V, d)
    ge = torch.randn((T,), generator=gen, device=cuda_device)
    none = torch.empty((T, 0), dtype=torch.int64, device=cuda_device)
    W.requires_grad_(True), H.requires_grad_(True)
    _, entropy = token_logps_and_entropy(W, H, none, softcap=30.0)
    first = torch.autograd.grad([entropy], [H, W], [ge], retain_graph=True)
    dH, dW, bH, bW = Reference(W.detach(), H.detach(), 30.0, kept=True).grads(none, None, ge)
    within(first[0], dH, bH, "d hidden")
    within(first[1], dW, bW, "d embedding")
    again = torch.autograd.grad([entropy], [H, W], [ge], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    # gradients of gradients are refused, where they are asked for
    (once,) = torch.autograd.grad([entropy], [H], [ge], create_graph=True)
    assert torch.equal(once, first[0])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        once.float().sum().backward()
    with torch.no_grad():
        W.mul_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([entropy], [H, W], [ge])


@pytest.mark.parametrize("group", [1, 2])
def test_either_cta_group(cuda_device, group):
    """Every product as single CTAs and as pairs, whatever the sizes would choose."""
    from gemma4_posttrain_jax_b200 import _lib, token_logps_and_entropy, top_token_logps

    try:
        _lib.set_cta_group(group)
        for T, V in ((5, 300), (130, 4099), (257, 9001)):
            for keep in (True, False):
                W, H, gen = _inputs(cuda_device, T, V, 72)
                y = _tokens(gen, cuda_device, T, V, 2)
                g, ge = torch.randn((T, 2), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
                W.requires_grad_(True), H.requires_grad_(True)
                logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0, keep_logits=keep)
                got = torch.autograd.grad([logps, entropy], [H, W], [g, ge])
                ref = Reference(W.detach(), H.detach(), 30.0, kept=keep)
                dH, dW, bH, bW = ref.grads(y, g, ge)
                within(got[0], dH, bH, "d hidden")
                within(got[1], dW, bW, "d embedding")
            top = top_token_logps(W, H, 30.0, 6)
            assert torch.equal(top.ids.long(), ref.order(6))
            within(top.entropy, ref.entropy, ref.entropy_bound(), "entropy")
    finally:
        _lib.set_cta_group(0)


class _OneOfMany:
    """A vocabulary mesh of ``size`` ranks, this one ``rank``; the test plays the collectives."""

    axis_names = ("d",)

    def __init__(self, size, rank):
        self.size, self.rank = size, rank


def test_vocabulary_mesh(cuda_device, monkeypatch):
    """Every rank's call in turn, with the all-gather played from all shards' statistics: each rank has
    the whole vocabulary's results and its own rows of dW, and the ranks' dH add up."""
    from gemma4_posttrain_jax_b200 import distribution, ops, token_logps_and_entropy

    T, V, d, K, P = 67, 1040, 128, 4, 4
    W, H, gen = _inputs(cuda_device, T, V, d)
    y = _tokens(gen, cuda_device, T, V, K)
    g, ge = torch.randn((T, K), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
    vs = V // P
    tokens = y.to(torch.int32).contiguous()

    def gathered(own, mesh):
        parts = [ops.dist_forward_shard(W[p * vs : (p + 1) * vs], H, tokens, 30.0, p * vs) for p in range(P)]
        parts = torch.stack([torch.cat([s.reshape(-1), z.reshape(-1)]) for s, z in parts])
        assert torch.equal(parts[mesh.rank], own)
        return parts

    monkeypatch.setattr(distribution, "all_gather_stats", gathered)
    monkeypatch.setattr(distribution, "all_reduce_sum", lambda t, mesh: t)  # leaves the rank's partial sum
    monkeypatch.setattr(distribution, "_SKIP_MIN_FLOPS", 0.0)
    off = torch.arange(T, device=cuda_device) % 3 == 0
    g[off], ge[off] = 0.0, 0.0
    ref = Reference(W, H, 30.0, kept=True)
    dH, dW, bH, bW = ref.grads(y, g, ge)
    total = torch.zeros_like(dH)
    for rank in range(P):
        shard = W[rank * vs : (rank + 1) * vs].clone().requires_grad_(True)
        leaf = H.clone().requires_grad_(True)
        logps, entropy = token_logps_and_entropy(shard, leaf, y, softcap=30.0, mesh=_OneOfMany(P, rank), dh_reduce_f32=True)
        picked = ref.picked(y)
        within(logps, picked, ref.logp_bound(picked), "logps")
        within(entropy, ref.entropy, ref.entropy_bound(), "entropy")
        got_H, got_W = torch.autograd.grad([logps, entropy], [leaf, shard], [g, ge])
        within(got_W, dW[rank * vs : (rank + 1) * vs], bW[rank * vs : (rank + 1) * vs], "d embedding")
        total += got_H.double()
    # each rank rounded its partial sum to bf16 once: 2^-8 of sizes that the bound's first term covers
    within(total, dH, P * bH, "d hidden")


def test_completions(cuda_device):
    from gemma4_posttrain_jax_b200 import completion_logps_and_entropy

    B, S, N, V, d, prompt = 5, 40, 23, 1036, 64, 12
    W, H, gen = _inputs(cuda_device, B * S, V, d)
    H = H.reshape(B, S, d)
    ids = torch.randint(V, (B, N), generator=gen, device=cuda_device)
    mask = torch.arange(N, device=cuda_device) < torch.tensor([23, 7, 0, 1, 15], device=cuda_device)[:, None]
    g, ge = torch.randn((B, N), generator=gen, device=cuda_device), torch.randn((B, N), generator=gen, device=cuda_device)
    W.requires_grad_(True)
    flat = H[:, prompt - 1 : prompt - 1 + N].reshape(-1, d)
    on = mask.reshape(-1)
    ref = Reference(W.detach(), flat[on], 30.0, kept=True)
    y = ids.reshape(-1)[on][:, None]
    dH, dW, bH, bW = ref.grads(y, g.reshape(-1)[on][:, None], ge.reshape(-1)[on])
    wide = torch.nn.functional.pad(H, (0, 4))[..., :d]  # rows that have to be copied first
    for hidden in (H.clone(), wide.detach()):
        hidden.requires_grad_(True)
        logps, entropy = completion_logps_and_entropy(W, hidden, ids, mask, prompt_width=prompt, softcap=30.0)
        assert logps.shape == entropy.shape == (B, N)
        assert (logps[~mask] == 0).all() and (entropy[~mask] == 0).all()
        picked = ref.picked(y)
        within(logps[mask][:, None], picked, ref.logp_bound(picked), "logps")
        within(entropy[mask], ref.entropy, ref.entropy_bound(), "entropy")
        got_H, got_W = torch.autograd.grad([logps, entropy], [hidden, W], [g, ge])
        rows = got_H[:, prompt - 1 : prompt - 1 + N].reshape(-1, d)
        within(rows[on], dH, bH, "d hidden")
        assert (rows[~on] == 0).all() and got_H.abs().sum() == rows.abs().sum()
        within(got_W, dW, bW, "d embedding")
    # no completion token at all
    logps, entropy = completion_logps_and_entropy(W, H, ids, torch.zeros_like(mask), prompt_width=prompt, softcap=30.0)
    assert (logps == 0).all() and (entropy == 0).all()
    (got_W,) = torch.autograd.grad([logps.sum() + entropy.sum()], [W])
    assert (got_W == 0).all()


def test_gradient_against_differences(cuda_device):
    """Central differences of the operator itself, along directions that bf16 holds exactly: hidden
    entries are multiples of 2^-2 below 4 and the step is 2^-6, so h +- step needs 8 bits."""
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    T, V, d, step = 33, 517, 64, 2.0**-6
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    H = (torch.randint(-7, 8, (T, d), generator=gen, device=cuda_device).float() / 4).to(torch.bfloat16)
    H = torch.where(H == 0, torch.ones_like(H), H)
    W = (torch.randn((V, d), generator=gen, device=cuda_device) * 0.2).to(torch.bfloat16)
    y = _tokens(gen, cuda_device, T, V, 3)
    g, ge = torch.randn((T, 3), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)

    def rows(h):
        logps, entropy = token_logps_and_entropy(W, h, y, softcap=20.0)
        return (logps * g).sum(-1).double() + (entropy * ge).double()

    leaf = H.clone().requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, leaf, y, softcap=20.0)
    (grad,) = torch.autograd.grad([logps, entropy], [leaf], [g, ge])
    for _ in range(4):
        way = torch.randint(0, 2, (T, d), generator=gen, device=cuda_device).float() * 2 - 1
        up, down = (H.float() + step * way).to(torch.bfloat16), (H.float() - step * way).to(torch.bfloat16)
        assert torch.equal(up.float() - down.float(), 2 * step * way)
        slope = (rows(up) - rows(down)) / (2 * step)
        along = (grad.double() * way.double()).sum(-1)
        # f32 results of size <= 40 (off by 2^-20 of it) over 2 * step; third-order term of a
        # direction that moves logits by <= 0.2 * 8 * 2^-6 * 4 sigma; bf16 gradients (2 * 2^-8)
        size = (grad.double().abs()).sum(-1)
        off = (slope - along).abs()
        assert (off <= 40 * 2.0**-20 / step + 2 * 2.0**-8 * size + 0.01 * (g.abs().sum(-1) + ge.abs())).all(), off.max()


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("send", ["both", "logps", "entropy"])
def test_rows_without_gradient_are_left_out(cuda_device, monkeypatch, keep, send):
    from gemma4_posttrain_jax_b200 import distribution, token_logps_and_entropy

    T, V, d = 300, 1036, 64
    W, H, gen = _inputs(cuda_device, T, V, d)
    y = _tokens(gen, cuda_device, T, V, 2)
    g, ge = torch.randn((T, 2), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
    off = torch.rand((T,), generator=gen, device=cuda_device) < 0.4
    g[off], ge[off] = 0.0, 0.0
    ge[3], g[3] = 0.0, torch.tensor([0.0, 1.0], device=cuda_device)  # one of several gradients is enough
    if send == "logps":
        ge.zero_()
    elif send == "entropy":
        g.zero_()
    W.requires_grad_(True), H.requires_grad_(True)
    results = []
    for least in (float("inf"), 0.0):
        monkeypatch.setattr(distribution, "_SKIP_MIN_FLOPS", least)
        logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0, keep_logits=keep)
        sent = {"both": ([logps, entropy], [g, ge]), "logps": ([logps], [g]), "entropy": ([entropy], [ge])}[send]
        results.append(torch.autograd.grad(sent[0], [H, W], sent[1]))
    dH, dW, bH, bW = Reference(W.detach(), H.detach(), 30.0, kept=keep).grads(y, g, ge)
    for got_H, got_W in results:
        within(got_H, dH, bH, "d hidden")
        within(got_W, dW, bW, "d embedding")
        assert (got_H[off] == 0).sum() >= (off.sum() - 1) * d
    # no gradient at all
    logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0)
    zeros = torch.autograd.grad([logps, entropy], [H, W], [torch.zeros_like(g), torch.zeros_like(ge)])
    assert all((x == 0).all() for x in zeros)


@pytest.mark.parametrize("V,P", [(1040, 4), (4098, 2)])
@pytest.mark.parametrize("keep", [True, False])
def test_shards_merge_to_the_whole(cuda_device, V, P, keep):
    """One GPU plays every rank of a vocabulary mesh in turn: the merged statistics and the summed
    partial gradients are the whole vocabulary's."""
    from gemma4_posttrain_jax_b200 import ops

    T, d, K = 67, 128, 4
    W, H, gen = _inputs(cuda_device, T, V, d)
    W[V // P] *= 40  # one shard's maximum far above the others'
    y = _tokens(gen, cuda_device, T, V, K).to(torch.int32).contiguous()
    g, ge = torch.randn((T, K), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
    ref = Reference(W, H, 30.0, kept=keep)
    vs = V // P
    shards = [W[p * vs : (p + 1) * vs] for p in range(P)]
    logp, entropy = torch.empty((T, K), device=cuda_device), torch.empty((T,), device=cuda_device)
    saved, kept = zip(*[ops.dist_saved(T, K, vs, 1e9 if keep else 0, cuda_device) for _ in range(P)])
    assert all(k == ops.dist_kept(s, T, K) for s, k in zip(saved, kept))
    parts = [ops.dist_forward_shard(w, H, y, 30.0, p * vs, kept[p]) for p, w in enumerate(shards)]
    for one in saved:
        ops.dist_combine(torch.stack([s for s, _ in parts]), torch.stack([z for _, z in parts]), y, V, logp, entropy, one)
    picked = ref.picked(y)
    within(logp, picked, ref.logp_bound(picked), "logps")
    within(entropy, ref.entropy, ref.entropy_bound(), "entropy")
    grads = [
        ops.dist_backward(w, 30.0, H, y, saved[p], entropy, g, ge, vocab_offset=p * vs, vocab=V, dh_dtype=torch.float32,
                          kept=kept[p])
        for p, w in enumerate(shards)
    ]
    dH, dW, bH, bW = ref.grads(y, g, ge)
    within(sum(a for a, _ in grads), dH, bH, "d hidden")
    within(torch.cat([b for _, b in grads]), dW, bW, "d embedding")


def test_logits_far_below_the_largest(cuda_device):
    """Kept logits reach 2^-48 of the largest of their 32 columns: what lies lower has no gradient to
    speak of, and where all of a row's mass is elsewhere, a group's own scale still holds."""
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    T, V, d = 64, 640, 64
    W, H, gen = _inputs(cuda_device, T, V, d)
    W[32:64] *= 30  # logits of +-100 next to one another
    W[100] *= 60
    y = _tokens(gen, cuda_device, T, V, 3)
    g, ge = torch.randn((T, 3), generator=gen, device=cuda_device), torch.randn((T,), generator=gen, device=cuda_device)
    W.requires_grad_(True), H.requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, H, y, softcap=None, keep_logits=True)
    got_H, got_W = torch.autograd.grad([logps, entropy], [H, W], [g, ge])
    dH, dW, bH, bW = Reference(W.detach(), H.detach(), None, kept=True).grads(y, g, ge)
    within(got_H, dH, bH, "d hidden")
    within(got_W, dW, bW, "d embedding")


def test_shapes_strides_and_empty_batches(cuda_device):
    from gemma4_posttrain_jax_b200 import sample_top_k, token_logps_and_entropy, top_token_logps

    W, H, gen = _inputs(cuda_device, 24, 517, 64)
    y = torch.randint(517, (2, 3, 4), generator=gen, device=cuda_device)
    h = H.reshape(2, 3, 4, 64)
    ref = token_logps_and_entropy(W, H, y.reshape(24), softcap=30.0)
    for hidden in (
        h,
        h.transpose(0, 1).contiguous().transpose(0, 1),  # another order of the batch axes
        torch.cat([h, h], -1)[..., :64],  # a row stride of two rows
        torch.nn.functional.pad(h, (3, 5))[..., 3:67],  # rows that are not 16-byte aligned
        h.mT.contiguous().mT,  # columns not adjacent
    ):
        got = token_logps_and_entropy(W, hidden, y, softcap=30.0)
        assert got[0].shape == y.shape and got[1].shape == y.shape
        assert torch.equal(got[0].reshape(24), ref[0]) and torch.equal(got[1].reshape(24), ref[1])
        top = top_token_logps(W, hidden, 30.0, 3, tokens=y)
        assert top.ids.shape == top.logps.shape == (2, 3, 4, 3) and top.token_logps.shape == y.shape
    # every row the same memory; its gradient is the sum
    one = H[:1].clone().requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, one.expand(5, 64), y.reshape(-1)[:5], softcap=30.0)
    (grad,) = torch.autograd.grad([logps.sum() + entropy.sum()], [one])
    many = H[:1].expand(5, 64).clone().requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, many, y.reshape(-1)[:5], softcap=30.0)
    (rows,) = torch.autograd.grad([logps.sum() + entropy.sum()], [many])
    assert torch.equal(grad, rows.sum(0, keepdim=True))
    # nothing to do
    leaf, none = W.clone().requires_grad_(True), H[:0].clone().requires_grad_(True)
    logps, entropy = token_logps_and_entropy(leaf, none, y.reshape(-1)[:0], softcap=30.0)
    assert logps.shape == entropy.shape == (0,)
    got = torch.autograd.grad([logps.sum() + entropy.sum()], [leaf, none])
    assert (got[0] == 0).all() and got[1].shape == (0, 64)
    assert top_token_logps(W, H[:0], None, 2).ids.shape == (0, 2)
    token, logp = sample_top_k(W, H[:0], None, torch.empty(0, device=cuda_device), temperature=1.0, top_k=2)
    assert token.shape == logp.shape == (0,)
    # the last axis of hidden alone: one position
    logps, entropy = token_logps_and_entropy(W, H[0], y[0, 0, 0], softcap=30.0)
    assert logps.shape == entropy.shape == () and torch.equal(logps, ref[0][0])


TOP_SHAPES = [
    (1, 1, 8, 1, None),
    (2, 130, 64, 128, 30.0),
    (1, 128, 64, 128, None),  # every token
    (19, 4099, 136, 5, None),
    (5, 9000, 64, 128, 30.0),
    (37, 1036, 160, 20, 30.0),
    (129, 70001, 64, 64, 50.0),
    (3, 262144, 256, 40, 30.0),
    (140, 33000, 72, 100, None),
    (2, 1600000, 8, 3, None),  # more keys than shared memory holds
    (3, 5000, 6000, 7, 30.0),  # wide rows
]


@pytest.mark.parametrize("T,V,d,k,softcap", TOP_SHAPES)
def test_top_tokens(cuda_device, T, V, d, k, softcap):
    from gemma4_posttrain_jax_b200 import _lib, top_token_logps

    W, H, gen = _inputs(cuda_device, T, V, d)
    if V > 700:
        W[V // 3 : V // 3 + 40] *= 1.5  # likely tokens next to one another
    y = torch.randint(V, (T,), generator=gen, device=cuda_device)
    y[0] = -1
    got = top_token_logps(W, H, softcap, k, tokens=y)
    assert got.ids.dtype == torch.int32
    ref = Reference(W, H, softcap)
    assert torch.equal(got.ids.long(), ref.order(k))
    best = ref.logp.gather(1, ref.order(k))
    within(got.logps, best, ref.logp_bound(best), "logps")
    within(got.entropy, ref.entropy, ref.entropy_bound(), "entropy")
    picked = ref.picked(y[:, None])
    within(got.token_logps[:, None], picked, ref.logp_bound(picked), "token logps")
    assert _lib.device_error(0) == 0


@pytest.mark.parametrize("V", [3001, 60000])
def test_top_tokens_of_equal_logits(cuda_device, V):
    """Equal rows of the embedding give equal logits: the lowest ids come first. A hidden state of
    zeros makes all of them equal."""
    from gemma4_posttrain_jax_b200 import top_token_logps

    d, k = 64, 50
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    W = torch.randn((V, d), generator=gen, device=cuda_device).to(torch.bfloat16)
    H = torch.randn((6, d), generator=gen, device=cuda_device).to(torch.bfloat16)
    H[1] = 0
    same = torch.randperm(V, generator=gen, device=cuda_device)[:600].sort().values
    W[same] = W[same[0]].clone()
    H[2] = W[same[0]]  # 600 tokens share the largest logit
    H[3] = -W[same[0]]  # and the smallest
    got = top_token_logps(W, H, None, k)
    ref = Reference(W, H, None)
    assert torch.equal(got.ids.long(), ref.order(k))
    assert got.ids[1].tolist() == list(range(k))
    assert torch.equal(got.ids[2].long(), same[:k])


def test_near_ties_follow_the_exact_order(cuda_device):
    """Dot products that differ by less than an f32 accumulation resolves are still ranked exactly."""
    from gemma4_posttrain_jax_b200 import top_token_logps

    V, d, k = 2048, 256, 12
    W = torch.zeros((V, d))
    W[:, 0] = 256.0  # a common large part, then a difference of j * 2^-20 each
    ids = torch.arange(0, 1024, 128)
    W[:, 1] = -2.0
    W[ids, 1] = 0.0
    for j, i in enumerate(ids.tolist()):
        W[i, 2] = (j * 5 % 8) * 2.0**-20
    W = W.to(torch.bfloat16).to(cuda_device)
    H = torch.ones((2, d), dtype=torch.bfloat16, device=cuda_device)
    got = top_token_logps(W, H, None, k)
    assert torch.equal(got.ids.long(), Reference(W, H, None).order(k))
    assert len(set(got.ids[0, :8].tolist()) & set(ids.tolist())) == 8


def test_ties_near_zero(cuda_device):
    """Equal dot products near 0 whose f32 sums differ, with the k-th place among them and larger ones
    before: the lowest ids come first."""
    from gemma4_posttrain_jax_b200 import top_token_logps

    V, d, k = 64, 1024, 12
    gen = torch.Generator().manual_seed(5)
    W = torch.zeros((V, d))
    # of sizes from 2^-16 to 2^6, whose sums f32 rounds
    part = torch.randn((256,), generator=gen) * 2.0 ** torch.randint(-16, 6, (256,), generator=gen)
    part = part.to(torch.bfloat16).float()
    W[:, :256] = part
    # seven rows of the same numbers in other places, which sum to 0 exactly
    some = [5, 9, 17, 33, 40, 51, 60]
    for i in some:
        W[i, :256] = part[torch.randperm(256, generator=gen)]
    W[:, 256:512] = -part
    W[:, 512] = -1.0
    W[some, 512] = 0.0
    W[torch.tensor([2, 3, 21, 22, 23, 24, 50, 63]), 512] = torch.arange(8) * 4.0 + 16.0
    H = torch.ones((1, d), dtype=torch.bfloat16, device=cuda_device)
    W = W.to(torch.bfloat16).to(cuda_device)
    got = top_token_logps(W, H, None, k)
    assert torch.equal(got.ids.long(), Reference(W, H, None).order(k))
    assert got.ids[0, 8:].tolist() == some[:4]


def test_rows_with_nan_stay_apart(cuda_device):
    """A row with a NaN answers NaN, with ids of the vocabulary, and leaves the other rows alone."""
    from gemma4_posttrain_jax_b200 import sample_top_k, token_logps_and_entropy, top_token_logps

    for V in (517, 20000):
        W, H, gen = _inputs(cuda_device, 9, V, 64)
        clean, y = H.clone(), torch.arange(9, device=cuda_device)
        H[4, 7] = float("nan")
        u = torch.full((9,), 0.5, device=cuda_device)
        keep = torch.arange(9, device=cuda_device) != 4
        for got, ref in (
            (token_logps_and_entropy(W, H, y, softcap=30.0), token_logps_and_entropy(W, clean, y, softcap=30.0)),
            (top_token_logps(W, H, 30.0, 7, tokens=y), top_token_logps(W, clean, 30.0, 7, tokens=y)),
            (sample_top_k(W, H, 30.0, u, temperature=1.0, top_k=7), sample_top_k(W, clean, 30.0, u, temperature=1.0, top_k=7)),
        ):
            for a, b in zip(got, ref):
                assert torch.equal(a[keep], b[keep])
                if a.dtype == torch.int32:
                    assert ((a[4] >= 0) & (a[4] < V)).all() and a[4].unique().numel() == a[4].numel()
                else:
                    assert a[4].isnan().all()


def test_infinite_scores_are_not_passed_off_as_finite(cuda_device):
    """Infinite dot products, which a softcap would bring back to +-c, answer NaN."""
    from gemma4_posttrain_jax_b200 import sample_top_k, top_token_logps

    for V in (517, 20000):
        W, H, gen = _inputs(cuda_device, 5, V, 64)
        clean = H.clone()
        H[2, 9] = float("inf")
        u = torch.full((5,), 0.5, device=cuda_device)
        keep = torch.arange(5, device=cuda_device) != 2
        for got, ref in (
            (top_token_logps(W, H, 30.0, 7)[:2], top_token_logps(W, clean, 30.0, 7)[:2]),
            (sample_top_k(W, H, 30.0, u, temperature=1.0, top_k=7), sample_top_k(W, clean, 30.0, u, temperature=1.0, top_k=7)),
        ):
            assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, ref))
            assert ((got[0][2] >= 0) & (got[0][2] < V)).all() and got[1][2].isnan().all()


def test_more_rows_than_one_launch(cuda_device):
    from gemma4_posttrain_jax_b200 import top_token_logps

    T, V, d, k = 1100, 262144, 64, 3
    W, H, gen = _inputs(cuda_device, T, V, d)
    y = torch.randint(V, (T,), generator=gen, device=cuda_device)
    got = top_token_logps(W, H, 30.0, k, tokens=y)
    for rows in (slice(0, 40), slice(1000, 1100)):
        ref = Reference(W, H[rows], 30.0)
        assert torch.equal(got.ids[rows].long(), ref.order(k))
        within(got.entropy[rows], ref.entropy, ref.entropy_bound(), "entropy")
        picked = ref.picked(y[rows, None])
        within(got.token_logps[rows, None], picked, ref.logp_bound(picked), "token logps")


@pytest.mark.parametrize("B,V,d,k,temperature,top_p,softcap", [
    (1, 5, 8, 5, 1.0, 1.0, None),
    (200, 1036, 64, 20, 0.7, 0.9, 30.0),
    (130, 70001, 64, 64, 1.0, 0.95, 30.0),
    (64, 262144, 128, 128, 1.5, 1.0, None),
    (33, 300, 64, 128, 0.3, 0.5, 15.0),
    (7, 4099, 64, 1, 1.0, 1.0, None),
])  # fmt: skip
def test_sampled_tokens(cuda_device, B, V, d, k, temperature, top_p, softcap):
    from gemma4_posttrain_jax_b200 import _lib, sample_top_k

    W, H, gen = _inputs(cuda_device, B, V, d)
    u = torch.rand((B,), generator=gen, device=cuda_device)
    u[0] = 0.0
    u[-1] = 1.0 - 2.0**-24
    token, logp = sample_top_k(W, H, softcap, u, temperature=temperature, top_k=k, top_p=top_p)
    assert token.dtype == torch.int32 and logp.dtype == torch.float32
    ref = Reference(W, H, softcap)
    assert torch.equal(token.long(), ref.draw(u, k, temperature, top_p))
    picked = ref.picked(token[:, None].long())
    within(logp[:, None], picked, ref.logp_bound(picked), "logp")
    greedy, _ = sample_top_k(W, H, softcap, u, temperature=temperature, top_k=k, top_p=1e-7)
    assert torch.equal(greedy.long(), ref.order(1)[:, 0])
    assert _lib.device_error(0) == 0


def test_sampled_distribution(cuda_device):
    """Evenly spaced numbers draw every kept token in proportion to its weight."""
    from gemma4_posttrain_jax_b200 import sample_top_k

    n, V, d, k = 4096, 300, 64, 10
    W, H, _ = _inputs(cuda_device, 1, V, d, seed=4)
    u = (torch.arange(n, device=cuda_device) + 0.5) / n
    token, _ = sample_top_k(W, H.expand(n, d), None, u, temperature=0.8, top_k=k, top_p=0.9)
    ref = Reference(W, H, None)
    ids = ref.order(k)[0]
    w = ((ref.z[0, ids] - ref.z[0, ids[0]]) / 0.8).exp()
    w = torch.where(w.cumsum(0) - w < 0.9 * w.sum(), w, 0.0)
    share = torch.bincount(token.long(), minlength=V)[ids].double() / n
    assert torch.bincount(token.long(), minlength=V).sum() == (share.sum() * n).round()
    assert ((share - w / w.sum()).abs() <= 2.0 / n).all()


def test_results_repeat_bit_for_bit(cuda_device):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy, top_token_logps

    W, H, gen = _inputs(cuda_device, 777, 9001, 128)
    y = _tokens(gen, cuda_device, 777, 9001, 4)
    W.requires_grad_(True), H.requires_grad_(True)

    def once():
        logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0)
        return (logps, entropy, *torch.autograd.grad(logps.sum() + entropy.sum(), [H, W]), *top_token_logps(W, H, 30.0, 9)[:3])

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_captured_graphs(cuda_device):
    """Forward, backward, selection and draw in two captured graphs, replayed in turn and with new
    inputs. Over a living eager graph of the same leaves the call is refused."""
    from gemma4_posttrain_jax_b200 import sample_top_k, token_logps_and_entropy, top_token_logps

    T, V, d, k = 70, 5003, 64, 8
    W, H, gen = _inputs(cuda_device, T, V, d)
    y = _tokens(gen, cuda_device, T, V, 3)
    u = torch.rand((T,), generator=gen, device=cuda_device)
    W.requires_grad_(True), H.requires_grad_(True)

    def work():
        logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0)
        dH, dW = torch.autograd.grad(logps.sum() + entropy.sum(), [H, W])
        top = top_token_logps(W, H, 30.0, k)
        return (logps.detach(), entropy.detach(), dH, dW, *top[:3], *sample_top_k(W, H, 30.0, u, temperature=0.9, top_k=k))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    alive = token_logps_and_entropy(W, H, y, softcap=30.0)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            token_logps_and_entropy(W, H, y, softcap=30.0)
    with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():  # nothing to differentiate
        token_logps_and_entropy(W, H, y, softcap=30.0)
    del alive
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work())
    for step in range(3):
        with torch.no_grad():
            H.add_(0.25 * torch.randn((T, d), generator=gen, device=cuda_device).to(torch.bfloat16))
            u.uniform_(generator=gen)
        for graph in graphs:
            graph.replay()
        want = work()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once(cuda_device):
    from gemma4_posttrain_jax_b200 import top_token_logps

    sets = [_inputs(cuda_device, 200, 30000 + 77 * i, 256, seed=i)[:2] for i in range(2)]
    want = [top_token_logps(W, H, 30.0, 20) for W, H in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, (stream, (W, H)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append(top_token_logps(W, H, 30.0, 20))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one[:3], want[i][:3]))


def test_distillation_and_rollout_together(cuda_device):
    """As they are used: the policy draws tokens; a teacher scores them and names its alternatives;
    the student's loss takes the alternatives' log-probabilities and an entropy bonus."""
    from gemma4_posttrain_jax_b200 import per_token_logps, sample_top_k, token_logps_and_entropy, top_token_logps

    T, V, d, k = 90, 2050, 128, 16
    W, H, gen = _inputs(cuda_device, T, V, d)
    teacher = (H.float() + 0.3 * torch.randn((T, d), generator=gen, device=cuda_device)).to(torch.bfloat16)
    u = torch.rand((T,), generator=gen, device=cuda_device)
    token, logp = sample_top_k(W, H, 30.0, u, temperature=1.0, top_k=k)
    alternatives = top_token_logps(W, teacher, 30.0, k, tokens=token)
    weight = alternatives.logps.exp()
    W.requires_grad_(True), H.requires_grad_(True)
    logps, entropy = token_logps_and_entropy(W, H, alternatives.ids, softcap=30.0)
    loss = (weight * (alternatives.logps - logps)).sum() - 0.1 * entropy.sum()
    dH, dW = torch.autograd.grad(loss, [H, W])
    ref = Reference(W.detach(), H.detach(), 30.0, kept=True)
    rH, rW, bH, bW = ref.grads(alternatives.ids.long(), -weight, torch.full((T,), -0.1, device=cuda_device))
    within(dH, rH, bH, "d hidden")
    within(dW, rW, bW, "d embedding")
    # the draw's, the given token's and per_token_logps' log-probabilities are the same quantity
    again = per_token_logps(W.detach(), H.detach(), token, softcap=30.0)
    bound = ref.logp_bound(ref.picked(token[:, None].long()))[:, 0]
    assert ((again - logp).abs() <= 2 * bound).all()
    own = top_token_logps(W.detach(), H.detach(), 30.0, k, tokens=token)
    # (each is within its bound of the exact value; their epilogues sum in different orders)
    again, _ = token_logps_and_entropy(W.detach(), H.detach(), token, softcap=30.0)
    assert ((again - own.token_logps).abs() <= 2 * bound).all()
