"""Calls of the distribution operators that their documentation allows and that are easily got wrong: under
capture, from other threads, on padded or masked inputs."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_completions_refuse_a_capture_and_their_replacement_is_captured(cuda_device):
    """What the refusal names gives the same numbers from a replayed graph, with another mask too."""
    from gemma4_posttrain_jax_b200 import completion_logps_and_entropy, token_logps_and_entropy

    B, S, N, V, d, prompt = 3, 20, 11, 1036, 64, 6
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    W = (torch.randn((V, d), generator=gen, device=cuda_device) / 8).to(torch.bfloat16).requires_grad_(True)
    H = torch.randn((B, S, d), generator=gen, device=cuda_device).to(torch.bfloat16)
    ids = torch.randint(V, (B, N), generator=gen, device=cuda_device)
    mask = torch.rand((B, N), generator=gen, device=cuda_device) < 0.6
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            completion_logps_and_entropy(W, H, ids, mask, prompt_width=prompt, softcap=30.0)

    def padded():
        rows = H[:, prompt - 1 : prompt - 1 + N]
        logps, entropy = token_logps_and_entropy(W, rows, torch.where(mask, ids, -1), softcap=30.0)
        return logps, torch.where(mask, entropy, 0.0)

    with torch.no_grad():
        padded()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logps, entropy = padded()
    for _ in range(2):
        graph.replay()
        want_logps, want_entropy = completion_logps_and_entropy(W, H, ids, mask, prompt_width=prompt, softcap=30.0)
        # the same products and formulas; compaction moves a row to another tile or launch shape, whose f32
        # sums of 1036 terms may be grouped otherwise: 2^-20 of sizes up to 32
        assert (logps - want_logps).abs().max() <= 32 * 2.0**-20 and (entropy - want_entropy).abs().max() <= 32 * 2.0**-20
        mask.copy_(torch.rand((B, N), generator=gen, device=cuda_device) < 0.4)


def _inputs(dev, T=150, V=2050, d=72, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    W = (torch.randn((V, d), generator=gen, device=dev) / d**0.5).to(torch.bfloat16)
    H = (torch.randn((T, d), generator=gen, device=dev) * 2).to(torch.bfloat16)
    y = torch.randint(V, (T, 3), generator=gen, device=dev)
    return W, H, y, gen


def test_inference_mode_gives_what_grad_mode_gives(cuda_device):
    from gemma4_posttrain_jax_b200 import completion_logps_and_entropy, sample_top_k, token_logps_and_entropy, top_token_logps

    W, H, y, gen = _inputs(cuda_device)
    u = torch.rand((H.shape[0],), generator=gen, device=cuda_device)
    mask = torch.rand((10, 9), generator=gen, device=cuda_device) < 0.5
    ids = y[:90, 0].reshape(10, 9)
    W.requires_grad_(True)

    def results():
        return (
            *token_logps_and_entropy(W, H, y, softcap=30.0, keep_logits=False),
            *completion_logps_and_entropy(W, H.reshape(10, 15, -1), ids, mask, prompt_width=4, softcap=30.0, keep_logits=False),
            *top_token_logps(W, H, 30.0, 9, tokens=y[:, 0]),
            *sample_top_k(W, H, 30.0, u, temperature=0.8, top_k=20, top_p=0.9),
        )

    want = results()
    with torch.inference_mode():
        got = results()
    with torch.no_grad():
        again = results()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


def test_checkpointed_and_offloaded_graphs(cuda_device):
    """The forward run again in the backward, and what it saves moved to the host in between."""
    from torch.utils.checkpoint import checkpoint

    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    W, H, y, gen = _inputs(cuda_device)
    W.requires_grad_(True), H.requires_grad_(True)
    g = torch.randn(y.shape, generator=gen, device=cuda_device)

    def loss(hidden):
        logps, entropy = token_logps_and_entropy(W, hidden * 1.0, y, softcap=30.0)
        return (logps * g).sum() + entropy.sum()

    want = torch.autograd.grad(loss(H), [H, W])
    for again in (lambda: checkpoint(loss, H, use_reentrant=False), lambda: checkpoint(loss, H, use_reentrant=True)):
        assert all(torch.equal(a, b) for a, b in zip(want, _grads(again(), [H, W])))
    with torch.autograd.graph.save_on_cpu():
        moved = loss(H)
    assert all(torch.equal(a, b) for a, b in zip(want, _grads(moved, [H, W])))


def _grads(value, leaves):
    for x in leaves:
        x.grad = None
    value.backward()
    return [x.grad for x in leaves]


def test_calls_from_several_threads_and_streams(cuda_device):
    import threading

    from gemma4_posttrain_jax_b200 import sample_top_k, token_logps_and_entropy, top_token_logps

    def work(seed):
        W, H, y, gen = _inputs(cuda_device, T=100 + 37 * seed, V=3000 + 1111 * seed, seed=seed)
        W.requires_grad_(True), H.requires_grad_(True)
        u = torch.rand((H.shape[0],), generator=gen, device=cuda_device)
        logps, entropy = token_logps_and_entropy(W, H, y, softcap=30.0)
        dH, dW = torch.autograd.grad(logps.sum() + entropy.sum(), [H, W])
        top = top_token_logps(W, H, 30.0, 12)
        return (logps.detach(), entropy.detach(), dH, dW, *top[:3], *sample_top_k(W, H, 30.0, u, temperature=1.0, top_k=12))

    want = [work(seed) for seed in range(4)]
    torch.cuda.synchronize()
    got, failed = [[] for _ in want], []

    def run(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(6):
                    got[seed].append(work(seed))
                torch.cuda.current_stream().synchronize()
        except Exception as exc:  # noqa: BLE001 - reported below
            failed.append(exc)

    threads = [threading.Thread(target=run, args=(seed,)) for seed in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(120)
    assert not failed and not any(thread.is_alive() for thread in threads)
    for seed, rounds in enumerate(got):
        assert len(rounds) == 6
        for one in rounds:
            assert all(torch.equal(a, b) for a, b in zip(one, want[seed]))


def test_gradients_that_are_views_or_absent(cuda_device):
    """Incoming gradients that autograd expands, and outputs of which one is not used."""
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    W, H, y, _ = _inputs(cuda_device)
    H.requires_grad_(True)
    ones = torch.ones(y.shape, device=cuda_device)
    logps, entropy = token_logps_and_entropy(W, H, y.to(torch.int16), softcap=None)
    (a,) = torch.autograd.grad([logps.sum()], [H], retain_graph=True)
    (b,) = torch.autograd.grad([logps], [H], [ones], retain_graph=True)
    (c,) = torch.autograd.grad([logps, entropy], [H], [ones, torch.zeros_like(entropy)], retain_graph=True)
    (e,) = torch.autograd.grad([logps], [H], [ones.T.contiguous().T], retain_graph=True)
    assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, e)
    (f,) = torch.autograd.grad([entropy.sum()], [H])
    assert f.isfinite().all() and (f != 0).any()


def test_captures_refuse_the_leaves_of_living_completions(cuda_device):
    """A graph of completions holds its hidden states as well as the embedding."""
    from gemma4_posttrain_jax_b200 import completion_logps_and_entropy, distribution, token_logps_and_entropy

    W, H, y, _ = _inputs(cuda_device)
    H = H.reshape(10, 15, -1)
    W.requires_grad_(True), H.requires_grad_(True)
    ids, mask = y[:90, 0].reshape(10, 9), torch.ones((10, 9), dtype=torch.bool, device=cuda_device)
    alive = completion_logps_and_entropy(W, H, ids, mask, prompt_width=4, softcap=30.0)
    assert distribution._eager_graphs.holds([W]) and distribution._eager_graphs.holds([H])
    fixed = W.detach()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            token_logps_and_entropy(fixed, H, y.reshape(10, 15, 3), softcap=30.0)
    del alive
    assert not distribution._eager_graphs.holds([W]) and not distribution._eager_graphs.holds([H])
