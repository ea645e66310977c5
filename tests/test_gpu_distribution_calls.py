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
