"""Refusals of the distribution operators, none of which reaches a GPU."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from gemma4_posttrain_jax_b200 import (
    _lib,
    build,
    completion_logps_and_entropy,
    distribution,
    sample_top_k,
    token_logps_and_entropy,
    top_token_logps,
)


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.load()


W = torch.zeros((10, 16), dtype=torch.bfloat16)
H = torch.zeros((2, 3, 16), dtype=torch.bfloat16)
Y = torch.zeros((2, 3), dtype=torch.int64)


@pytest.mark.parametrize("change,message", [
    ({"tokens": Y[:1]}, "does not match"),
    ({"tokens": Y.reshape(3, 2)}, "does not match"),
    ({"tokens": Y.reshape(2, 3, 1, 1)}, "does not match"),
    ({"tokens": Y.float()}, "integers"),
    ({"tokens": Y.bool()}, "integers"),
    ({"tokens": torch.zeros((2, 3, 257), dtype=torch.int32)}, "at most 256"),
    ({"hidden": H[..., :8]}, "incompatible"),
    ({"embed_tokens": W[0]}, "incompatible"),
    ({"embed_tokens": W[:0]}, "no rows"),
    ({"softcap": 0.0}, "softcap"),
    ({"softcap": float("nan")}, "softcap"),
    ({"backend": "pallas"}, "entropy"),
    ({"backend": "triton"}, "unknown logprob backend"),
    ({}, "CUDA tensors"),
])  # fmt: skip
def test_logps_refusals(change, message):
    args = {"embed_tokens": W, "hidden": H, "tokens": Y, "softcap": 30.0} | change
    embed, hidden, tokens = (args.pop(name) for name in ("embed_tokens", "hidden", "tokens"))
    with pytest.raises(ValueError, match=message):
        token_logps_and_entropy(embed, hidden, tokens, **args)


@pytest.mark.parametrize("change,message", [
    ({"hidden": H[0]}, r"\[B, S, d\]"),
    ({"ids": torch.zeros((2, 1), dtype=torch.int64)}, "completion ids"),
    ({"hidden": torch.zeros((3, 3, 16), dtype=torch.bfloat16)}, "sequences"),
    ({"prompt_width": 0}, "prompt_width"),
    ({"prompt_width": 3}, "prompt_width"),
    ({"softcap": -1.0}, "softcap"),
    ({"embed_tokens": W[:, :8]}, "incompatible"),
    ({"ids": torch.zeros((2, 2))}, "integers"),
    ({}, "CUDA tensors"),
])  # fmt: skip
def test_completion_refusals(change, message):
    args = {"embed_tokens": W, "hidden": H, "ids": torch.zeros((2, 2), dtype=torch.int64),
            "mask": torch.ones((2, 2), dtype=torch.bool), "prompt_width": 2, "softcap": 30.0} | change
    first = [args.pop(name) for name in ("embed_tokens", "hidden", "ids", "mask")]
    with pytest.raises(ValueError, match=message):
        completion_logps_and_entropy(*first, **args)


@pytest.mark.parametrize("args,tokens,message", [
    ((W, H, 30.0, 0), None, "k must be"),
    ((W, H, 30.0, 11), None, "k must be"),
    ((torch.zeros((500, 16)), H, 30.0, 129), None, "k must be"),
    ((W, H, -1.0, 2), None, "softcap"),
    ((W, H[..., :8], None, 2), None, "incompatible"),
    ((W, H, None, 2), Y[:1], "does not match"),
    ((W, H, None, 2), Y.float(), "integers"),
    ((W, H, None, 2), None, "CUDA tensors"),
])  # fmt: skip
def test_top_refusals(args, tokens, message):
    with pytest.raises(ValueError, match=message):
        top_token_logps(*args, tokens=tokens)


@pytest.mark.parametrize("change,message", [
    ({"hidden": H}, r"\[B, d\]"),
    ({"embed_tokens": W[:, :8]}, "incompatible"),
    ({"softcap": 0.0}, "softcap"),
    ({"temperature": 0.0}, "temperature"),
    ({"temperature": float("inf")}, "temperature"),
    ({"top_k": 0}, "top_k"),
    ({"top_k": 11}, "top_k"),
    ({"top_p": 0.0}, "top_p"),
    ({"top_p": 1.5}, "top_p"),
    ({"top_p": float("nan")}, "top_p"),
    ({"uniform": torch.zeros(5)}, "uniform"),
    ({"uniform": torch.zeros(6, dtype=torch.float64)}, "uniform"),
    ({}, "CUDA tensors"),
])  # fmt: skip
def test_sample_refusals(change, message):
    args = {"embed_tokens": W, "hidden": H.reshape(6, 16), "softcap": 30.0, "uniform": torch.zeros(6), "temperature": 1.0,
            "top_k": 4} | change
    first = [args.pop(name) for name in ("embed_tokens", "hidden", "softcap", "uniform")]
    with pytest.raises(ValueError, match=message):
        sample_top_k(*first, **args)


def test_c_entries_refuse_before_the_device(lib):
    P = ctypes.c_void_p
    fake = P(4096)

    def refused(rc, fragment):
        assert rc == _lib.LP_EINVAL and fragment in lib.lp_last_error().decode()

    def fwd(T=4, d=8, ldh=8, K=2, y=fake):
        return lib.lp_dist_fwd(None, fake, T, d, ldh, fake, 10, 0, y, K, 0.0, None, fake, fake, fake, fake, None, fake, 1 << 20)

    refused(fwd(d=12), "multiple of 8")
    refused(fwd(ldh=4), "ldh")
    refused(fwd(T=-1), "bad sizes")
    refused(fwd(K=257), "at most 256")
    refused(fwd(K=-1), "at most 256")
    refused(fwd(y=None), "null tokens")
    refused(lib.lp_dist_combine(None, fake, fake, 0, 4, 1, 10, fake, fake, fake, fake, fake), "bad P")
    refused(lib.lp_dist_combine(None, fake, None, 2, 4, 1, 10, fake, fake, fake, fake, fake), "null shard_zt")

    def bwd(v_off=0, V=10, zt=fake, dH=fake, dW=fake, kept=None, kept_rows=4, row_of=None):
        return lib.lp_dist_bwd(None, fake, 4, 8, 8, fake, 10, v_off, V, fake, 2, 0.0, zt, fake, fake, fake, fake, kept,
                               kept_rows, row_of, dH, 8, dW, 0, 0, fake, 1 << 20)

    refused(bwd(v_off=5), "outside the vocabulary")
    refused(bwd(zt=None), "null lse")
    refused(bwd(dH=None), "dH")
    refused(bwd(dW=None), "dW")
    refused(bwd(kept=P(4100)), "kept logits")
    refused(bwd(kept=fake, kept_rows=3), "kept logits")
    assert lib.lp_dist_kept_bytes(3, 300) == 3 * 304 * 2 + 224 + 3 * 16 * 4  # 16-bit rows, 256-byte step, f32 maxima
    assert lib.lp_dist_kept_bytes(0, 300) == 0

    def rows(T=4, d=8, H=fake, y_out=fake, g_out=fake, ws=1 << 20):
        return lib.lp_dist_rows(None, H, T, d, 8, fake, 2, fake, fake, fake, fake, fake, fake, y_out, fake, fake, fake, g_out,
                                fake, fake, fake, fake, fake, ws)

    refused(rows(T=0), "bad sizes")
    refused(rows(d=12), "bad sizes")
    refused(rows(y_out=None), "null input")
    refused(rows(g_out=None), "null input")
    refused(rows(H=P(4104)), "aligned")
    assert rows(ws=1) == _lib.LP_EWORKSPACE
    for k in (0, 11, 129):
        refused(lib.lp_top(None, fake, 4, 8, 8, fake, 10, 0.0, k, None, fake, fake, fake, None, fake, 1 << 20), "k=")
    refused(lib.lp_top(None, fake, 4, 8, 8, fake, 10, 0.0, 2, fake, fake, fake, fake, None, fake, 1 << 20), "token_logps")

    def draw(temperature=1.0, top_p=1.0, uniform=fake):
        return lib.lp_sample_top_k(None, fake, 4, 8, 8, fake, 10, 0.0, 2, uniform, temperature, top_p, fake, fake, fake, 1 << 20)

    refused(draw(temperature=0.0), "temperature")
    refused(draw(temperature=float("nan")), "temperature")
    refused(draw(top_p=0.0), "top_p")
    refused(draw(top_p=1.5), "top_p")
    refused(draw(uniform=None), "null uniform")


def test_no_logits_are_kept_where_no_gradient_can_follow(lib, monkeypatch):
    """Scoring under no_grad, with parameters that otherwise train, leaves nothing for a backward."""
    kept_calls = []

    def forward(embed, hidden, tokens, softcap, logp, entropy, saved, kept=None):
        kept_calls.append(kept is not None)
        logp.zero_(), entropy.zero_()

    monkeypatch.setattr(distribution.ops, "dist_forward", forward)
    for embed, hidden in ((W.clone().requires_grad_(), H), (W, H.clone().requires_grad_())):
        for keep in (None, True):
            logps, entropy = token_logps_and_entropy(embed, hidden, Y, softcap=30.0, keep_logits=keep)
            assert logps.requires_grad and entropy.requires_grad
            with torch.no_grad():
                token_logps_and_entropy(embed, hidden, Y, softcap=30.0, keep_logits=keep)
            token_logps_and_entropy(embed.detach(), hidden.detach(), Y, softcap=30.0, keep_logits=keep)
    assert kept_calls == [True, False, False] * 4


def test_captures_look_at_the_eager_graphs_while_other_threads_add_to_them():
    """A thread's eager call may finish while another thread's captured one looks for graphs of its leaves."""

    class Node:
        def __init__(self, *leaves):
            self.leaves = leaves

    leaf, other = W.clone(), W.clone()
    threads, nodes = [], [Node(), Node(), Node()]

    def added_meanwhile():  # stands for a weak reference
        nodes.append(Node())
        threads.append(threading.Thread(target=distribution._eager_graphs.add, args=(nodes[-1], [other])))
        threads[-1].start()
        threads[-1].join(0.2)

    try:
        for node in nodes[:3]:
            distribution._eager_graphs.add(node, [other])
            node.leaves = (added_meanwhile,)
        assert not distribution._eager_graphs.holds([leaf])
        for thread in threads:
            thread.join(10)
            assert not thread.is_alive()
        assert len(threads) == 3 and distribution._eager_graphs.holds([other])
    finally:
        nodes.clear()
        threads.clear()
    assert not distribution._eager_graphs.holds([other])


def test_completions_refuse_a_capture(monkeypatch):
    """They wait for the number of valid slots, which a stream that is captured must not."""

    class OnGpu(torch.Tensor):
        is_cuda = property(lambda self: True)

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        completion_logps_and_entropy(
            W, H.as_subclass(OnGpu), torch.zeros((2, 2), dtype=torch.int64), torch.ones((2, 2), dtype=torch.bool), prompt_width=2, softcap=30.0
        )


def test_compaction_and_scatter_run_on_the_device_of_their_tensors(monkeypatch):
    """The rows of completions on another device than the current one: their kernels are launched with that
    device current, on its stream, as the distribution kernels are."""
    ops = distribution.ops
    calls = []

    class Lib:
        lp_compact_workspace_bytes = staticmethod(lambda B, N: 256)
        lp_compact = staticmethod(lambda stream, *args: calls.append(("lp_compact", stream)) or _lib.LP_OK)
        lp_scatter_rows = staticmethod(lambda stream, *args: calls.append(("lp_scatter_rows", stream)) or _lib.LP_OK)

    def on_device(dev, what, call):
        calls.append((what, dev))
        assert call("its stream") == _lib.LP_OK

    cpu = torch.device("cpu")
    monkeypatch.setattr(ops._lib, "load", Lib)
    monkeypatch.setattr(ops, "_require_cuda", lambda *tensors: cpu)
    monkeypatch.setattr(ops, "_on_device", on_device)
    ops.compact(torch.ones((2, 2), dtype=torch.bool), H, torch.zeros((2, 2), dtype=torch.int64), row_offset=1)
    ops.scatter_rows(H[0], torch.zeros(4, dtype=torch.int32), torch.zeros((4, 16), dtype=torch.bfloat16))
    assert calls == [("lp_compact", cpu), ("lp_compact", "its stream"), ("lp_scatter_rows", cpu), ("lp_scatter_rows", "its stream")]


def test_kernels_run_with_the_device_of_their_tensors_current(monkeypatch):
    ops = distribution.ops
    current = [0]

    class Current:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            current.append(self.dev.index)

        def __exit__(self, *exc):
            current.pop()

    monkeypatch.setattr(ops, "_current_device", lambda: current[-1])
    monkeypatch.setattr(ops, "_raw_stream", lambda index: f"stream of {index}")
    monkeypatch.setattr(torch.cuda, "device", Current)
    seen = []
    for index in (0, 1):
        ops._on_device(torch.device("cuda", index), "a kernel", lambda stream: seen.append((stream, current[-1])) or _lib.LP_OK)
    assert seen == [("stream of 0", 0), ("stream of 1", 1)] and current == [0]
