"""Log-probabilities of several given tokens, entropies and the most likely tokens of the LM head.

``token_logps_and_entropy`` is ``per_token_logps`` for what a loss takes besides the sampled token's
log-probability: any number of given tokens per position (a distillation or KL term over a
teacher's alternatives) and the entropy of the policy (an entropy bonus), with the gradients of
both; ``completion_logps_and_entropy`` is its caller for completions, as ``completion_logps`` is
``per_token_logps``'. ``top_token_logps`` gives such alternatives: the k most likely tokens of each position.
Neither writes ``[..., vocab]`` probabilities. What is written of that shape: the logits in 16 bits that a
differentiable call keeps for its backward, where they take at most 4 GiB; that backward's dZ, a chunk of
rows at a time; and the f32 logits of a vocabulary of a few thousand that ``top_token_logps`` searches.
The reference has no counterpart.
"""

from __future__ import annotations

import math
import operator
import threading
import weakref
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .losses import _SKIP_ZERO_GRAD_MIN_FRACTION, _check_device, _validate_softcap
from .phase_timer import phase
from .sharding import VocabMesh, all_gather_stats, all_reduce_sum, vocab_offset


class TopTokenLogps(NamedTuple):
    """What ``top_token_logps`` returns."""

    ids: torch.Tensor  #: int32 [..., k], most likely first
    logps: torch.Tensor  #: f32 [..., k]
    entropy: torch.Tensor  #: f32 [...]
    token_logps: torch.Tensor | None  #: f32 [...]: of the given tokens


def _check_embed(embed: torch.Tensor, hidden: torch.Tensor) -> None:
    if embed.ndim != 2 or hidden.ndim < 1 or hidden.shape[-1] != embed.shape[-1]:
        raise ValueError(f"incompatible embedding {tuple(embed.shape)} and hidden {tuple(hidden.shape)}")
    if embed.shape[0] == 0:
        raise ValueError("the embedding has no rows")


def _as_int32(tokens: torch.Tensor) -> torch.Tensor:
    """Contiguous int32 ids; an id beyond int32 stays outside every vocabulary."""
    if tokens.dtype.is_floating_point or tokens.dtype.is_complex or tokens.dtype == torch.bool:
        raise ValueError(f"tokens must be integers, got {tokens.dtype}")
    if tokens.dtype in (torch.int64, torch.uint64, torch.uint32):
        tokens = tokens.to(torch.int64).clamp(-1, 2**31 - 1)
    return tokens.to(torch.int32).contiguous()


class _TokenLogpsAndEntropy(torch.autograd.Function):
    """hidden [..., d] and int32 tokens [T, K] to logps ``shape`` and entropy [...]. The reshapes are in
    here: outside, each would be a node of the autograd graph of its own."""

    @staticmethod
    def forward(ctx, embed, hidden, tokens, shape, softcap, mesh, token_chunk, dh_reduce_f32, skip_zero_grad, keep_logits):
        T, K = tokens.shape
        dev = hidden.device
        h = hidden if hidden.ndim == 2 else hidden.reshape(T, hidden.shape[-1])
        logp = torch.empty(shape, dtype=torch.float32, device=dev)
        entropy = torch.empty(hidden.shape[:-1], dtype=torch.float32, device=dev)
        most = 0  # bytes of kept logits
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            most = _KEPT_MAX_BYTES if keep_logits is None else (math.inf if keep_logits else 0)
        saved, kept = ops.dist_saved(T, K, embed.shape[0], most, dev)
        P = mesh.size if mesh is not None else 1
        off = 0
        if P > 1:
            off = vocab_offset(embed.shape[0], mesh)
            stats, zt = ops.dist_forward_shard(embed, h, tokens, softcap, off, kept)
            with phase("stats_all_gather"):
                both = all_gather_stats(torch.cat([stats.reshape(-1), zt.reshape(-1)]), mesh)
            ops.dist_combine(
                both[:, : 3 * T].reshape(P, 3, T), both[:, 3 * T :].reshape(P, T, K), tokens, embed.shape[0] * P, logp,
                entropy, saved,
            )
        else:
            ops.dist_forward(embed, h, tokens, softcap, logp, entropy, saved, kept)
        ctx.save_for_backward(embed, hidden, tokens, saved, entropy)
        ctx.meta = (softcap, mesh, P, off, token_chunk, dh_reduce_f32, skip_zero_grad)
        ctx.set_materialize_grads(False)
        return logp, entropy

    @staticmethod
    def backward(ctx, g, ge):
        if not torch.is_grad_enabled():
            return _dist_gradients(ctx, g, ge)
        # A graph of the backward itself is asked for. once_differentiable lets its results refuse a
        # second derivative, if an incoming gradient takes part in the graph: these do, here.
        return _once(ctx, *(None if x is None else x.detach().requires_grad_() for x in (g, ge)))


def _dist_gradients(ctx, g, ge):
    need_dw, need_dh = ctx.needs_input_grad[:2]
    none = (None,) * 8
    if (g is None and ge is None) or not (need_dw or need_dh):
        return None, None, *none
    embed, hidden, tokens, saved, entropy = ctx.saved_tensors
    softcap, mesh, P, off, token_chunk, dh_reduce_f32, skip_zero_grad = ctx.meta
    T, K = tokens.shape
    d = hidden.shape[-1]
    if T == 0:
        return (torch.zeros_like(embed) if need_dw else None), (torch.zeros_like(hidden) if need_dh else None), *none
    g = None if g is None else g.contiguous()
    ge = None if ge is None else ge.contiguous()
    args = (hidden if hidden.ndim == 2 else hidden.reshape(T, d), tokens, saved, entropy, g, ge)
    rows = pos = row_of = None
    if (
        skip_zero_grad
        and 6.0 * T * d * embed.shape[0] >= _SKIP_MIN_FLOPS
        and not torch.cuda.is_current_stream_capturing()
    ):
        idx, where, count, gathered = ops.dist_rows(*args)
        m = int(count.item())
        _check_device(hidden.device, "token_logps_and_entropy backward")  # the host has waited anyway
        if m == 0:
            return (torch.zeros_like(embed) if need_dw else None), (torch.zeros_like(hidden) if need_dh else None), *none
        if T - m >= _SKIP_ZERO_GRAD_MIN_FRACTION * T:
            args, rows, pos, row_of = gathered, m, where, idx
    dH, dW = ops.dist_backward(
        embed, softcap, *args, rows=rows, kept=ops.dist_kept(saved, T, K), row_of=row_of, vocab_offset=off,
        vocab=embed.shape[0] * P, need_dh=need_dh, need_dw=need_dw,
        dh_dtype=torch.float32 if P > 1 and dh_reduce_f32 else torch.bfloat16, token_chunk=token_chunk,
    )
    if dH is not None:
        if P > 1:
            with phase("dh_all_reduce"):
                all_reduce_sum(dH, mesh)
        if pos is not None:
            dH = ops.scatter_rows(dH, pos, torch.empty((T, d), dtype=hidden.dtype, device=hidden.device))
        elif dH.dtype != hidden.dtype:
            dH = dH.to(hidden.dtype)
        if hidden.ndim != 2:
            dH = dH.view(hidden.shape)
    return dW, dH, *none


_once = once_differentiable(_dist_gradients)


class _EagerGraphs:
    """Autograd nodes of this operator's eager calls that are still alive, each with its leaves. Calls of
    several threads may add to it while others look."""

    def __init__(self):
        self._nodes: weakref.WeakSet = weakref.WeakSet()
        self._lock = threading.RLock()

    def add(self, node, leaves: list[torch.Tensor]) -> None:
        node.leaves = [weakref.ref(x) for x in leaves]
        with self._lock:
            self._nodes.add(node)

    def holds(self, leaves: list[torch.Tensor]) -> bool:
        with self._lock:
            nodes = list(self._nodes)
        return any(ref() is x for node in nodes for ref in node.leaves for x in leaves)


_eager_graphs = _EagerGraphs()

# Logits are kept for the backward up to this many bytes (7710 rows of a vocabulary of 262144, 16 bits
# each and an f32 for every 32), the size of the backward's own dZ scratch.
_KEPT_MAX_BYTES = 4 << 30

# Rows without a gradient add nothing, and a backward of at least this much work (about 3 ms)
# leaves them out. Below it, the wait for their number and whole tiles of 256 rows that a few rows
# fewer do not save cost what a tenth of the rows would.
_SKIP_MIN_FLOPS = 5e12


def token_logps_and_entropy(
    embed_tokens: torch.Tensor,
    hidden: torch.Tensor,
    tokens: torch.Tensor,
    *,
    softcap: float | None,
    mesh: VocabMesh | None = None,
    backend: str = "cuda",
    token_chunk: int | None = None,
    dh_reduce_f32: bool = False,
    skip_zero_grad: bool = True,
    keep_logits: bool | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Log-probabilities of given tokens and the entropy of every position's distribution.

    ``hidden`` is [..., d]; ``tokens`` holds one id per position ([...]) or K of them ([..., K],
    0 <= K <= 256). Returns (logps f32 of the shape of ``tokens``, entropy f32 [...]), both
    differentiable in ``embed_tokens`` and ``hidden``. An id outside the vocabulary (-1, say) is no
    token: its logp is 0 and sends no gradient, so lists of different lengths can be padded. A token
    named twice in a row counts twice.

    A differentiable call keeps the logits in 16 bits each for its backward when they take at most
    4 GiB, and recomputes them there otherwise; ``keep_logits`` says so either way. They live as long as
    the call's graph does, so several forwards before their backwards hold as many of them:
    ``keep_logits=False`` trades that memory for the recompute. (A kept logit is within 2.6e-4 of its
    value, which moves the gradients by a fifteenth of their bf16 rounding. Among 32 neighbours of which
    one is within 3 % of the softcap it is within 5.1e-4, or within 1.3e-5 of the softcap where it is so
    near itself; the softcap's slope there is within 4.2e-4 of itself. The given tokens' own entries come
    from their f32 logits.)

    ``mesh``, ``token_chunk``, ``dh_reduce_f32`` and ``skip_zero_grad`` are those of
    ``per_token_logps``, but rows without a gradient are left out only of a backward of 5e12 flops or
    more (counted as 6 T V d), where that saves more than it costs; over a mesh the shards' statistics are
    exchanged by one all-gather and the dH partials summed by one all-reduce. The call and its backward can be captured into a CUDA graph;
    rows without a gradient are then computed like the others, since leaving them out takes a read
    on the host. A captured backward must not meet an eager graph of the same leaves: autograd would
    tie the capture to the stream of the eager one. While such a graph of this operator lives, a
    differentiable call under capture is refused; those of other operators are the caller's to free.
    """
    if backend != "cuda":
        raise ValueError(f"unknown logprob backend: {backend}" if backend not in ("jax", "pallas") else
                         f"logprob backend {backend!r} has no entropy; this package provides backend='cuda'")
    _check_embed(embed_tokens, hidden)
    _validate_softcap(softcap)
    prefix = tuple(hidden.shape[:-1])
    single = tuple(tokens.shape) == prefix
    if not single and (tokens.ndim != len(prefix) + 1 or tuple(tokens.shape[:-1]) != prefix):
        raise ValueError(f"hidden prefix {prefix} does not match tokens {tuple(tokens.shape)}")
    K = 1 if single else tokens.shape[-1]
    if K > _lib.LP_DIST_MAX_TOKENS:
        raise ValueError(f"at most {_lib.LP_DIST_MAX_TOKENS} tokens per position, got {K}")
    if mesh is not None and mesh.size > 1 and mesh.axis_names != ("d",):
        raise ValueError(f"vocab-parallel mesh needs axis 'd': {mesh.axis_names}")
    if not torch.is_grad_enabled():
        keep_logits = False  # autograd.Function cannot see it: its forward is always outside grad mode
    leaves = [x for x in (embed_tokens, hidden) if x.requires_grad and x.is_leaf] if torch.is_grad_enabled() else []
    capturing = bool(leaves) and hidden.is_cuda and torch.cuda.is_current_stream_capturing()
    if capturing and _eager_graphs.holds(leaves):
        raise RuntimeError(
            "token_logps_and_entropy: an eager graph of the same leaves is alive; free it (or use detached leaves) "
            "before capturing this call"
        )
    logps, entropy = _TokenLogpsAndEntropy.apply(
        embed_tokens, hidden, _as_int32(tokens).view(math.prod(prefix), K), tuple(tokens.shape), softcap, mesh, token_chunk,
        dh_reduce_f32, skip_zero_grad, keep_logits,
    )
    if leaves and not capturing:
        _eager_graphs.add(logps.grad_fn, leaves)
    return logps, entropy


class _ValidSlots(torch.autograd.Function):
    """The rows of hidden [B, S, d] and ids [B, N] at the valid slots of mask [B, N], in slot order."""

    @staticmethod
    def forward(ctx, hidden, ids, mask, first):
        rows, tokens, idx, pos, count = ops.compact(mask, hidden, ids, row_offset=first)
        n = int(count.item())
        _check_device(hidden.device, "completion_logps_and_entropy")  # the host has waited anyway
        ctx.save_for_backward(pos)
        ctx.meta = (tuple(hidden.shape), hidden.dtype, first, mask.shape[1])
        tokens, idx = tokens[:n], idx[:n]
        ctx.mark_non_differentiable(tokens, idx)
        return rows[:n], tokens, idx

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _tokens, _idx):
        (pos,) = ctx.saved_tensors
        shape, dtype, first, width = ctx.meta
        out = torch.zeros(shape, dtype=dtype, device=g.device)
        ops.scatter_rows(g.contiguous(), pos, out[:, first : first + width])
        return out, None, None, None


def completion_logps_and_entropy(
    embed_tokens: torch.Tensor,
    hidden: torch.Tensor,
    completion_ids: torch.Tensor,
    completion_mask: torch.Tensor,
    *,
    prompt_width: int,
    softcap: float | None,
    **options,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``completion_logps`` with the entropy: (logps [B, N], entropy [B, N]) of the completion tokens of
    hidden [B, P + N, d], differentiable, computed at the valid slots only and 0 elsewhere. The host
    waits once for the number of valid slots, so the call cannot be captured into a CUDA graph and is
    refused there (``token_logps_and_entropy``, with -1 for the tokens of the other slots, can be).
    ``options`` are those of ``token_logps_and_entropy``.
    """
    if hidden.ndim != 3 or completion_ids.ndim != 2 or completion_mask.shape != completion_ids.shape:
        raise ValueError("hidden must be [B, S, d] and completion ids / mask [B, N]")
    if completion_ids.shape[0] != hidden.shape[0]:
        raise ValueError(f"hidden has {hidden.shape[0]} sequences, completion ids {completion_ids.shape[0]}")
    if prompt_width < 1 or prompt_width - 1 + completion_ids.shape[1] > hidden.shape[1]:
        raise ValueError("prompt_width and completion width do not fit the hidden sequence")
    _check_embed(embed_tokens, hidden)
    _validate_softcap(softcap)
    if hidden.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            "completion_logps_and_entropy waits for the number of valid slots and cannot be captured; capture "
            "token_logps_and_entropy with -1 for the tokens of the other slots"
        )
    rows = hidden
    if hidden.stride(-1) != 1 or hidden.stride(0) % 8 or hidden.stride(1) % 8 or hidden.data_ptr() % 16:
        rows = hidden.contiguous()
    rows, tokens, idx = _ValidSlots.apply(rows, _as_int32(completion_ids), completion_mask, prompt_width - 1)
    if rows.grad_fn is not None and hidden.is_leaf:
        _eager_graphs.add(rows.grad_fn, [hidden])
    logps, entropy = token_logps_and_entropy(embed_tokens, rows, tokens, softcap=softcap, **options)
    slots = idx.long()

    def scattered(values):
        out = torch.zeros(completion_ids.numel(), dtype=values.dtype, device=values.device)
        return out.index_put((slots,), values).view(completion_ids.shape)

    return scattered(logps), scattered(entropy)


def top_token_logps(
    embed_tokens: torch.Tensor,
    hidden: torch.Tensor,
    softcap: float | None,
    k: int,
    *,
    tokens: torch.Tensor | None = None,
) -> TopTokenLogps:
    """The ``k`` most likely tokens of every position of ``hidden`` [..., d] over the whole vocabulary,
    with their log-probabilities and the entropy; with ``tokens`` [...], those tokens'
    log-probabilities too (0 for an id outside the vocabulary). 1 <= k <= min(128, V).

    Tokens are ranked by their exact dot products with the hidden state, the lowest id first among
    equals. Not differentiable: ``token_logps_and_entropy`` of the ids is.
    """
    _check_embed(embed_tokens, hidden)
    _validate_softcap(softcap)
    k = operator.index(k)
    if not 1 <= k <= min(_lib.LP_TOP_MAX, embed_tokens.shape[0]):
        raise ValueError(f"k must be between 1 and min({_lib.LP_TOP_MAX}, {embed_tokens.shape[0]}), got {k}")
    prefix = tuple(hidden.shape[:-1])
    token_logps = None
    if tokens is not None:
        if tuple(tokens.shape) != prefix:
            raise ValueError(f"hidden prefix {prefix} does not match tokens {tuple(tokens.shape)}")
        tokens = _as_int32(tokens)
        token_logps = torch.empty(prefix, dtype=torch.float32, device=hidden.device)
    ids = torch.empty((*prefix, k), dtype=torch.int32, device=hidden.device)
    logps = torch.empty((*prefix, k), dtype=torch.float32, device=hidden.device)
    entropy = torch.empty(prefix, dtype=torch.float32, device=hidden.device)
    with torch.no_grad():
        rows = hidden if hidden.ndim == 2 else hidden.reshape(math.prod(prefix), hidden.shape[-1])
        ops.top(embed_tokens, rows, softcap, k, tokens, ids, logps, entropy, token_logps)
    return TopTokenLogps(ids, logps, entropy, token_logps)
