"""Log-probabilities of several given tokens, entropies and the most likely tokens of the LM head.

``token_logps_and_entropy`` is ``per_token_logps`` for what a loss takes besides the sampled token's
log-probability: any number of given tokens per position (a distillation or KL term over a
teacher's alternatives) and the entropy of the policy (an entropy bonus), with the gradients of
both. ``top_token_logps`` gives such alternatives: the k most likely tokens of each position.
Neither writes a ``[..., vocab]`` array of probabilities. The reference has no counterpart.
"""

from __future__ import annotations

import math
import weakref
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .losses import _gather_rows, _nonzero_grad_rows, _validate_softcap
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


def _gather(rows: torch.Tensor, idx: torch.Tensor) -> torch.Tensor:
    """``rows`` [n] or [n, w] (f32 or int32) at ``idx``."""
    return _gather_rows(rows.view(torch.float32), idx).view(rows.dtype)


class _TokenLogpsAndEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, embed, hidden, tokens, softcap, mesh, token_chunk, dh_reduce_f32, skip_zero_grad):
        P = mesh.size if mesh is not None else 1
        vocab = embed.shape[0] * P
        off = 0
        if P > 1:
            off = vocab_offset(embed.shape[0], mesh)
            stats, zt = ops.dist_forward(embed, hidden, tokens, softcap, vocab_offset=off, shard=True)
            with phase("stats_all_gather"):
                both = all_gather_stats(torch.cat([stats.reshape(-1), zt.reshape(-1)]), mesh)
            T, K = tokens.shape
            logp, entropy, zt, lse = ops.dist_combine(
                both[:, : 3 * T].reshape(P, 3, T), both[:, 3 * T :].reshape(P, T, K), tokens, vocab
            )
        else:
            logp, entropy, zt, lse = ops.dist_forward(embed, hidden, tokens, softcap)
        ctx.save_for_backward(embed, hidden, tokens, zt, lse, entropy)
        ctx.meta = (softcap, mesh, P, off, vocab, token_chunk, dh_reduce_f32, skip_zero_grad)
        ctx.set_materialize_grads(False)
        return logp, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, g, ge):
        embed, hidden, tokens, zt, lse, entropy = ctx.saved_tensors
        softcap, mesh, P, off, vocab, token_chunk, dh_reduce_f32, skip_zero_grad = ctx.meta
        need_dw, need_dh = ctx.needs_input_grad[:2]
        none = (None,) * 8
        if (g is None and ge is None) or not (need_dw or need_dh):
            return none
        g = None if g is None else g.to(torch.float32).contiguous()
        ge = None if ge is None else ge.to(torch.float32).contiguous()
        T, d = hidden.shape
        if T == 0:
            return (torch.zeros_like(embed) if need_dw else None, torch.zeros_like(hidden) if need_dh else None) + none[2:]
        sel = None
        if skip_zero_grad and 6.0 * T * d * embed.shape[0] >= _SKIP_MIN_FLOPS and not torch.cuda.is_current_stream_capturing():
            sent = torch.zeros((T,), dtype=torch.bool, device=hidden.device) if ge is None else ge != 0
            if g is not None and g.shape[1] > 0:
                sent = sent | (g != 0).any(dim=1)
            sel = _nonzero_grad_rows(sent)
        pos = None
        rows = hidden
        if sel is not None:
            idx, pos, m = sel
            if m == 0:
                dW = torch.zeros_like(embed) if need_dw else None
                return (dW, torch.zeros_like(hidden) if need_dh else None) + none[2:]
            rows = _gather_rows(hidden, idx)
            tokens, zt, lse, entropy = (_gather(x, idx) if x.numel() else x[:m] for x in (tokens, zt, lse, entropy))
            g = g if g is None else (_gather(g, idx) if g.numel() else g[:m])
            ge = ge if ge is None else _gather(ge, idx)
        dh_dtype = torch.float32 if P > 1 and dh_reduce_f32 else torch.bfloat16
        dH, dW = ops.dist_backward(
            embed, rows, tokens, softcap, zt, lse, entropy, g, ge, vocab_offset=off, vocab=vocab, need_dh=need_dh,
            need_dw=need_dw, dh_dtype=dh_dtype, token_chunk=token_chunk,
        )
        if dH is not None:
            if P > 1:
                with phase("dh_all_reduce"):
                    all_reduce_sum(dH, mesh)
            if pos is not None:
                dH = ops.scatter_rows(dH, pos, torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device))
            else:
                dH = dH.to(hidden.dtype)
        return (dW, dH) + none[2:]


# Autograd nodes of this operator's eager calls that are still alive, each with its leaves.
_eager_graphs: weakref.WeakSet = weakref.WeakSet()

# Rows without a gradient add nothing, and a backward of at least this much work (about 2 ms)
# leaves them out; below it, finding them on the host costs more than computing them.
_SKIP_MIN_FLOPS = 3e12


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
) -> tuple[torch.Tensor, torch.Tensor]:
    """Log-probabilities of given tokens and the entropy of every position's distribution.

    ``hidden`` is [..., d]; ``tokens`` holds one id per position ([...]) or K of them ([..., K],
    0 <= K <= 256). Returns (logps f32 of the shape of ``tokens``, entropy f32 [...]), both
    differentiable in ``embed_tokens`` and ``hidden``. An id outside the vocabulary (-1, say) is no
    token: its logp is 0 and sends no gradient, so lists of different lengths can be padded. A token
    named twice in a row counts twice.

    ``mesh``, ``token_chunk``, ``dh_reduce_f32`` and ``skip_zero_grad`` are those of
    ``per_token_logps``; over a mesh the shards' statistics are exchanged by one all-gather and the
    dH partials summed by one all-reduce. The call and its backward can be captured into a CUDA graph;
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
    n = math.prod(prefix)
    leaves = [x for x in (embed_tokens, hidden) if torch.is_grad_enabled() and x.requires_grad and x.is_leaf]
    capturing = bool(leaves) and hidden.is_cuda and torch.cuda.is_current_stream_capturing()
    if capturing and any(ref() is x for node in _eager_graphs for ref in node.leaves for x in leaves):
        raise RuntimeError(
            "token_logps_and_entropy: an eager graph of the same leaves is alive; free it (or use detached leaves) "
            "before capturing this call"
        )
    logps, entropy = _TokenLogpsAndEntropy.apply(
        embed_tokens, hidden.reshape(n, hidden.shape[-1]), _as_int32(tokens).reshape(n, K), softcap, mesh, token_chunk,
        dh_reduce_f32, skip_zero_grad,
    )
    if leaves and not capturing:
        logps.grad_fn.leaves = [weakref.ref(x) for x in leaves]
        _eager_graphs.add(logps.grad_fn)
    return logps.reshape(tokens.shape), entropy.reshape(prefix)


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
    if not 1 <= k <= min(_lib.LP_TOP_MAX, embed_tokens.shape[0]):
        raise ValueError(f"k must be between 1 and min({_lib.LP_TOP_MAX}, {embed_tokens.shape[0]}), got {k}")
    prefix = tuple(hidden.shape[:-1])
    n = math.prod(prefix)
    flat = None
    if tokens is not None:
        if tuple(tokens.shape) != prefix:
            raise ValueError(f"hidden prefix {prefix} does not match tokens {tuple(tokens.shape)}")
        flat = _as_int32(tokens).reshape(n)
    ids, logps, entropy, token_logps = ops.top(
        embed_tokens.detach(), hidden.detach().reshape(n, hidden.shape[-1]), softcap, int(k), flat
    )
    return TopTokenLogps(
        ids.reshape(*prefix, k), logps.reshape(*prefix, k), entropy.reshape(prefix),
        None if token_logps is None else token_logps.reshape(prefix),
    )
