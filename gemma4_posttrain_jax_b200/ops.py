"""Torch-facing wrappers over the C ABI: raw device pointers in, torch tensors out.

torch supplies device memory, the current CUDA stream and (in ``sharding``) the NCCL
process group; all arithmetic runs in liblp_b200.so. Nothing here computes on the host
and nothing falls back to torch ops: a missing library or a non-CUDA tensor raises.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

_MIN_ALIGN = 1024


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("the cuda logprob backend needs CUDA tensors; it has no CPU fallback")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    if dev is None:
        raise ValueError("no tensor given")
    return dev


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _workspace(nbytes: int, device: torch.device) -> tuple[torch.Tensor, ctypes.c_void_p, int]:
    """A scratch buffer from torch's caching allocator, aligned to 1 KiB."""
    buf = torch.empty(int(nbytes) + _MIN_ALIGN, dtype=torch.uint8, device=device)
    base = buf.data_ptr()
    off = (-base) % _MIN_ALIGN
    return buf, ctypes.c_void_p(base + off), int(nbytes)


def _rows(h: torch.Tensor) -> tuple[torch.Tensor, int]:
    """View ``h`` as [T, d] with unit column stride; returns (view, row stride)."""
    h2 = h.reshape(-1, h.shape[-1])
    if h2.stride(-1) != 1 or (h2.shape[0] > 1 and h2.stride(0) % 8 != 0):
        h2 = h2.contiguous()
    ld = h2.stride(0) if h2.shape[0] > 1 else h2.shape[1]
    return h2, int(ld)


def _check_bf16(name: str, t: torch.Tensor) -> None:
    if t.dtype != torch.bfloat16:
        raise ValueError(f"the cuda logprob backend needs bf16 {name}, got {t.dtype}")


def shard_forward(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    targets: torch.Tensor,
    softcap: float | None,
    *,
    vocab_offset: int = 0,
    want_logp: bool = True,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``lp_fwd`` on one vocabulary shard.

    Returns ``stats`` f32 [3, T] (shard max, shard sum exp(z - max), owned target logit)
    and, when ``want_logp``, logp f32 [T] (valid when the shard is the whole vocabulary).
    """
    dev = _require_cuda(embed, hidden, targets)
    _check_bf16("embedding", embed)
    _check_bf16("hidden", hidden)
    lib = _lib.load()
    h2, ldh = _rows(hidden)
    T, d = h2.shape
    Vs = embed.shape[0]
    w = embed if embed.is_contiguous() else embed.contiguous()
    y = targets.reshape(-1).to(torch.int32).contiguous()
    stats = torch.empty((3, T), dtype=torch.float32, device=dev)
    logp = torch.empty((T,), dtype=torch.float32, device=dev) if want_logp else None
    if T == 0:
        return stats, logp
    ws, wsp, wsn = _workspace(lib.lp_fwd_workspace_bytes(T, Vs), dev)
    cap = float(softcap) if softcap is not None else 0.0
    rc = lib.lp_fwd(
        _stream(dev), _ptr(h2), T, d, ldh, _ptr(w), Vs, int(vocab_offset), _ptr(y), cap, _ptr(stats), _ptr(logp), wsp, wsn
    )
    _lib.check(rc, "lp_fwd")
    return stats, logp


def shard_forward_sum(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    targets: torch.Tensor,
    softcap: float | None,
    exchange,
    *,
    vocab_offset: int,
    timeout_ms: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``lp_fwd_sum``: the forward of this rank's shard with the triples exchanged over
    NVLink (``exchange`` is a ``sharding.StatsExchange`` with room for T rows; every rank of
    the mesh makes the same call). Returns the global (logp [T], normalization [2, T])."""
    dev = _require_cuda(embed, hidden, targets)
    _check_bf16("embedding", embed)
    _check_bf16("hidden", hidden)
    lib = _lib.load()
    h2, ldh = _rows(hidden)
    T, d = h2.shape
    Vs = embed.shape[0]
    if T > exchange.rows:
        raise ValueError(f"stats exchange holds {exchange.rows} rows, {T} needed")
    w = embed if embed.is_contiguous() else embed.contiguous()
    y = targets.reshape(-1).to(torch.int32).contiguous()
    logp = torch.empty((T,), dtype=torch.float32, device=dev)
    norm = torch.empty((2, T), dtype=torch.float32, device=dev)
    if T == 0:
        return logp, norm
    ws, wsp, wsn = _workspace(lib.lp_fwd_workspace_bytes(T, Vs), dev)
    cap = float(softcap) if softcap is not None else 0.0
    xch, xch_mc, cnt, cnt_mc, arr, epoch = exchange.next_call()
    rc = lib.lp_fwd_sum(
        _stream(dev), _ptr(h2), T, d, ldh, _ptr(w), Vs, int(vocab_offset), _ptr(y), cap, ctypes.c_void_p(xch),
        ctypes.c_void_p(xch_mc), exchange.rows, ctypes.c_void_p(cnt), ctypes.c_void_p(cnt_mc), ctypes.c_void_p(arr),
        epoch, exchange.rank, exchange.world, int(timeout_ms), _ptr(logp), _ptr(norm), wsp, wsn,
    )
    _lib.check(rc, "lp_fwd_sum")
    return logp, norm


def head(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    softcap: float | None,
    *,
    want_logits: bool = True,
    log_probs: bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``lp_head`` over the whole vocabulary for B rows: (logits f32 [B, V] or None,
    normalization [2, B], argmax int32 [B], logp of the argmax [B]). ``log_probs`` makes the
    first output the full log-softmax instead of the logits."""
    dev = _require_cuda(embed, hidden)
    _check_bf16("embedding", embed)
    _check_bf16("hidden", hidden)
    if log_probs and not want_logits:
        raise ValueError("log_probs needs want_logits")
    lib = _lib.load()
    h2, ldh = _rows(hidden)
    B, d = h2.shape
    V = embed.shape[0]
    w = embed if embed.is_contiguous() else embed.contiguous()
    ld = -(-V // 4) * 4
    logits = torch.empty((B, ld), dtype=torch.float32, device=dev)[:, :V] if want_logits else None
    norm = torch.empty((2, B), dtype=torch.float32, device=dev)
    top = torch.empty((B,), dtype=torch.int32, device=dev)
    top_logp = torch.empty((B,), dtype=torch.float32, device=dev)
    if B == 0:
        return logits, norm, top, top_logp
    ws, wsp, wsn = _workspace(lib.lp_head_workspace_bytes(B, V), dev)
    cap = float(softcap) if softcap is not None else 0.0
    rc = lib.lp_head(
        _stream(dev), _ptr(h2), B, d, ldh, _ptr(w), V, cap, _ptr(logits), ld,
        _lib.LP_HEAD_LOGPROBS if log_probs else 0, _ptr(norm), _ptr(top), _ptr(top_logp), wsp, wsn,
    )
    _lib.check(rc, "lp_head")
    return logits, norm, top, top_logp


def _dense_rows(h: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``h`` [T, d] as the distribution kernels read it: unit column stride, 16-byte aligned rows
    that do not overlap (an expanded or oddly sliced ``h`` is copied); (view, row stride)."""
    T, d = h.shape
    ld, step = h.stride()
    if T <= 1:
        ld = d
    if step != 1 or ld % 8 or ld < d or h.data_ptr() % 16:
        return h.clone(memory_format=torch.contiguous_format), d
    return h, ld


def _dense_embed(w: torch.Tensor) -> torch.Tensor:
    if w.is_contiguous() and w.data_ptr() % 16 == 0:
        return w
    return w.clone(memory_format=torch.contiguous_format)


def _check_head(embed: torch.Tensor, hidden: torch.Tensor, *others: torch.Tensor | None) -> torch.device:
    dev = embed.device
    if not embed.is_cuda or hidden.device != dev or any(t is not None and t.device != dev for t in others):
        _require_cuda(embed, hidden, *others)  # says what is wrong
    _check_bf16("embedding", embed)
    _check_bf16("hidden", hidden)
    return dev


def _addr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# Small calls take as long as the host takes to make them, so these look things up by the shortest way
# (torch.cuda.current_stream builds a Stream object, torch.cuda.current_device checks its set-up).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda i: torch.cuda.current_stream(i).cuda_stream)


def _on_device(dev: torch.device, what: str, call) -> None:
    """``call(stream)`` with ``dev`` current, and its return code checked."""
    if dev.index == _current_device():
        rc = call(_raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = call(_raw_stream(dev.index))
    if rc != _lib.LP_OK:
        _lib.check(rc, what)


def dist_saved(T: int, K: int, vocab_rows: int, most: float, dev: torch.device) -> tuple[torch.Tensor, int | None]:
    """What a forward leaves for its backward, as one f32 tensor: the tokens' logits [T, K], the rows'
    log-normalisers [T] and, where they take at most ``most`` bytes, the logits in 16 bits;
    (tensor, address of those or None)."""
    n = T * K + T
    at = -(-n // 64) * 64
    nbytes = _lib.load().lp_dist_kept_bytes(T, vocab_rows) if most > 0 else 0
    keep = 0 < nbytes <= most
    saved = torch.empty((at + -(-nbytes // 4) if keep else n,), dtype=torch.float32, device=dev)
    return saved, saved.data_ptr() + 4 * at if keep else None


def dist_kept(saved: torch.Tensor, T: int, K: int) -> int | None:
    """Address of the kept logits in ``dist_saved``'s tensor, if it has them."""
    at = -(-(T * K + T) // 64) * 64
    return saved.data_ptr() + 4 * at if saved.numel() > T * K + T else None


def dist_forward(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    tokens: torch.Tensor,
    softcap: float | None,
    logp: torch.Tensor,
    entropy: torch.Tensor,
    saved: torch.Tensor,
    kept: int | None = None,
) -> None:
    """``lp_dist_fwd`` for int32 ``tokens`` [T, K] into f32 ``logp`` (T * K), ``entropy`` (T) and
    ``dist_saved``'s tensor."""
    dev = _check_head(embed, hidden, tokens)
    lib = _lib.load()
    T, K = tokens.shape
    if T == 0:
        return
    h, ldh = _dense_rows(hidden)
    w = _dense_embed(embed)
    V, d = w.shape

    def call(stream):
        ws, wsp, wsn = _workspace(lib.lp_dist_fwd_workspace_bytes(T, V), dev)
        zt = saved.data_ptr()
        return lib.lp_dist_fwd(
            stream, h.data_ptr(), T, d, ldh, w.data_ptr(), V, 0, tokens.data_ptr(), K, softcap or 0.0, None, zt,
            zt + 4 * T * K, entropy.data_ptr(), logp.data_ptr(), kept, wsp, wsn,
        )

    _on_device(dev, "lp_dist_fwd", call)


def dist_forward_shard(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    tokens: torch.Tensor,
    softcap: float | None,
    vocab_offset: int,
    kept: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``lp_dist_fwd`` over one shard of the vocabulary: (stats [3, T], zt [T, K]) for ``dist_combine``."""
    dev = _check_head(embed, hidden, tokens)
    lib = _lib.load()
    T, K = tokens.shape
    stats = torch.empty((3, T), dtype=torch.float32, device=dev)
    zt = torch.empty((T, K), dtype=torch.float32, device=dev)
    if T > 0:
        h, ldh = _dense_rows(hidden)
        w = _dense_embed(embed)

        def call(stream):
            ws, wsp, wsn = _workspace(lib.lp_dist_fwd_workspace_bytes(T, w.shape[0]), dev)
            return lib.lp_dist_fwd(
                stream, h.data_ptr(), T, h.shape[1], ldh, w.data_ptr(), w.shape[0], int(vocab_offset),
                tokens.data_ptr(), K, softcap or 0.0, stats.data_ptr(), zt.data_ptr(), None, None, None, kept, wsp, wsn,
            )

        _on_device(dev, "lp_dist_fwd", call)
    return stats, zt


def dist_combine(
    shard_stats: torch.Tensor,
    shard_zt: torch.Tensor,
    tokens: torch.Tensor,
    vocab: int,
    logp: torch.Tensor,
    entropy: torch.Tensor,
    saved: torch.Tensor,
) -> None:
    """``lp_dist_combine``: [P, 3, T] and [P, T, K] into f32 ``logp`` (T * K), ``entropy`` (T) and
    ``dist_saved``'s tensor."""
    dev = _require_cuda(shard_stats, shard_zt, tokens)
    lib = _lib.load()
    T, K = tokens.shape
    stats, parts = shard_stats.contiguous(), shard_zt.contiguous()
    zt = saved.data_ptr()
    _on_device(dev, "lp_dist_combine", lambda stream: lib.lp_dist_combine(
        stream, stats.data_ptr(), parts.data_ptr(), stats.shape[0], T, K, int(vocab), tokens.data_ptr(), zt + 4 * T * K,
        entropy.data_ptr(), zt, logp.data_ptr(),
    ))


def dist_rows(
    hidden: torch.Tensor,
    tokens: torch.Tensor,
    saved: torch.Tensor,
    entropy: torch.Tensor,
    grad_logp: torch.Tensor | None,
    grad_entropy: torch.Tensor | None,
):
    """``lp_dist_rows``: (idx [T], pos [T], count [1], rows), where ``rows`` are the arguments of
    ``dist_backward`` from ``hidden`` on (without softcap), holding the ``count`` rows that send a
    gradient first."""
    dev = _require_cuda(hidden, tokens, saved, entropy, grad_logp, grad_entropy)
    lib = _lib.load()
    T, K = tokens.shape
    h, ldh = _dense_rows(hidden)
    d = h.shape[1]
    h_out = torch.empty((T, d), dtype=h.dtype, device=dev)
    y_out = torch.empty_like(tokens)
    saved_out, _ = dist_saved(T, K, 0, 0, dev)
    entropy_out = torch.empty((T,), dtype=torch.float32, device=dev)
    g_out = None if grad_logp is None else torch.empty((T, K), dtype=torch.float32, device=dev)
    ge_out = None if grad_entropy is None else torch.empty((T,), dtype=torch.float32, device=dev)
    index = torch.empty((2 * T + 1,), dtype=torch.int32, device=dev)
    lse = 4 * T * K

    def call(stream):
        ws, wsp, wsn = _workspace(lib.lp_dist_rows_workspace_bytes(T), dev)
        zt, zt_out, at = saved.data_ptr(), saved_out.data_ptr(), index.data_ptr()
        return lib.lp_dist_rows(
            stream, h.data_ptr(), T, d, ldh, tokens.data_ptr(), K, zt, zt + lse, entropy.data_ptr(), _addr(grad_logp),
            _addr(grad_entropy), h_out.data_ptr(), y_out.data_ptr(), zt_out, zt_out + lse, entropy_out.data_ptr(),
            _addr(g_out), _addr(ge_out), at, at + 4 * T, at + 8 * T, wsp, wsn,
        )

    _on_device(dev, "lp_dist_rows", call)
    return index[:T], index[T : 2 * T], index[2 * T :], (h_out, y_out, saved_out, entropy_out, g_out, ge_out)


def dist_backward(
    embed: torch.Tensor,
    softcap: float | None,
    hidden: torch.Tensor,
    tokens: torch.Tensor,
    saved: torch.Tensor,
    entropy: torch.Tensor,
    grad_logp: torch.Tensor | None,
    grad_entropy: torch.Tensor | None,
    *,
    rows: int | None = None,
    kept: int | None = None,
    row_of: torch.Tensor | None = None,
    vocab_offset: int = 0,
    vocab: int | None = None,
    need_dh: bool = True,
    need_dw: bool = True,
    dh_dtype: torch.dtype = torch.bfloat16,
    dw_dtype: torch.dtype = torch.bfloat16,
    token_chunk: int | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``lp_dist_bwd``: (dH [T, d], partial over this shard; dW [Vs, d]) of contiguous f32 ``grad_logp``
    (T * K) and ``grad_entropy`` (T), either of which may be None. ``saved`` is the forward's;
    ``vocab`` is the whole vocabulary's size. ``rows`` takes the first that many rows only (of
    ``dist_rows``). ``kept`` is the address of the forward's kept logits of as many rows as ``tokens``
    has, of which row t's are at ``row_of[t]`` (int32; None: t)."""
    dev = _check_head(embed, hidden, tokens, saved, entropy, grad_logp, grad_entropy)
    lib = _lib.load()
    all_rows, K = tokens.shape
    T = all_rows if rows is None else rows
    Vs, d = embed.shape
    flags = 0
    dH = dW = None
    if need_dh:
        dH = torch.empty((T, d), dtype=dh_dtype, device=dev)
        flags |= _lib.LP_BWD_DH_F32 if dh_dtype == torch.float32 else 0
    else:
        flags |= _lib.LP_BWD_NO_DH
    if need_dw:
        dW = torch.empty((Vs, d), dtype=dw_dtype, device=dev)
        flags |= _lib.LP_BWD_DW_BF16 if dw_dtype == torch.bfloat16 else 0
    else:
        flags |= _lib.LP_BWD_NO_DW
    h, ldh = _dense_rows(hidden) if T > 0 else (hidden, d)
    w = _dense_embed(embed)
    chunk = int(token_chunk) if token_chunk else 0

    def call(stream):
        ws, wsp, wsn = _workspace(lib.lp_dist_bwd_workspace_bytes(T, d, Vs, chunk, flags), dev)
        zt = saved.data_ptr()
        return lib.lp_dist_bwd(
            stream, h.data_ptr(), T, d, ldh, w.data_ptr(), Vs, int(vocab_offset), int(vocab) if vocab else Vs,
            tokens.data_ptr(), K, softcap or 0.0, zt, zt + 4 * all_rows * K, entropy.data_ptr(), _addr(grad_logp),
            _addr(grad_entropy), kept, all_rows, _addr(row_of), _addr(dH), d, _addr(dW), flags, chunk, wsp, wsn,
        )

    _on_device(dev, "lp_dist_bwd", call)
    return dH, dW


def top(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    softcap: float | None,
    k: int,
    tokens: torch.Tensor | None,
    ids: torch.Tensor,
    logps: torch.Tensor,
    entropy: torch.Tensor,
    token_logps: torch.Tensor | None,
) -> None:
    """``lp_top`` of hidden [T, d] into int32 ``ids`` and f32 ``logps`` (T * k), f32 ``entropy`` (T) and,
    with int32 ``tokens`` (T), their ``token_logps`` (T)."""
    dev = _check_head(embed, hidden, tokens)
    lib = _lib.load()
    T, V = hidden.shape[0], embed.shape[0]
    if T == 0:
        return
    h, ldh = _dense_rows(hidden)
    w = _dense_embed(embed)

    def call(stream):
        ws, wsp, wsn = _workspace(lib.lp_top_workspace_bytes(T, V, k), dev)
        return lib.lp_top(
            stream, h.data_ptr(), T, h.shape[1], ldh, w.data_ptr(), V, softcap or 0.0, k, _addr(tokens), ids.data_ptr(),
            logps.data_ptr(), entropy.data_ptr(), _addr(token_logps), wsp, wsn,
        )

    _on_device(dev, "lp_top", call)


def sample_top_k(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    softcap: float | None,
    uniform: torch.Tensor,
    *,
    temperature: float,
    top_k: int,
    top_p: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``lp_sample_top_k``: (token int32 [B], logp [B]) for f32 ``uniform`` [B]."""
    dev = _check_head(embed, hidden, uniform)
    lib = _lib.load()
    B, V = hidden.shape[0], embed.shape[0]
    token = torch.empty((B,), dtype=torch.int32, device=dev)
    logp = torch.empty((B,), dtype=torch.float32, device=dev)
    if B == 0:
        return token, logp
    h, ldh = _dense_rows(hidden)
    w = _dense_embed(embed)

    def call(stream):
        ws, wsp, wsn = _workspace(lib.lp_top_workspace_bytes(B, V, top_k), dev)
        return lib.lp_sample_top_k(
            stream, h.data_ptr(), B, h.shape[1], ldh, w.data_ptr(), V, softcap or 0.0, top_k, uniform.data_ptr(),
            temperature, top_p, token.data_ptr(), logp.data_ptr(), wsp, wsn,
        )

    _on_device(dev, "lp_sample_top_k", call)
    return token, logp


def combine(shard_stats: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``lp_combine``: [P, 3, T] per-shard triples -> (logp [T], normalization [2, T])."""
    dev = _require_cuda(shard_stats)
    lib = _lib.load()
    s = shard_stats.to(torch.float32).contiguous()
    P, three, T = s.shape
    if three != 3:
        raise ValueError(f"shard stats must be [P, 3, T], got {tuple(s.shape)}")
    logp = torch.empty((T,), dtype=torch.float32, device=dev)
    norm = torch.empty((2, T), dtype=torch.float32, device=dev)
    _lib.check(lib.lp_combine(_stream(dev), _ptr(s), P, T, _ptr(logp), _ptr(norm)), "lp_combine")
    return logp, norm


def shard_backward(
    embed: torch.Tensor,
    hidden: torch.Tensor,
    targets: torch.Tensor,
    softcap: float | None,
    norm: torch.Tensor,
    grad_logp: torch.Tensor,
    *,
    vocab_offset: int = 0,
    need_dh: bool = True,
    need_dw: bool = True,
    dh_dtype: torch.dtype = torch.bfloat16,
    dw_dtype: torch.dtype = torch.float32,
    token_chunk: int | None = None,
    dh_out: torch.Tensor | None = None,
    dh_mesh_sum=None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``lp_bwd`` on one vocabulary shard: (dH [T, d] partial over this shard, dW [Vs, d]).

    With ``dh_mesh_sum`` (a ``sharding.DhSumBuffer`` with at least T rows; every rank makes
    the same call, its counters zero, and zeroes them again and calls ``peer_barrier`` after it)
    this is ``lp_bwd_sum``: the returned dH is this rank's bf16 copy, which holds the sum over
    the mesh's shards once that barrier has passed.
    """
    dev = _require_cuda(embed, hidden, targets, norm, grad_logp)
    _check_bf16("embedding", embed)
    _check_bf16("hidden", hidden)
    if dh_dtype not in (torch.bfloat16, torch.float32) or dw_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("dH / dW dtypes must be bf16 or f32")
    lib = _lib.load()
    h2, ldh = _rows(hidden)
    T, d = h2.shape
    Vs = embed.shape[0]
    w = embed if embed.is_contiguous() else embed.contiguous()
    y = targets.reshape(-1).to(torch.int32).contiguous()
    g = grad_logp.reshape(-1).to(torch.float32).contiguous()
    nrm = norm.reshape(2, -1).to(torch.float32).contiguous()
    flags = 0
    dH = dW = None
    if need_dh and dh_mesh_sum is not None:
        if dh_mesh_sum.rows < T or dh_mesh_sum.d != d or dh_dtype != torch.bfloat16:
            raise ValueError("dh_mesh_sum needs a buffer of at least [T, d] rows and a bf16 dH")
        dH = dh_mesh_sum.local(T)
    elif need_dh:
        if dh_out is not None:
            if dh_out.shape != (T, d) or dh_out.dtype != dh_dtype or dh_out.stride(-1) != 1:
                raise ValueError("dh_out must be a [T, d] row-major tensor of dh_dtype")
            dH = dh_out
        else:
            dH = torch.empty((T, d), dtype=dh_dtype, device=dev)
        if dh_dtype == torch.float32:
            flags |= _lib.LP_BWD_DH_F32
    else:
        flags |= _lib.LP_BWD_NO_DH
    if need_dw:
        dW = torch.empty((Vs, d), dtype=dw_dtype, device=dev)
        if dw_dtype == torch.bfloat16:
            flags |= _lib.LP_BWD_DW_BF16
    else:
        flags |= _lib.LP_BWD_NO_DW
    chunk = int(token_chunk) if token_chunk else 0
    ws, wsp, wsn = _workspace(lib.lp_bwd_workspace_bytes(T, d, Vs, chunk, flags), dev)
    cap = float(softcap) if softcap is not None else 0.0
    ld_dh = int(dH.stride(0)) if dH is not None and T > 1 else d
    if need_dh and dh_mesh_sum is not None:
        from .sharding import peer_timeout_ms  # noqa: PLC0415

        m = dh_mesh_sum
        rc = lib.lp_bwd_sum(
            _stream(dev), _ptr(h2), T, d, ldh, _ptr(w), Vs, int(vocab_offset), _ptr(y), cap, _ptr(nrm), _ptr(g),
            _ptr(dH), ctypes.c_void_p(m.dh_mc), ld_dh, _ptr(m.counters), ctypes.c_void_p(m.counters_mc), m.rank,
            m.world, peer_timeout_ms(), _ptr(dW), flags, chunk, wsp, wsn,
        )
        _lib.check(rc, "lp_bwd_sum")
        return dH, dW
    rc = lib.lp_bwd(
        _stream(dev), _ptr(h2), T, d, ldh, _ptr(w), Vs, int(vocab_offset), _ptr(y), cap, _ptr(nrm), _ptr(g), _ptr(dH),
        ld_dh, _ptr(dW), flags, chunk, wsp, wsn,
    )
    _lib.check(rc, "lp_bwd")
    return dH, dW


def compact(
    mask: torch.Tensor,
    hidden: torch.Tensor | None = None,
    ids: torch.Tensor | None = None,
    *,
    row_offset: int = 0,
):
    """``lp_compact``: valid slots of ``mask`` [B, N] in slot order.

    With ``hidden`` [B, S, d] (bf16) and ``ids`` [B, N], also gathers the rows
    ``hidden[b, j + row_offset]`` and targets ``ids[b, j]`` of the valid slots. Returns
    ``(H_c [B*N, d] | None, y_c [B*N] | None, idx [B*N], pos [B*N], count [1])``; only the
    first ``count`` rows of H_c / y_c / idx are meaningful.
    """
    dev = _require_cuda(mask, hidden, ids)
    lib = _lib.load()
    if mask.ndim != 2:
        raise ValueError(f"mask must be [B, N], got {tuple(mask.shape)}")
    B, N = mask.shape
    m = mask.to(torch.uint8).contiguous()
    idx = torch.empty((B * N,), dtype=torch.int32, device=dev)
    pos = torch.empty((B * N,), dtype=torch.int32, device=dev)
    count = torch.empty((1,), dtype=torch.int32, device=dev)
    Hc = yc = None
    hb = hr = d = 0
    if hidden is not None:
        _check_bf16("hidden", hidden)
        if hidden.ndim != 3 or hidden.shape[0] != B or hidden.stride(-1) != 1:
            raise ValueError("hidden must be [B, S, d] with unit last stride")
        if row_offset < 0 or row_offset + N > hidden.shape[1]:
            raise ValueError("row_offset + N exceeds the hidden sequence length")
        d = hidden.shape[-1]
        hb, hr = hidden.stride(0), hidden.stride(1)
        Hc = torch.empty((B * N, d), dtype=torch.bfloat16, device=dev)
        if ids is not None:
            if ids.shape != (B, N):
                raise ValueError("ids must match the mask shape")
            ids = ids.to(torch.int32).contiguous()
            yc = torch.empty((B * N,), dtype=torch.int32, device=dev)

    def call(stream):
        ws, wsp, wsn = _workspace(lib.lp_compact_workspace_bytes(B, N), dev)
        return lib.lp_compact(
            stream, _ptr(m), B, N, _ptr(hidden), hb, hr, int(row_offset), d, _ptr(ids), _ptr(Hc), _ptr(yc), _ptr(idx),
            _ptr(pos), _ptr(count), wsp, wsn,
        )

    _on_device(dev, "lp_compact", call)
    return Hc, yc, idx, pos, count


def scatter_rows(src: torch.Tensor, pos: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """``lp_scatter_rows``: out row s = src[pos[s]] where pos[s] >= 0, else 0.

    ``out`` is [slots] / [slots, width] or a strided [B, N, width] view (slot s = b * N + j),
    e.g. the response slice of a [B, S, d] gradient. Also serves as a row gather
    (``pos`` = source row of every output row). f32 ``src`` may be written to a bf16 ``out``.
    """
    dev = _require_cuda(src, pos, out)
    lib = _lib.load()
    if src.dtype not in (torch.bfloat16, torch.float32) or not (
        src.dtype == out.dtype or (src.dtype == torch.float32 and out.dtype == torch.bfloat16)
    ):
        raise ValueError("src / out must share a bf16 or f32 dtype, or be f32 -> bf16")
    if out.ndim == 3:
        B, N, width = out.shape
        rows_per_group, group_stride, row_stride = N, int(out.stride(0)), int(out.stride(1))
        if out.stride(2) != 1:
            raise ValueError("scatter needs unit column stride")
    else:
        o2 = out.reshape(out.shape[0], -1) if out.ndim > 1 else out.reshape(-1, 1)
        if o2.stride(-1) != 1:
            raise ValueError("scatter needs unit column stride")
        B, (N, width) = 1, o2.shape
        rows_per_group, row_stride = N, int(o2.stride(0))
        group_stride = N * row_stride
    s2 = src.reshape(src.shape[0], width)
    slots = B * N
    if s2.stride(-1) != 1:
        s2 = s2.contiguous()
    if pos.numel() != slots or s2.shape[1] != width:
        raise ValueError("pos / src / out shapes disagree")
    p = pos.to(torch.int32).contiguous()
    # an empty src is never read (every pos is -1); any valid pointer stands in for it
    src_ptr = _ptr(s2) if s2.shape[0] > 0 else _ptr(out)
    src_ld = int(s2.stride(0)) if s2.shape[0] > 0 else width
    _on_device(dev, "lp_scatter_rows", lambda stream: lib.lp_scatter_rows(
        stream, src_ptr, src_ld, _ptr(p), slots, width, src.element_size(), _ptr(out), row_stride, rows_per_group,
        group_stride, out.element_size(),
    ))
    return out


def peer_barrier(buf, timeout_ms: int) -> None:
    """``lp_peer_barrier`` over the signal pads of a ``sharding.DhSumBuffer``, on the current
    stream of its device (every rank of the mesh must make the same calls in the same order)."""
    lib = _lib.load()
    rc = lib.lp_peer_barrier(_stream(buf.device), ctypes.c_void_p(buf.pads_dev), buf.rank, buf.world, buf.channel,
                             int(timeout_ms))
    _lib.check(rc, "lp_peer_barrier")


def bwd_sum_counters(rows: int) -> int:
    """Number of u32 row-block counters ``lp_bwd_sum`` uses for ``rows`` rows."""
    return int(_lib.load().lp_bwd_sum_counters(int(rows)))
