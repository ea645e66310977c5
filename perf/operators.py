"""The distribution operators of the LM head, as they are measured: what they are given, their plain form, the
framework's calls, and their values in 64 bits.

``logps``  : ``token_logps_and_entropy``, log-probabilities of one or several given tokens per position and the
             entropy of the position's distribution, with the gradients of both.
``top``    : ``top_token_logps``, the k most likely tokens of each position with their log-probabilities, the entropy
             and the log-probability of one given token.
``sample`` : ``sample_top_k``, one token per row drawn from the temperature / top-k / top-p filtered distribution by a
             given uniform number, with its log-probability under the unfiltered policy.

All of them work on softcap(hidden . embed^T), softcap(x) = c tanh(x / c) or x, over the whole vocabulary.
"""

import math

import torch

#: False: ``run`` computes the plain form; True: it makes the framework's calls.
own = False

_VOCAB, _WIDTH = 262144, 2048  # the head that the benchmark is quoted on


def _case(name, op, tokens, vocab, width, softcap, **more):
    return {"name": name, "op": op, "tokens": tokens, "vocab": vocab, "width": width, "softcap": softcap, **more}


def listed():
    return [
        # a policy update on one microbatch: log-probabilities with an entropy bonus, gradients for hidden states and head
        _case("logps_train", "logps", 4096, _VOCAB, _WIDTH, 30.0, per_position=0, grad="both"),
        # distillation on a teacher's 20 alternatives per position (short lists padded), frozen head
        _case("logps_distill", "logps", 1021, _VOCAB, _WIDTH, 30.0, per_position=20, grad="hidden"),
        # one rank's share of the vocabulary (eight ranks), no softcap, four tokens per position
        _case("logps_shard", "logps", 2051, _VOCAB // 8, _WIDTH, 0.0, per_position=4, grad="both"),
        # old-policy log-probabilities and entropies of a batch of rollouts, no gradients
        _case("logps_score", "logps", 6000, _VOCAB, _WIDTH, 30.0, per_position=0, grad="none"),
        # a tiny model's training step, where the call itself is what costs
        _case("logps_tiny", "logps", 37, 1036, 160, 0.0, per_position=0, grad="both"),
        # one decoded position whose 20 alternatives are reported
        _case("top_one", "top", 1, _VOCAB, _WIDTH, 30.0, k=20),
        # a teacher's 64 alternatives for the positions of a few sequences
        _case("top_teacher", "top", 2048, _VOCAB, _WIDTH, 30.0, k=64),
        # alternatives of a short prompt under a small head
        _case("top_small", "top", 19, 4099, 136, 0.0, k=5),
        # one sequence being decoded
        _case("sample_one", "sample", 1, _VOCAB, _WIDTH, 30.0, k=64, temperature=1.0, top_p=0.95),
        # a rollout batch being decoded
        _case("sample_batch", "sample", 128, _VOCAB, _WIDTH, 30.0, k=64, temperature=0.7, top_p=0.95),
        # a ragged batch on a rank's share of the vocabulary, the widest filter, no nucleus
        _case("sample_wide", "sample", 301, _VOCAB // 8, _WIDTH, 0.0, k=128, temperature=1.3, top_p=1.0),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["logps", "top", "sample"])
    vocab = _log_uniform(rng, 300, _VOCAB)
    width = 8 * _log_uniform(rng, 8, 512)
    most = 4096 * _VOCAB * _WIDTH // (vocab * width) // (1 if op == "logps" else 2)
    tokens = _log_uniform(rng, 1, min(most, {"logps": 8000, "top": 4000, "sample": 512}[op]))
    softcap = rng.choice([0.0, 15.0, 30.0, 50.0])
    case = {"op": op, "tokens": tokens, "vocab": vocab, "width": width, "softcap": softcap}
    if op == "logps":
        return {**case, "per_position": rng.choice([0, 1, 2, 5, 16, 32]), "grad": rng.choice(["both", "both", "hidden", "none"])}
    case["k"] = min(_log_uniform(rng, 1, 128), vocab)
    if op == "sample":
        case |= {"temperature": round(rng.uniform(0.3, 1.5), 3), "top_p": rng.choice([1.0, 0.99, 0.95, 0.8, 0.5])}
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, v, d = case["tokens"], case["vocab"], case["width"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    def whole(high, *shape):
        return torch.randint(high, shape, generator=gen, device="cuda")

    # Logits of spread 0.9, and in every row four tokens that the model thinks likely: between flat and nearly certain.
    embed = (normal(v, d) * (0.9 / math.sqrt(d))).to(torch.bfloat16)
    likely = whole(v, n, 4)
    lift = uniform(n, 4) * (4.0 + 9.0 * uniform(n, 1)) / 0.81
    hidden = (normal(n, d) + torch.einsum("nj,njd->nd", lift, embed[likely].float())).to(torch.bfloat16)
    state = {**case, "embed": embed, "hidden": hidden, "softcap": case["softcap"] or None}

    def chosen(*shape):  # mostly what the model thinks likely, else anything
        picked = torch.gather(likely, 1, whole(4, n, math.prod(shape))).reshape(n, *shape)
        return torch.where(uniform(n, *shape) < 0.7, picked, whole(v, n, *shape))

    if case["op"] == "logps":
        k = case["per_position"]
        if k == 0:
            tokens = chosen()
        else:  # distinct tokens; a position's list may be shorter than k, or empty: -1 is no token
            tokens = (whole(v, n, 1) + torch.arange(k, device="cuda") * max(1, v // k)) % v
            tokens[:, 0] = torch.where(uniform(n) < 0.7, likely[:, 0], tokens[:, 0])
            length = whole(k + 1, n, 1)
            tokens = torch.where((torch.arange(k, device="cuda") < length) | (uniform(n, 1) < 0.7), tokens, -1)
        state["tokens"] = tokens.to(torch.int32)
        kept = uniform(n) < 0.9  # masked positions send no gradient
        state["d_logps"] = normal(*tokens.shape) * kept.reshape(-1, *[1] * (tokens.ndim - 1))
        state["d_entropy"] = 0.3 * normal(n) * kept
    elif case["op"] == "top":
        state["tokens"] = chosen().to(torch.int32)
    else:
        state["uniform"] = uniform(n)
    return state


def _capped(x, c):
    return x if c is None else c * torch.tanh(x / c)


def _log_normaliser(z):
    top = z.amax(-1, keepdim=True)
    return top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))


def _plain_logps(s):
    w, h, c = s["embed"].float(), s["hidden"].float(), s["softcap"]
    z = _capped(h @ w.T, c)
    logp = z - _log_normaliser(z)
    p = torch.exp(logp)
    entropy = -(p * logp).sum(-1)
    tokens = s["tokens"].long().reshape(len(h), -1)
    given = tokens >= 0
    picked = torch.where(given, torch.gather(logp, 1, tokens.clamp(min=0)), 0.0)
    out = {"logps": picked.reshape(s["tokens"].shape), "entropy": entropy}
    if s["grad"] == "none":
        return out
    g = torch.where(given, s["d_logps"].reshape(len(h), -1), 0.0)
    dz = -p * (g.sum(-1, keepdim=True) + s["d_entropy"][:, None] * (logp + entropy[:, None]))
    dz.scatter_add_(1, tokens.clamp(min=0), g)
    if c is not None:
        dz = dz * (1.0 - torch.square(z / c))
    out["d_hidden"] = (dz @ w).to(s["hidden"].dtype)
    if s["grad"] == "both":
        out["d_embed"] = (dz.T @ h).to(s["embed"].dtype)
    return out


def _ranked(raw, k):
    """The k largest of each row in descending order, the lowest index first among equals."""
    some = torch.topk(raw, min(raw.shape[-1], k + 32), dim=-1).indices.sort(dim=-1).values
    order = torch.gather(raw, 1, some).sort(dim=-1, descending=True, stable=True).indices
    return torch.gather(some, 1, order)[:, :k]


def _plain_top(s):
    raw = s["hidden"].double() @ s["embed"].double().T  # 64 bits: neighbours in the order can be very near
    ids = _ranked(raw, s["k"])
    z = _capped(raw.float(), s["softcap"])
    logp = z - _log_normaliser(z)
    return {
        "ids": ids.to(torch.int32),
        "logps": torch.gather(logp, 1, ids),
        "entropy": -(torch.exp(logp) * logp).sum(-1),
        "token_logps": torch.gather(logp, 1, s["tokens"].long()[:, None])[:, 0],
    }


def _plain_sample(s):
    raw = s["hidden"].double() @ s["embed"].double().T
    ids = _ranked(raw, s["k"])
    best = _capped(torch.gather(raw, 1, ids), s["softcap"])
    weight = torch.exp((best - best[:, :1]) / s["temperature"])  # 64 bits: the drawn number may lie next to a border
    upto = weight.cumsum(-1)
    keep = upto - weight < s["top_p"] * upto[:, -1:]
    keep[:, 0] = True
    weight = torch.where(keep, weight, 0.0)
    upto = weight.cumsum(-1)
    place = (upto <= s["uniform"].double()[:, None] * upto[:, -1:]).sum(-1)
    place = torch.minimum(place, keep.sum(-1) - 1)[:, None]
    z = _capped(raw.float(), s["softcap"])
    logp = torch.gather(best, 1, place).float() - _log_normaliser(z)
    return {"token": torch.gather(ids, 1, place)[:, 0].to(torch.int32), "logp": logp[:, 0]}


def _own_logps(s):
    from gemma4_posttrain_jax_b200 import token_logps_and_entropy

    if s["grad"] == "none":
        with torch.no_grad():
            logps, entropy = token_logps_and_entropy(s["embed"], s["hidden"], s["tokens"], softcap=s["softcap"])
        return {"logps": logps, "entropy": entropy}
    hidden = s["hidden"].detach().requires_grad_(True)
    embed = s["embed"].detach().requires_grad_(s["grad"] == "both")
    logps, entropy = token_logps_and_entropy(embed, hidden, s["tokens"], softcap=s["softcap"])
    wanted = [hidden, embed] if s["grad"] == "both" else [hidden]
    grads = torch.autograd.grad([logps, entropy], wanted, [s["d_logps"], s["d_entropy"]])
    return {"logps": logps.detach(), "entropy": entropy.detach(), **dict(zip(["d_hidden", "d_embed"], grads))}


def _own_top(s):
    from gemma4_posttrain_jax_b200 import top_token_logps

    got = top_token_logps(s["embed"], s["hidden"], s["softcap"], s["k"], tokens=s["tokens"])
    return {"ids": got.ids, "logps": got.logps, "entropy": got.entropy, "token_logps": got.token_logps}


def _own_sample(s):
    from gemma4_posttrain_jax_b200 import sample_top_k

    token, logp = sample_top_k(
        s["embed"], s["hidden"], s["softcap"], s["uniform"],
        temperature=s["temperature"], top_k=s["k"], top_p=s["top_p"],
    )
    return {"token": token, "logp": logp}


def run(state):
    if own:
        return {"logps": _own_logps, "top": _own_top, "sample": _own_sample}[state["op"]](state)
    return {"logps": _plain_logps, "top": _plain_top, "sample": _plain_sample}[state["op"]](state)


def work(case):
    n, v, d = case["tokens"], case["vocab"], case["width"]
    nbytes, flops = 2 * v * d + 2 * n * d, 2.0 * n * v * d
    if case["op"] == "logps":
        k = max(1, case["per_position"])
        nbytes += 8 * n * k + 4 * n
        if case["grad"] != "none":  # the logits once, and a product for each gradient
            nbytes += 4 * n * k + 4 * n + 2 * n * d + (2 * v * d if case["grad"] == "both" else 0)
            flops *= 3.0 if case["grad"] == "both" else 2.0
    elif case["op"] == "top":
        nbytes += 8 * n * case["k"] + 12 * n
    else:
        nbytes += 12 * n
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    """Rows in blocks, in 64 bits; the gradients by differentiating the definition."""
    s = prepare(case, seed)
    n, op = case["tokens"], case["op"]
    embed = s["embed"].double().requires_grad_(op == "logps" and case["grad"] == "both")
    parts = []
    for lo in range(0, n, 512):
        hi = min(n, lo + 512)
        hidden = s["hidden"][lo:hi].double().requires_grad_(op == "logps" and case["grad"] != "none")
        logits = torch.matmul(hidden, embed.transpose(0, 1))
        if s["softcap"] is not None:
            logits = torch.tanh(logits / s["softcap"]) * s["softcap"]
        logp = torch.log_softmax(logits, dim=-1)
        entropy = torch.distributions.Categorical(logits=logp, validate_args=False).entropy() if op == "logps" else None
        row = {}
        if op == "logps":
            tokens = s["tokens"][lo:hi].long().reshape(hi - lo, -1)
            got = torch.take_along_dim(logp, tokens.clamp(min=0), dim=-1) * (tokens >= 0)
            if case["grad"] != "none":
                sent = (got * s["d_logps"][lo:hi].double().reshape(got.shape)).sum()
                (sent + (entropy * s["d_entropy"][lo:hi].double()).sum()).backward()
                row["d_hidden"] = hidden.grad
            row |= {"logps": got.detach().reshape(s["tokens"][lo:hi].shape), "entropy": entropy.detach()}
        else:
            order = _exact_order(logits, case["k"])
            if op == "top":
                at = s["tokens"][lo:hi].long().unsqueeze(-1)
                row = {
                    "ids": order.to(torch.int32), "logps": torch.take_along_dim(logp, order, dim=-1),
                    "entropy": -torch.special.xlogy(logp.exp(), logp.exp()).sum(-1),
                    "token_logps": torch.take_along_dim(logp, at, dim=-1).squeeze(-1),
                }
            else:
                scores = torch.take_along_dim(logits, order, dim=-1) / case["temperature"]
                prob = torch.softmax(scores, dim=-1)
                before = prob.cumsum(-1) - prob
                prob = prob.masked_fill((before >= case["top_p"]) & (torch.arange(case["k"], device="cuda") > 0), 0.0)
                prob = prob / prob.sum(-1, keepdim=True)
                at = torch.searchsorted(prob.cumsum(-1), s["uniform"][lo:hi].double().unsqueeze(-1), right=True)
                at = torch.minimum(at, (prob > 0).sum(-1, keepdim=True) - 1)
                token = torch.take_along_dim(order, at, dim=-1)
                row = {"token": token.squeeze(-1).to(torch.int32), "logp": torch.take_along_dim(logp, token, dim=-1).squeeze(-1)}
        parts.append({name: value.detach() for name, value in row.items()})
    out = {name: torch.cat([part[name] for part in parts]) for name in parts[0]}
    if embed.grad is not None:
        out["d_embed"] = embed.grad
    return out


def _exact_order(logits, k):
    return torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
