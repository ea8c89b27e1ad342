"""Operators at the two ends of the vocabulary, as cases that can be timed and whose outputs can be compared.

Kinds of case:

  logprobs   ``kernels.k_token_logprobs``: log probability of given tokens under the rows' softmax at a temperature, the rows'
             entropy and their most likely alternatives; with ``backward``, the gradient of all three
  distill    ``kernels.k_distill_topk``: KL divergence from a teacher of whom only the most likely tokens' log probabilities are
             kept (renormalised over them, or with the rest of the vocabulary as one more outcome), and its gradient
  embed      ``kernels.k_embedding``: scaled rows of a table; with ``backward``, the table's gradient

Logits look like a language model's: normal noise, a bias that falls with the token's rank, and one token per row that the
model expects.  Token ids are Zipf(1.1), as the rest of the benchmarks' are.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = 8192 * 32768 * 2          # bytes of the largest logits
IGNORE = -100


# --------------------------------------------------------------------------- the cases
def listed():
    logprobs = dict(kind="logprobs", dtype="bf16", k=0, temperature=1.0, backward=False, banned=0.0, ignored=0.0)
    distill = dict(kind="distill", dtype="bf16", temperature=1.0, tail=False, unused=0.0)
    embed = dict(kind="embed", dtype="bf16", scale=1.0, padding=False, backward=True)
    return [
        # one decoded token and its alternatives, as a server reports them: latency
        dict(logprobs, name="logprobs_one_token", rows=1, V=50257, k=20),
        # one decoding step of a batch under a grammar that bans most of the vocabulary
        dict(logprobs, name="logprobs_decode_batch", rows=61, V=131072, dtype="fp32", k=8, temperature=0.7, banned=0.6),
        # a teacher's pass over the headline model's batch (128 x 64 tokens): what the student's loss keeps of it
        dict(logprobs, name="logprobs_teacher", rows=8192, V=2048, k=32, temperature=2.0),
        # the same for the scale-up model: large vocabulary, long list
        dict(logprobs, name="logprobs_teacher_wide", rows=8192, V=32768, k=64),
        # a policy update: log probabilities and an entropy bonus of padded answers, forward and backward, odd vocabulary
        dict(logprobs, name="logprobs_policy", rows=1531, V=50257, banned=0.02, ignored=0.2, backward=True),
        # distillation of the smallest model anybody trains here: latency
        dict(distill, name="distill_small", rows=256, V=2048, dtype="fp32", k=16),
        # distillation of the scale-up model's batch at a temperature, the rest of the vocabulary as one outcome
        dict(distill, name="distill_wide", rows=8192, V=32768, k=64, temperature=2.0, tail=True),
        # stored teacher lists of uneven length, odd vocabulary, half precision
        dict(distill, name="distill_ragged", rows=1999, V=50257, dtype="fp16", k=50, unused=0.3),
        # the embedding of a few decoded tokens: latency
        dict(embed, name="embed_few_tokens", tokens=16, V=32768, d=1024, scale=32.0, backward=False),
        # a training batch of the scale-up model
        dict(embed, name="embed_wide", tokens=8192, V=32768, d=1024, scale=32.0),
        # a long batch on sizes that are no multiple of anything, padded at the end of its samples
        dict(embed, name="embed_ragged", tokens=33333, V=50257, d=770, dtype="fp32", scale=27.75, padding=True),
        # the longest batch, a large table
        dict(embed, name="embed_long", tokens=131072, V=131072, d=2048),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "distill", "embed"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    if kind == "embed":
        d = _log_uniform(rng, 32, 2048)
        if rng.random() < 0.7:
            d = (d + 7) // 8 * 8
        V = _log_uniform(rng, 256, min(131072, LARGEST // (d * size)))
        tokens = _log_uniform(rng, 1, min(131072, LARGEST // (d * size)))
        return dict(kind=kind, dtype=dtype, tokens=tokens, V=V, d=d, scale=rng.choice([1.0, round(rng.uniform(0.1, 40.0), 3)]), padding=rng.random() < 0.4,
                    backward=rng.random() < 0.7)
    V = _log_uniform(rng, 256, 131072)
    if rng.random() < 0.5:
        V = (V + 7) // 8 * 8
    rows = _log_uniform(rng, 1, min(16384, LARGEST // (V * size)))
    temperature = rng.choice([1.0, round(rng.uniform(0.5, 4.0), 2)])
    if kind == "distill":
        return dict(kind=kind, dtype=dtype, rows=rows, V=V, k=_log_uniform(rng, 1, 128), temperature=temperature, tail=rng.random() < 0.5,
                    unused=rng.choice([0.0, 0.25]))
    return dict(kind=kind, dtype=dtype, rows=rows, V=V, k=rng.choice([0, _log_uniform(rng, 1, 128)]), temperature=temperature, backward=rng.random() < 0.5,
                banned=rng.choice([0.0, 0.0, 0.5]), ignored=rng.choice([0.0, 0.15]))


# --------------------------------------------------------------------------- inputs
def _zipf(shape, V, gen):
    weight = torch.arange(1, V + 1, dtype=torch.float64, device=DEV).pow(-1.1)
    cdf = weight.cumsum(0) / weight.sum()
    return torch.searchsorted(cdf, torch.rand(shape, dtype=torch.float64, device=DEV, generator=gen)).clamp_(max=V - 1)


def _logits(rows, V, expected, gen):
    x = torch.randn(rows, V, device=DEV, generator=gen).mul_(2.0)
    x.sub_(torch.arange(1, V + 1, dtype=torch.float32, device=DEV).log_())
    x.scatter_add_(1, expected[:, None], 4.0 + 3.0 * torch.randn(rows, 1, device=DEV, generator=gen))
    return x


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "embed":
        N, V, d = case["tokens"], case["V"], case["d"]
        ids = _zipf((N,), V, gen)
        pad = 0 if case["padding"] else None
        if case["padding"]:
            ids[torch.rand(N, device=DEV, generator=gen) < 0.15] = 0
        s = dict(ids=ids, weight=torch.randn(V, d, device=DEV, generator=gen).mul_(0.02).to(dtype), scale=case["scale"], pad=pad)
        if case["backward"]:
            s["dy"] = torch.randn(N, d, device=DEV, generator=gen).mul_(1e-3).to(dtype)
        return dict(case=case, **s)
    rows, V, k = case["rows"], case["V"], case["k"]
    scale = (32768.0 if dtype == torch.float16 else 1.0) / rows         # half precision is trained with its loss scaled
    expected = _zipf((rows,), V, gen)
    x = _logits(rows, V, expected, gen)
    if case["kind"] == "distill":
        k = min(k, V)
        teacher = 0.8 * x + torch.randn(rows, V, device=DEV, generator=gen)
        teacher.div_(case["temperature"])
        top, ids = teacher.topk(k, dim=-1)
        logprobs = top - teacher.logsumexp(-1, keepdim=True)
        if case["unused"]:              # lists of uneven length, some of them empty
            length = (torch.rand(rows, 1, device=DEV, generator=gen) > case["unused"]) * torch.randint(0, 2 * k, (rows, 1), device=DEV, generator=gen)
            ids = ids.masked_fill(torch.arange(k, device=DEV) >= length, -1)
        return dict(case=case, logits=x.to(dtype), teacher=logprobs, ids=ids, dloss=scale * torch.rand(rows, device=DEV, generator=gen))
    tokens = torch.where(torch.rand(rows, device=DEV, generator=gen) < 0.7, expected, _zipf((rows,), V, gen))
    if case["banned"]:
        ban = torch.rand(rows, V, device=DEV, generator=gen) < case["banned"]
        ban.scatter_(1, tokens[:, None], False)
        x.masked_fill_(ban, -math.inf)
        del ban
    if case["ignored"]:
        tokens = tokens.masked_fill(torch.rand(rows, device=DEV, generator=gen) < case["ignored"], IGNORE)
    s = dict(logits=x.to(dtype), tokens=tokens, k=min(k, V))
    if case["backward"]:
        s["grads"] = [scale * torch.randn(rows, device=DEV, generator=gen), 0.1 * scale * torch.rand(rows, device=DEV, generator=gen)]
        if s["k"]:
            s["grads"].append(scale / s["k"] * torch.randn(rows, s["k"], device=DEV, generator=gen))
    return dict(case=case, **s)


# --------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"logprobs": _own_logprobs, "distill": _own_distill, "embed": _own_embed}[kind](state)
    return {"logprobs": _plain_logprobs, "distill": _plain_distill, "embed": _plain_embed}[kind](state)


def _own_logprobs(s):
    from speedup_thingy_b200 import kernels as K

    case, backward = s["case"], "grads" in s
    x = s["logits"].detach().requires_grad_(backward)
    out = K.k_token_logprobs(x, s["tokens"], top_k=s["k"], temperature=case["temperature"], ignore_index=IGNORE)
    res = dict(logprob=out.logprob.detach(), entropy=out.entropy.detach())
    if s["k"]:
        res |= dict(top_logprobs=out.top_logprobs.detach(), top_ids=out.top_ids)
    if backward:
        outs = [out.logprob, out.entropy] + ([out.top_logprobs] if s["k"] else [])
        res["dlogits"], = torch.autograd.grad(outs, [x], s["grads"])
    return res


def _own_distill(s):
    from speedup_thingy_b200 import kernels as K

    case = s["case"]
    x = s["logits"].detach().requires_grad_()
    loss = K.k_distill_topk(x, s["teacher"], s["ids"], temperature=case["temperature"], tail=case["tail"])
    dx, = torch.autograd.grad([loss], [x], [s["dloss"]])
    return dict(loss=loss.detach(), dlogits=dx)


def _own_embed(s):
    from speedup_thingy_b200 import kernels as K

    w = s["weight"].detach().requires_grad_("dy" in s)
    y = K.k_embedding(s["ids"], w, scale=s["scale"], padding_idx=s["pad"])
    if "dy" not in s:
        return dict(y=y)
    dw, = torch.autograd.grad([y], [w], [s["dy"]])
    return dict(y=y.detach(), dweight=dw)


def _plain_logprobs(s):
    x, tokens, k, T = s["logits"], s["tokens"], s["k"], s["case"]["temperature"]
    keep = tokens != IGNORE
    at = tokens.clamp(min=0)[:, None]
    v = x.float()
    z = (v - v.amax(-1, keepdim=True)) / T
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    p, logp = e / total, z - total.log()
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    zero = torch.zeros((), device=DEV)
    out = dict(logprob=torch.where(keep, logp.gather(1, at)[:, 0], zero), entropy=torch.where(keep, entropy, zero))
    if k:
        # one whole number per logit that orders by value, then by the lower index
        bits = (v + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + torch.arange(x.shape[1] - 1, -1, -1, device=DEV)
        ids = key.topk(k, dim=-1)[1]
        out["top_logprobs"] = torch.where(keep[:, None], logp.gather(1, ids), zero)
        out["top_ids"] = torch.where(keep[:, None], ids, -1)
    if "grads" in s:
        g, gh = s["grads"][0][:, None], s["grads"][1][:, None]
        gt = s["grads"][2] if k else None
        total_g = g + gt.sum(-1, keepdim=True) if k else g
        dz = -total_g * p - gh * (plogp + p * entropy[:, None])
        dz.scatter_add_(1, at, g)
        if k:
            dz.scatter_add_(1, ids, gt)
        out["dlogits"] = torch.where(keep[:, None], dz / T, zero).to(x.dtype)
    return out


def _plain_distill(s):
    x, ids, T, tail = s["logits"], s["ids"], s["case"]["temperature"], s["case"]["tail"]
    used = ids >= 0
    at = ids.clamp(min=0)
    some = used.any(-1)
    # the lists and the sums in 64 bits: what a teacher leaves to the rest of the vocabulary is a small difference, and so is the loss
    t = s["teacher"].double().masked_fill(~used, -math.inf)
    if tail:
        q = t.exp()
        rest = (1.0 - q.sum(-1)).clamp(min=0.0)
        logq = t
    else:
        logq = t - torch.where(some, t.amax(-1), 0.0)[:, None]
        logq = logq - torch.where(some, logq.exp().sum(-1), 1.0).log()[:, None]
        q = logq.exp()
    v = x.float()
    z = (v - v.amax(-1, keepdim=True)) / T
    e = z.exp()
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    p = e / total.float()
    logp = z.gather(1, at) - total.log()
    loss = torch.where(q > 0, q * (logq - logp), 0.0).sum(-1)
    if tail:
        listed = torch.zeros_like(e).scatter_add_(1, at, used.float()) > 0
        others = e.masked_fill(listed, 0.0).sum(-1, dtype=torch.float64)
        logr = (others / total[:, 0]).log()
        loss = loss + torch.where(rest > 0, rest * (rest.log() - logr), 0.0)
        mass = q.sum(-1) + rest
        dz = p * torch.where(listed, mass[:, None].float(), (mass - rest * total[:, 0] / others)[:, None].float())
    else:
        dz = p * q.sum(-1, keepdim=True).float()
    dz.scatter_add_(1, at, -q.float())
    zero = torch.zeros((), device=DEV)
    scale = torch.where(some, s["dloss"] * T, zero)
    return dict(loss=torch.where(some, loss * (T * T), 0.0).float(), dlogits=(dz * scale[:, None]).to(x.dtype))


def _plain_embed(s):
    w, ids, scale = s["weight"], s["ids"], s["scale"]
    out = dict(y=(w[ids].float() * scale).to(w.dtype))
    if "dy" in s:
        dy = s["dy"].float()
        if s["pad"] is not None:
            dy = dy * (ids != s["pad"])[:, None]
        dw = torch.zeros(w.shape, device=DEV).index_add_(0, ids, dy)
        out["dweight"] = (dw * scale).to(w.dtype)
    return out


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "embed":
        N, V, d = case["tokens"], case["V"], case["d"]
        weight = torch.arange(1, V + 1, dtype=torch.float64).pow(-1.1)
        distinct = float((1 - (1 - weight / weight.sum()).pow(N)).sum())
        moved = 8 * N + (distinct + N) * d * size
        return {"bytes": moved + ((N + V) * d * size if case["backward"] else 0), "flops": N * d * (2 if case["backward"] else 1)}
    rows, V, k = case["rows"], case["V"], min(case["k"], case["V"])
    if case["kind"] == "distill":
        kept = rows * (1 - case["unused"])
        return {"bytes": kept * V * size + rows * (V * size + 12 * k + 8), "flops": kept * V * 8}
    kept = rows * (1 - case["ignored"])
    moved = kept * V * size + rows * (16 + 12 * k)
    if case["backward"]:
        moved += rows * (V * size + 8 + 4 * k)
    return {"bytes": moved, "flops": kept * V * (14 if case["backward"] else 6)}


# --------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "embed":
        return _exact_embed(state)
    one = _exact_logprobs if case["kind"] == "logprobs" else _exact_distill
    step = max(1, (1 << 24) // case["V"])
    parts = [one(state, slice(a, a + step)) for a in range(0, case["rows"], step)]
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _exact_logprobs(state, rows):
    logits, tokens = state["logits"][rows].double(), state["tokens"][rows]
    T, k, n = state["case"]["temperature"], state["k"], tokens.numel()
    ignored = tokens == IGNORE
    logp = torch.log_softmax(logits / T, -1)
    p = logp.exp()
    finite = logp.masked_fill(p == 0, 0.0)                 # 0 log 0 = 0
    entropy = -(p * finite).sum(-1)
    target = tokens.masked_fill(ignored, 0)
    line = torch.arange(n, device=DEV)
    out = {"logprob": logp[line, target].masked_fill(ignored, 0.0), "entropy": entropy.masked_fill(ignored, 0.0)}
    order = logits.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    if k:
        out["top_logprobs"] = logp.gather(1, order).masked_fill(ignored[:, None], 0.0)
        out["top_ids"] = order.masked_fill(ignored[:, None], -1)
    if "grads" in state:
        # d logp_i / d x_j = (1[i = j] - p_j) / T;  d H / d x_j = -p_j (log p_j + H) / T
        upstream = torch.zeros_like(logits)
        upstream[line, target] += state["grads"][0][rows].double()
        if k:
            upstream.scatter_add_(1, order, state["grads"][2][rows].double())
        dx = upstream - p * upstream.sum(-1, keepdim=True)
        dx -= state["grads"][1][rows].double()[:, None] * p * (finite + entropy[:, None])
        out["dlogits"] = (dx / T).masked_fill(ignored[:, None], 0.0)
    return out


def _exact_distill(state, rows):
    logits, ids, teacher = state["logits"][rows].double(), state["ids"][rows], state["teacher"][rows].double()
    T, tail = state["case"]["temperature"], state["case"]["tail"]
    unused = ids < 0
    empty = unused.all(-1)
    # the teacher over the whole vocabulary: nothing outside its list
    column = ids.masked_fill(unused, logits.shape[1])
    q = torch.zeros(logits.shape[0], logits.shape[1] + 1, dtype=torch.float64, device=DEV)
    q.scatter_(1, column, teacher.exp())
    member = torch.zeros_like(q, dtype=torch.bool).scatter_(1, column, True)[:, :-1]
    q = q[:, :-1]
    if not tail:
        q = q / q.sum(-1, keepdim=True).masked_fill(empty[:, None], 1.0)
    logp = torch.log_softmax(logits / T, -1)
    p = logp.exp()
    loss = torch.special.xlogy(q, q).sum(-1) - (q * logp).sum(-1)
    dz = p * q.sum(-1, keepdim=True) - q
    if tail:
        r = (1.0 - q.sum(-1)).clamp(min=0.0)
        outside = p.masked_fill(member, 0.0)
        pr = outside.sum(-1)
        loss += torch.special.xlogy(r, r) - torch.special.xlogy(r, pr)
        dz += r[:, None] * (p - outside / pr[:, None])
    loss = (T * T * loss).masked_fill(empty, 0.0)
    dx = (T * state["dloss"][rows].double()[:, None] * dz).masked_fill(empty[:, None], 0.0)
    return {"loss": loss, "dlogits": dx}


def _exact_embed(state):
    ids, scale = state["ids"], state["scale"]
    table = state["weight"].double()
    out = {"y": table.index_select(0, ids) * scale}
    if "dy" in state:
        keep = torch.ones_like(ids, dtype=torch.bool) if state["pad"] is None else ids != state["pad"]
        out["dweight"] = torch.zeros_like(table).index_add_(0, ids[keep], state["dy"][keep].double() * scale)
    return out
