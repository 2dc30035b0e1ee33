"""The operators at the two ends of the language model, with the inputs a user's program has in
hand, the call itself in elementary torch operations and through the framework, and the same
results in float64.

* ``embed``        -- the embedding lookup without gradients (serving, evaluation);
* ``embed_train``  -- the lookup and the table's gradient;
* ``logprob``      -- log-probabilities of given tokens, the entropy and the best alternatives;
* ``logprob_train``-- log-probabilities and entropy with the gradient of the logits;
* ``distill``      -- the distillation loss from a teacher's best tokens (validation);
* ``distill_train``-- the same with the gradient of the student's logits.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100


def listed():
    return [
        # one token for one user of the byte LM: the smallest call, latency alone
        dict(name="embed_b1", kind="embed", vocab=256, width=768, batch=1, length=1, dtype="f32",
             scale=1.0, padded=0.0),
        # the byte LM's training batch: few ids, the commonest on a sixth of all positions
        dict(name="embed_train_bytes", kind="embed_train", vocab=256, width=768, batch=16,
             length=2048, dtype="f32", scale=1.0, padded=0.0),
        # a subword vocabulary, scaled embeddings, documents of uneven length padded to the longest
        dict(name="embed_train_subwords", kind="embed_train", vocab=50001, width=1024, batch=8,
             length=2048, dtype="f32", scale=32.0, padded=0.2),
        # a bf16 table of odd width and a short ragged batch
        dict(name="embed_train_bf16_odd", kind="embed_train", vocab=32003, width=515, batch=3,
             length=259, dtype="bf16", scale=22.7, padded=0.1),
        # interactive serving: the drawn token's log-probability and 20 alternatives, one row
        dict(name="logprob_b1", kind="logprob", vocab=131072, batch=1, length=1, dtype="f32", top=20,
             temperature=1.0, padded=0.0),
        # scoring text with the byte LM, five alternatives at each byte
        dict(name="logprob_bytes", kind="logprob", vocab=256, batch=16, length=2048, dtype="f32",
             top=5, temperature=1.0, padded=0.0),
        # a teacher's pass that leaves its 64 best tokens: bf16 logits, an odd vocabulary
        dict(name="logprob_teacher", kind="logprob", vocab=50001, batch=3, length=333, dtype="bf16",
             top=64, temperature=1.5, padded=0.1),
        # policy-gradient training: log-probabilities of drawn tokens and an entropy bonus
        dict(name="logprob_train_subwords", kind="logprob_train", vocab=32000, batch=4, length=2048,
             dtype="f32", top=0, temperature=0.8, padded=0.1),
        # distilling the byte LM: every position's 16 best bytes and the true byte
        dict(name="distill_train_bytes", kind="distill_train", vocab=256, batch=16, length=2048,
             dtype="f32", teacher=16, temperature=2.0, hard=True, padded=0.0),
        # distilling a subword model, the largest call: 32 teacher tokens, mixed with the true one
        dict(name="distill_train_subwords", kind="distill_train", vocab=50001, batch=4, length=2048,
             dtype="f32", teacher=32, temperature=2.0, hard=True, padded=0.1),
        # the same in bf16 at temperature one, no true tokens
        dict(name="distill_train_bf16", kind="distill_train", vocab=65536, batch=2, length=1024,
             dtype="bf16", teacher=64, temperature=1.0, hard=False, padded=0.0),
        # a validation batch of few rows
        dict(name="distill_rows", kind="distill", vocab=50001, batch=1, length=37, dtype="f32",
             teacher=32, temperature=2.0, hard=True, padded=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_train", "embed_train", "logprob", "logprob", "logprob_train",
                       "distill", "distill_train", "distill_train"])
    vocab = 256 if rng.random() < 0.25 else _log_int(rng, 200, 131072)
    case = dict(kind=kind, vocab=vocab, dtype=rng.choice(["f32", "f32", "bf16"]),
                padded=rng.choice([0.0, 0.0, 0.1, 0.3]))
    if kind.startswith("embed"):
        width = rng.choice([64 * rng.randint(1, 24), 64 * rng.randint(1, 24), _log_int(rng, 17, 1536)])
        rows = _log_int(rng, 1, 32768)
        case.update(width=width, scale=rng.choice([1.0, round(math.sqrt(width), 1)]))
    else:
        # no more logits than the largest listed case has
        rows = _log_int(rng, 1, min(32768, max(1, 4 * 2048 * 50001 // vocab)))
        case.update(temperature=rng.choice([1.0, 1.0, 0.7, 2.0]))
        if kind == "logprob":
            case.update(top=rng.choice([0, 1, 5, 20, 64]))
        elif kind == "logprob_train":
            case.update(top=0)
        else:
            case.update(teacher=_log_int(rng, 1, 64), hard=rng.random() < 0.5)
    batch = _log_int(rng, 1, min(16, rows))
    case.update(batch=batch, length=max(1, rows // batch))
    return case


# ----------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _ids(gen, vocab, shape):
    """Zipf-like token ids, P(v) about 1 / (v + 1), their order scattered over the vocabulary."""
    u = torch.rand(shape, generator=gen, device=DEVICE, dtype=torch.float64)
    rank = torch.floor(torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=gen, device=DEVICE)[rank]


def _tail(case):
    """Which positions lie behind their sequence's end: sequences get shorter down the batch."""
    b, l = case["batch"], case["length"]
    cut = torch.linspace(0.0, 2.0 * case["padded"], b, device=DEVICE, dtype=torch.float64)
    kept = l - torch.floor(cut * l).long().clamp_(max=l - 1)
    return torch.arange(l, device=DEVICE).unsqueeze(0) >= kept.unsqueeze(1)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, vocab, dt = case["kind"], case["vocab"], _dtype(case)
    shape = (case["batch"], case["length"])
    state = dict(case=case)
    if own:
        import __graft_entry__

        state["m3"] = __graft_entry__.load_package()
    if kind.startswith("embed"):
        d = case["width"]
        tokens = _ids(gen, vocab, shape)
        state["table"] = (0.02 * _randn(gen, vocab, d)).to(dt).requires_grad_(kind == "embed_train")
        state["pad"] = None
        if case["padded"]:
            state["pad"] = vocab - 1
            tokens = torch.where(_tail(case), torch.full_like(tokens, vocab - 1), tokens)
        state["tokens"] = tokens
        if kind == "embed_train":
            state["dy"] = (0.01 * _randn(gen, *shape, d)).to(dt)
        return state
    # logits as a model leaves them: a few likely tokens over a broad tail
    x = _randn(gen, *shape, vocab).mul_(1.5)
    likely = _ids(gen, vocab, (*shape, 8))
    x.scatter_add_(-1, likely, 4.0 + 2.0 * _randn(gen, *shape, 8))
    x = x.to(dt)
    targets = likely[..., 0].contiguous()
    if case["padded"]:
        targets = targets.masked_fill(_tail(case), IGNORE)
    state["targets"] = targets
    if kind.startswith("distill"):
        k = min(case["teacher"], vocab)
        t = x.float().mul_(0.8).add_(_randn(gen, *shape, vocab))
        top, ids = torch.topk(t, k, dim=-1)
        state["teacher_logits"] = top.to(dt)
        state["teacher_ids"] = ids.masked_fill((targets == IGNORE).unsqueeze(-1), -1)
        del t
    rows = float(shape[0] * shape[1])
    if kind == "logprob_train":
        # what the loss sends back: an advantage for each drawn token, a small entropy bonus
        state["dlogp"] = _randn(gen, *shape) / rows
        state["dentropy"] = torch.full(shape, -0.01 / rows, device=DEVICE)
    if kind == "distill_train":
        state["dkd"] = torch.full(shape, 0.7 / rows, device=DEVICE)
        state["dnll"] = torch.full(shape, 0.3 / rows, device=DEVICE)
    state["logits"] = x.requires_grad_(kind.endswith("train"))
    return state


# ----------------------------------------------------------------------------------------
# the calls, and their plain form
# ----------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    form = _own if own else _plain
    if kind.endswith("train"):
        return form(kind, state)
    with torch.no_grad():
        return form(kind, state)


def _own(kind, state):
    case, T = state["case"], state["m3"].tokens
    if kind == "embed":
        return T.embed_tokens(state["table"], state["tokens"], scale=case["scale"],
                              padding_idx=state["pad"])
    if kind == "embed_train":
        y = T.embed_tokens(state["table"], state["tokens"], scale=case["scale"],
                           padding_idx=state["pad"])
        (dtable,) = torch.autograd.grad(y, state["table"], state["dy"])
        return y.detach(), dtable
    x = state["logits"]
    if kind == "logprob":
        out = T.token_logprobs(x, state["targets"], top=min(case["top"], case["vocab"]),
                               temperature=case["temperature"])
        return (out.logp, out.entropy, out.top_logp, out.top_ids) if case["top"] else (out.logp, out.entropy)
    if kind == "logprob_train":
        out = T.token_logprobs(x, state["targets"], temperature=case["temperature"])
        (dx,) = torch.autograd.grad((out.logp, out.entropy), x, (state["dlogp"], state["dentropy"]))
        return out.logp.detach(), out.entropy.detach(), dx
    out = T.distill_loss(x, state["teacher_ids"], state["teacher_logits"],
                         temperature=case["temperature"],
                         targets=state["targets"] if case["hard"] else None)
    if kind == "distill":
        return (out.kd, out.nll) if case["hard"] else (out.kd,)
    if case["hard"]:
        (dx,) = torch.autograd.grad((out.kd, out.nll), x, (state["dkd"], state["dnll"]))
        return out.kd.detach(), out.nll.detach(), dx
    (dx,) = torch.autograd.grad(out.kd, x, state["dkd"])
    return out.kd.detach(), dx


@torch.no_grad()
def _plain(kind, state):
    case = state["case"]
    if kind.startswith("embed"):
        table, tokens = state["table"], state["tokens"]
        y = (table[tokens].float() * case["scale"]).to(table.dtype)
        if kind == "embed":
            return y
        dy = state["dy"].float().reshape(-1, case["width"]) * case["scale"]
        ids = tokens.reshape(-1)
        if state["pad"] is not None:
            dy = dy * (ids != state["pad"]).unsqueeze(-1)
        dtable = torch.zeros(table.shape, device=table.device).index_add_(0, ids, dy)
        return y, dtable.to(table.dtype)
    x, targets, inv_t = state["logits"], state["targets"], 1.0 / case["temperature"]
    live = targets != IGNORE
    at = targets.clamp(min=0).unsqueeze(-1)
    z = x.float()
    if kind.startswith("logprob"):
        d = (z - z.amax(-1, keepdim=True)) * inv_t
        e = torch.exp(d)
        s = e.sum(-1, keepdim=True)
        logs = torch.log(s)
        logp = torch.where(live, (d.gather(-1, at) - logs).squeeze(-1), 0.0)
        h = logs.squeeze(-1) - (e * d).sum(-1) / s.squeeze(-1)
        entropy = torch.where(live, h, 0.0)
        if kind == "logprob_train":
            gl = torch.where(live, state["dlogp"], 0.0).unsqueeze(-1) * inv_t
            gh = torch.where(live, state["dentropy"], 0.0).unsqueeze(-1) * inv_t
            dx = -(e / s) * (gl + gh * (d - logs + h.unsqueeze(-1)))
            dx.scatter_add_(-1, at, gl)
            return logp, entropy, dx.to(x.dtype)
        if not case["top"]:
            return logp, entropy
        k = min(case["top"], case["vocab"])
        ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :k]
        top = torch.where(live.unsqueeze(-1), d.gather(-1, ids) - logs, -math.inf)
        return logp, entropy, top, torch.where(live.unsqueeze(-1), ids, -1)
    t, ids, temp = state["teacher_logits"].float(), state["teacher_ids"], case["temperature"]
    there = ids >= 0
    some = there.any(-1)
    t = torch.where(there, t, -math.inf)
    tm = torch.where(some, t.amax(-1), 0.0).unsqueeze(-1)
    pe = torch.exp((t - tm) * inv_t)
    ps = pe.sum(-1, keepdim=True)
    p = torch.where(there, pe / ps, 0.0)
    logp = torch.where(there, (t - tm) * inv_t - torch.log(ps), 0.0)
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d * inv_t)
    s = e.sum(-1, keepdim=True)
    at_k = ids.clamp(min=0)
    logq = d.gather(-1, at_k) * inv_t - torch.log(s)
    kd = torch.where(some, temp * temp * (p * (logp - logq)).sum(-1), 0.0)
    out = (kd,)
    if case["hard"]:
        e1 = e if temp == 1.0 else torch.exp(d)
        s1 = e1.sum(-1, keepdim=True)
        out += (torch.where(live, (torch.log(s1) - d.gather(-1, at)).squeeze(-1), 0.0),)
    if kind == "distill":
        return out
    g = torch.where(some, state["dkd"], 0.0).unsqueeze(-1) * temp
    dx = e * (g / s)
    dx.scatter_add_(-1, at_k, -g * p)
    if case["hard"]:
        gn = torch.where(live, state["dnll"], 0.0).unsqueeze(-1)
        dx += e1 * (gn / s1)
        dx.scatter_add_(-1, at, -gn)
    return (*out, dx.to(x.dtype))


# ----------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------


def work(case):
    rows, vocab = case["batch"] * case["length"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"].startswith("embed"):
        d = case["width"]
        nbytes = 8 * rows + min(rows, vocab) * d * size + rows * d * size
        if case["kind"] == "embed_train":
            nbytes += rows * d * size + vocab * d * size
        return dict(bytes=nbytes, flops=(2 if case["kind"] == "embed_train" else 1) * rows * d)
    nbytes, per = rows * (vocab * size + 8 + 8), 5
    if case["kind"].startswith("logprob"):
        nbytes += rows * case["top"] * 12
    else:
        nbytes += rows * case["teacher"] * (8 + size)
        per = 7 if case["hard"] else 4
    if case["kind"].endswith("train"):
        # the gradient needs every row's sum first, so a logit is read once and written once
        nbytes += rows * (vocab * size + 8)
        per += 4
    return dict(bytes=nbytes, flops=per * rows * vocab)


# ----------------------------------------------------------------------------------------
# float64, from the definitions
# ----------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"].startswith("embed"):
            return _exact_embed(case, state)
        shape = (case["batch"], case["length"])
        rows, vocab = shape[0] * shape[1], case["vocab"]
        flat = lambda key: state[key].reshape(rows, *state[key].shape[2:]) if key in state else None  # noqa: E731
        block = max(1, (1 << 26) // vocab)
        one = _exact_logprob if case["kind"].startswith("logprob") else _exact_distill
        parts = []
        for lo in range(0, rows, block):
            sl = slice(lo, min(lo + block, rows))
            take = lambda key: None if flat(key) is None else flat(key)[sl]  # noqa: E731
            parts.append(one(case, take))
        return tuple(torch.cat(c).reshape(*shape, *c[0].shape[1:]) for c in zip(*parts))


def _exact_embed(case, state):
    table, tokens = state["table"].detach().double(), state["tokens"]
    y = table.index_select(0, tokens.reshape(-1)).mul_(case["scale"]).reshape(*tokens.shape, -1)
    if case["kind"] == "embed":
        return y
    # every id's rows stand together after a sort; its sum is a difference of running sums
    ids, order = torch.sort(tokens.reshape(-1))
    run_sum = state["dy"].double().reshape(-1, case["width"])[order].cumsum(0)
    uniq, counts = torch.unique_consecutive(ids, return_counts=True)
    upto = run_sum[counts.cumsum(0) - 1]
    sums = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1])) * case["scale"]
    if state["pad"] is not None:
        sums[uniq == state["pad"]] = 0.0
    dtable = torch.zeros_like(table)
    dtable[uniq] = sums
    return y, dtable


def _exact_logprob(case, take):
    x, targets = take("logits").double() / case["temperature"], take("targets")
    live = targets != IGNORE
    lsm = x - torch.logsumexp(x, -1, keepdim=True)
    onehot = torch.zeros_like(x).scatter_(-1, targets.clamp(min=0).unsqueeze(-1), 1.0)
    logp = (lsm * onehot).sum(-1) * live
    prob = lsm.exp()
    entropy = -(prob * lsm).sum(-1) * live
    if case["kind"] == "logprob_train":
        gl, gh = take("dlogp").double() * live, take("dentropy").double() * live
        dx = gl[:, None] * (onehot - prob) - gh[:, None] * prob * (lsm + entropy[:, None])
        return logp, entropy, dx / case["temperature"]
    if not case["top"]:
        return logp, entropy
    k = min(case["top"], case["vocab"])
    vals, ids = torch.sort(take("logits").double(), dim=-1, descending=True, stable=True)
    ids = ids[:, :k]
    top = torch.gather(lsm, 1, ids)
    top[~live] = -math.inf
    return logp, entropy, top, ids.masked_fill(~live[:, None], -1)


def _exact_distill(case, take):
    temp = case["temperature"]
    x, ids = take("logits").double(), take("teacher_ids")
    some = (ids >= 0).any(-1)
    t = (take("teacher_logits").double() / temp).masked_fill(ids < 0, -math.inf)
    t[~some] = 0.0
    p = torch.softmax(t, -1) * some[:, None]
    lsm = x / temp - torch.logsumexp(x / temp, -1, keepdim=True)
    logq = torch.gather(lsm, 1, ids.clamp(min=0))
    kd = temp ** 2 * (torch.special.xlogy(p, p) - p * logq).sum(-1)
    out = (kd,)
    live = take("targets") != IGNORE
    at = take("targets").clamp(min=0)[:, None]
    if case["hard"]:
        ls1 = x - torch.logsumexp(x, -1, keepdim=True)
        out += (-torch.gather(ls1, 1, at)[:, 0] * live,)
    if case["kind"] == "distill":
        return out
    soft = torch.zeros_like(x).scatter_add_(-1, ids.clamp(min=0), p)
    dx = temp * (take("dkd").double() * some)[:, None] * (lsm.exp() - soft)
    if case["hard"]:
        gn = (take("dnll").double() * live)[:, None]
        dx += gn * ls1.exp()
        dx.scatter_add_(-1, at, -gn)
    return (*out, dx)
