"""GPU parity of the operators that read the logits (`m3s_logprob_*`, `m3s_distill_*`) against their
formulas in float64 on the CPU, from the same (float32 or bf16) logits.

Tolerances, from the arithmetic (eps = 2^-24, half a float32 step). Let a row have d = max x - x and
D = min(max d / T, 104), past which a term is zero in float32:
  * a term e^{-d/T} is off by 2 eps (d / T) of its value from its argument (the difference's
    rounding, and the product with 1 / (T ln 2), itself rounded: 3 roundings of an argument
    d / (T ln 2), times ln 2) and 2 eps from exp2, so by at most E = (3 D + 2) eps of it;
  * a sum of V of them, in 256 or more running sums of at most V / 256 + 16 additions and joins,
    by E + (V / 256 + 40) eps of its value, and so log s by that much absolutely, plus eps |log s|;
  * logp and entropy add a few roundings of numbers up to D + log V: 8 (D + log V) eps. The entropy
    also holds sum e d / s, off by the sums' relative error times at most D;
  * p = e^{-d/T} / s: relative E + the sum's; a gradient is at most (|g| + |g_H| (D + log V)) p so
    its error is that relative error, applied to p times the magnitudes, plus the same number of
    roundings; the entropy's own error enters as |g_H| p times it; then half a step of the type.
    exp2 flushes results under 2^-126 to zero, so p is also off by up to that absolutely, times the
    same magnitudes (a row of spread 200 has p of 1e-38 next to |g_H| log p of 100).
Everything is doubled once for the second order and for the float32 1 / T.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
FLUSH = 2.0 ** -126
INF = float("inf")


def type_step(dtype):
    return EPS if dtype == torch.float32 else 2.0 ** -8


def bounds(x, temp):
    """(relative error of p and of the sum, absolute error of logp, of the entropy), per row."""
    v = x.shape[-1]
    fin = x.masked_fill(~x.isfinite(), 0.0)
    dmax = ((x.masked_fill(~x.isfinite(), -INF).amax(-1) - fin.amin(-1)) / min(temp, 1.0)).clamp(0, 104)
    e = (3 * dmax + 2) * EPS
    rel = 2 * (2 * e + (v / 256 + 40) * EPS)
    size = dmax + math.log(v) + 1
    return rel, rel + 16 * size * EPS, rel * (1 + dmax) + 16 * size * EPS


def log_softmax_ref(x, temp):
    """Relative to the row's maximum: a row of the type's lowest value would lose log V in x - lse."""
    m = x.amax(-1, keepdim=True)
    empty = m == -INF
    z = (x - torch.where(empty, 0.0, m)) / temp
    return torch.where(empty, -INF, z - torch.log(torch.where(empty, 1.0, z.exp().sum(-1, keepdim=True))))


def logprob_ref(x, targets, top, temp, ignore=-100):
    """Formulas in float64 for rows (R, V): logp, entropy, top_logp, top_ids, p, log p."""
    r, v = x.shape
    x = x.double()
    nan = (x.isnan() | (x == INF)).any(-1)
    lp = log_softmax_ref(x, temp)
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    top_lp = lp.gather(-1, ids)
    logp = None
    if targets is not None:
        ok = (targets >= 0) & (targets < v)
        logp = torch.where(ok, lp.gather(-1, targets.clamp(0, v - 1)[:, None])[:, 0], math.nan)
        logp[nan] = math.nan
    h[nan] = math.nan
    top_lp[nan], ids[nan] = math.nan, -1
    if targets is not None:
        skip = targets == ignore
        logp[skip], h[skip], top_lp[skip], ids[skip] = 0.0, 0.0, -INF, -1
    return logp, h, top_lp, ids, p, lp


def same(got, want, tol, what):
    """Equal where not finite, within ``tol`` elsewhere."""
    got, want = got.detach().cpu().double(), want.double()
    fin = want.isfinite()
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()], want[want.isinf()]), what
    over = torch.where(fin, (got - want).abs() / tol.expand_as(want), 0.0).flatten()
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 1.0, (what, worst, int(over.argmax()), got.flatten()[over.argmax()].item(),
                          want.flatten()[over.argmax()].item())


def make_logits(shape, dtype, gen, kind="model"):
    x = 1.5 * torch.randn(shape, generator=gen)
    if kind == "model":
        hot = torch.randint(0, shape[-1], (*shape[:-1], min(8, shape[-1])), generator=gen)
        x.scatter_add_(-1, hot, 4 + 2 * torch.randn(hot.shape, generator=gen))
    elif kind == "wide":
        x *= 40
    elif kind == "masked":   # few allowed tokens
        x.masked_fill_(torch.rand(shape, generator=gen) > 8.0 / shape[-1], -INF)
    elif kind == "flat":
        x = torch.zeros(shape)
    elif kind == "ties":
        x = (x * 2).round()
    elif kind == "far":      # one row far from zero: x - max must not lose the small differences
        x += 3.0e4
    return x.to(dtype)


def check_logprob(m3, dev, x, targets, top, temp, grads, seed=0):
    """Forward and every gradient of `token_logprobs` for rows (R, V)."""
    r, v = x.shape
    gen = torch.Generator().manual_seed(seed)
    xd = x.to(dev).requires_grad_(True)
    out = m3.token_logprobs(xd, None if targets is None else targets.to(dev), top=top, temperature=temp)
    logp, h, top_lp, ids, p, lp = logprob_ref(x, targets, top, temp)
    rel, tol_lp, tol_h = bounds(x.double(), temp)
    same(out.entropy, h, tol_h, "entropy")
    if targets is not None:
        same(out.logp, logp, tol_lp, "logp")
    if top:
        assert torch.equal(out.top_ids.cpu(), ids)
        same(out.top_logp, top_lp, tol_lp[:, None], "top_logp")
    bare = m3.token_logprobs(xd.detach(), None if targets is None else targets.to(dev), top=top, temperature=temp)
    for a, b in zip(out, bare):
        assert (a is None) == (b is None) and (a is None or torch.equal(a.isnan(), b.isnan())
                                               and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)))
    for which in grads:
        gl = torch.randn(r, generator=gen) if "l" in which and targets is not None else None
        gh = torch.randn(r, generator=gen) if "h" in which else None
        gt = torch.randn(r, top, generator=gen) if "t" in which and top else None
        pairs = [(o, g.to(dev)) for o, g in ((out.logp, gl), (out.entropy, gh), (out.top_logp, gt)) if g is not None]
        if not pairs:
            continue
        (dx,) = torch.autograd.grad([a for a, _ in pairs], xd, [b for _, b in pairs], retain_graph=True)
        assert dx.dtype == x.dtype and dx.shape == x.shape
        dead = (x == -INF).all(-1) | (targets == -100 if targets is not None else torch.zeros(r, dtype=torch.bool))
        zero = torch.zeros(r, dtype=torch.float64)
        g1, g2 = zero if gl is None else gl.double(), zero if gh is None else gh.double()
        g3 = torch.zeros(r, 0, dtype=torch.float64) if gt is None else gt.double()
        total = g1 + g3.sum(-1)
        lpz = torch.where(p > 0, lp, 0.0)
        hz = h.nan_to_num(0.0)[:, None]
        want = -p * (total[:, None] + g2[:, None] * (lpz + hz))
        coef = (g1.abs() + g3.abs().sum(-1) + g2.abs() * (lpz.abs().amax(-1) + hz[:, 0]))[:, None]
        mag = p * coef
        if gl is not None:
            want.scatter_add_(-1, targets.clamp(0, v - 1)[:, None], g1[:, None])
            want[(targets < 0) | (targets >= v)] = math.nan
            mag.scatter_add_(-1, targets.clamp(0, v - 1)[:, None], g1.abs()[:, None])
        if gt is not None:
            safe = ids.clamp(min=0)
            want.scatter_add_(-1, safe, g3)
            mag.scatter_add_(-1, safe, g3.abs())
        want[(x.isnan() | (x == INF)).any(-1)] = math.nan
        want[dead] = 0.0
        want, mag = want / temp, mag / temp
        tol = (rel[:, None] + (top + 8) * EPS) * mag + (g2.abs() * tol_h)[:, None] * 2 * p / temp
        tol = tol + want.abs() * 2 * type_step(x.dtype) + FLUSH * (coef / temp + 1)
        same(dx, want, tol.nan_to_num(1.0), f"dlogits of {which}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top,temp", [
    (5, 1, 1, 1.0), (3, 2, 2, 0.5), (7, 17, 5, 1.0), (9, 64, 64, 2.0), (33, 255, 3, 1.0), (6, 256, 20, 0.7),
    (5, 257, 64, 1.0), (4, 1000, 1, 1.3), (3, 4099, 20, 1.0), (2, 16384, 64, 1.0), (2, 50001, 20, 0.8),
    (1, 131072, 64, 1.0), (300, 311, 0, 1.0)])
def test_logprobs_and_gradients(m3, dev, dtype, rows, vocab, top, temp):
    gen = torch.Generator().manual_seed(rows * 1000 + vocab)
    x = make_logits((rows, vocab), dtype, gen)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    check_logprob(m3, dev, x, targets, top, temp, ("l", "h", "lht"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["wide", "masked", "flat", "ties", "far"])
@pytest.mark.parametrize("vocab", [40, 700, 9001, 40007])
def test_logprobs_of_hard_rows(m3, dev, dtype, kind, vocab):
    """Wide rows, rows with almost every token masked to -inf, rows of ties, and rows far from zero;
    with ignored positions, ids outside the vocabulary, empty rows, NaN and infinities among them."""
    gen = torch.Generator().manual_seed(vocab)
    rows = 12
    x = make_logits((rows, vocab), dtype, gen, kind)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    targets[1], targets[2], targets[3] = -100, -1, vocab
    x[4] = -INF
    x[5, vocab // 2] = math.nan
    x[6, 0] = INF
    x[7], targets[7] = math.nan, -100          # garbage behind a sequence's end
    x[8, : vocab - 1] = torch.finfo(dtype).min   # masks of the type's lowest value
    x[9, 3:] = -INF
    for top in (0, 5, 33):
        check_logprob(m3, dev, x, targets, top, 1.0, ("l", "lht"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(600, 9001), (130, 20003), (2100, 700), (10, 260), (4200, 250), (4500, 1001),
                                        (1100, 2049)])
def test_whole_rows_of_hard_kinds(m3, dev, dtype, rows, vocab):
    """Enough rows that none is cut: masks, ties, flat rows, empty ones and ordinary ones together,
    and rows whose best logits all lie at the places of few threads."""
    gen = torch.Generator().manual_seed(rows)
    kinds = ("model", "masked", "flat", "ties", "wide")
    x = torch.cat([make_logits((rows // 5, vocab), dtype, gen, k) for k in kinds])
    x[3], x[5] = -INF, torch.finfo(dtype).min
    place = torch.arange(vocab) // (4 if dtype == torch.float32 else 8) % 256
    x[7] = (10 * (place < 40) + torch.rand(vocab, generator=gen)).to(dtype)
    x[8] = torch.where(place == 3, 5.0, -INF)
    targets = torch.randint(0, vocab, (len(x),), generator=gen)
    targets[::11] = -100
    for top in (0, 1, 2, 3, 5, 14, 15, 20, 64):
        check_logprob(m3, dev, x, targets, top, 1.0, ("lht",) if top in (0, 20) else ())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [24, 31, 64, 130, 251, 256])
def test_many_short_rows(m3, dev, dtype, vocab):
    """As many rows as make 16 lanes pick the alternatives of each, around the numbers at which they
    do it another way: ordinary rows, masks, ties and flat rows, and rows that rise or fall throughout."""
    gen = torch.Generator().manual_seed(vocab)
    kinds = ("model", "masked", "flat", "ties", "wide")
    x = torch.cat([make_logits((830, vocab), dtype, gen, k) for k in kinds])
    x[3], x[5] = -INF, torch.finfo(dtype).min
    x[7], x[8] = torch.arange(vocab).to(dtype), -torch.arange(vocab).to(dtype)
    x[9, : vocab - 3], x[10, 5:] = -INF, -INF
    x[11, ::16], x[12, 1::2] = 9.0, 9.0
    targets = torch.randint(0, vocab, (len(x),), generator=gen)
    targets[::11] = -100
    for top in (1, 2, 7, 8, 9, 16, 17, 23, 24):
        check_logprob(m3, dev, x, targets, top, 1.0, ())
    if vocab > 24:
        check_logprob(m3, dev, x, targets, 25, 1.0, ("lht",))


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1000), (torch.float32, 1024), (torch.bfloat16, 1023),
                                         (torch.float32, 250), (torch.bfloat16, 500)])
def test_few_lanes_hold_more_than_the_list(m3, dev, dtype, vocab):
    """Rows of a wave whose lanes hold falling blocks of logits: the lanes that reach a bound on their
    maxima reach it with all they hold."""
    gen = torch.Generator().manual_seed(vocab)
    lane = torch.arange(vocab) // (4 if dtype == torch.float32 else 8) % 64
    rows = [(100 - slope * lane + 0.1 * torch.rand(vocab, generator=gen)) for slope in (0.25, 0.5, 0.9, 1.5)]
    rows += [100 - 0.9 * lane, 50.0 + 0 * lane, torch.where(lane < 40, 7.0, -INF)]
    x = torch.stack([r.float() for r in rows]).to(dtype)
    targets = torch.arange(len(rows))
    for top in (1, 5, 20, 24, 25, 30, 31, 64):
        check_logprob(m3, dev, x, targets, top, 1.0, ())


def test_one_thread_holds_the_best(m3, dev):
    """The best tokens all at one stride, equal or falling, so that one part of the workgroup has
    them all."""
    for stride in (1024, 1000, 4096, 16):
        x = torch.full((2, 140000), -5.0)
        at = torch.arange(0, 140000, stride)
        x[0, at] = 9.0
        x[1, at] = 9.0 - 0.01 * torch.arange(len(at))
        check_logprob(m3, dev, x, torch.tensor([5, 0]), 64, 1.0, ("lht",))


def test_shapes_strides_and_types(m3, dev):
    """No leading axis, several, a shifted view of (B, L, V), an expanded row, strided last axis, and
    int32 targets; results of the dense copy."""
    gen = torch.Generator().manual_seed(2)
    full = make_logits((3, 7, 301), torch.float32, gen).to(dev)
    targets = torch.randint(0, 301, (3, 7), generator=gen).to(dev)
    T = m3.token_logprobs
    cases = [(full[:, :-1], targets[:, 1:]), (full[0, 0], targets[0, 0]), (full[1], targets[1].int()),
             (full.view(3, 1, 7, 301), targets.view(3, 1, 7)), (full[:, ::2], targets[:, ::2]),
             (full[:1].expand(4, 7, 301), targets[:1].expand(4, 7)), (full.transpose(1, 2), targets.new_zeros(3, 301)),
             (full[..., 5:205], targets % 200), (full.transpose(0, 1), targets.t())]
    for x, t in cases:
        xg = x.detach().requires_grad_(True)
        out = T(xg, t, top=3)
        ref = T(x.contiguous(), t.contiguous(), top=3)
        assert out.logp.shape == t.shape and out.top_ids.shape == (*t.shape, 3)
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
        (dx,) = torch.autograd.grad(out.logp.sum() + out.top_logp.sum(), xg)
        xc = x.detach().contiguous().requires_grad_(True)
        ref = T(xc, t, top=3)
        (dc,) = torch.autograd.grad(ref.logp.sum() + ref.top_logp.sum(), xc)
        assert torch.equal(dx, dc)
    for shape in ((0, 7, 301), (3, 0, 301), (0, 301), (2, 3, 0, 301), (0, 2, 3, 301)):
        x = full.new_zeros(shape).requires_grad_(True)
        t = targets.new_zeros(shape[:-1])
        e = T(x, t, top=2)
        assert e.logp.shape == shape[:-1] and e.top_ids.shape == (*shape[:-1], 2)
        d = m3.distill_loss(x, e.top_ids, e.top_logp.detach(), targets=t)
        (dx,) = torch.autograd.grad(e.logp.sum() + d.kd.sum() + d.nll.sum(), x)
        assert dx.shape == shape
    only = T(full, top=4)
    assert only.logp is None and torch.equal(only.top_ids, T(full, targets, top=4).top_ids)
    out = T(full.requires_grad_(True), targets)
    out.logp.mul_(2.0)   # a result may be changed in place
    (2 * out.logp).sum().backward()
    assert full.grad.isfinite().all()


def distill_ref(x, ids, teacher, targets, temp, ignore=-100):
    """Formulas in float64 for rows (R, V): kd, nll, and what the gradient is made of."""
    r, v = x.shape
    x, u = x.double(), teacher.double()
    u = torch.where(ids >= 0, u, -INF)
    bad = (ids >= v).any(-1) | ((ids >= 0) & (u.isnan() | (u == INF))).any(-1)
    some = (u > -INF).any(-1) | bad
    um = torch.where(some, u.nan_to_num(0.0, 0.0).masked_fill(u == -INF, -INF).amax(-1), 0.0)[:, None]
    um = um.masked_fill(um == -INF, 0.0)
    w = torch.exp((u - um) / temp)
    w = torch.where(u == -INF, 0.0, w)
    w = w / torch.where(some, w.sum(-1), 1.0)[:, None]
    empty = (x == -INF).all(-1)
    nan = (x.isnan() | (x == INF)).any(-1)
    lq, l1 = log_softmax_ref(x, temp), log_softmax_ref(x, 1.0)
    at = ids.clamp(0, v - 1)
    terms = torch.where(w > 0, w * (w.log() - lq.gather(-1, at)), 0.0)
    kd = temp ** 2 * terms.sum(-1)
    kd[nan | bad] = math.nan
    kd[~some] = 0.0
    nll = None
    if targets is not None:
        hard = targets != ignore
        nll = -l1.gather(-1, targets.clamp(0, v - 1)[:, None])[:, 0]
        nll[nan | (targets < 0) | (targets >= v)] = math.nan
        nll[~hard] = 0.0
    soft = torch.zeros_like(x).scatter_add_(-1, at, w.nan_to_num(0.0))
    return kd, nll, w, soft, lq.exp(), l1.exp(), some, bad, empty, nan


def check_distill(m3, dev, x, ids, teacher, targets, temp, seed=0):
    r, v = x.shape
    k = ids.shape[1]
    gen = torch.Generator().manual_seed(seed)
    xd = x.to(dev).requires_grad_(True)
    tgt = None if targets is None else targets.to(dev)
    out = m3.distill_loss(xd, ids.to(dev), teacher.to(dev), temperature=temp, targets=tgt)
    kd, nll, w, soft, q, q1, some, bad, empty, nan = distill_ref(x, ids, teacher, targets, temp)
    rel, tol_lp, _ = bounds(x.double(), temp)
    # the teacher's weights: K terms, arguments up to the spread of its logits
    u = teacher.double().masked_fill(ids < 0, -INF)
    fin = torch.where(u.isfinite(), u, 0.0)
    spread = ((torch.where(u.isfinite(), u, -INF).amax(-1) - fin.amin(-1)).clamp(min=0).nan_to_num(0.0, 0.0) / temp).clamp(0, 104)
    tol_w = 2 * (2 * (3 * spread + 2) + k + 8) * EPS
    size = (x.double().nan_to_num(0.0, 0.0, 0.0).abs().amax(-1) / temp + spread + 20 + math.log(v))
    tol_kd = temp ** 2 * (2 * (tol_w + tol_lp) + (tol_w + (k + 16) * EPS) * 2 * size) + 1e-37
    same(out.kd, kd, tol_kd, "kd")
    if targets is not None:
        same(out.nll, nll, bounds(x.double(), 1.0)[1], "nll")
    with torch.no_grad():
        bare = m3.distill_loss(xd, ids.to(dev), teacher.to(dev), temperature=temp, targets=tgt)
        assert torch.equal(bare.kd.nan_to_num(7.0), out.kd.nan_to_num(7.0))
    zero = torch.zeros(r, dtype=torch.float64)
    for which in ("k", "n", "kn"):
        gk = torch.randn(r, generator=gen) if "k" in which else None
        gn = torch.randn(r, generator=gen) if "n" in which and targets is not None else None
        pairs = [(o, g.to(dev)) for o, g in ((out.kd, gk), (out.nll, gn)) if g is not None]
        if not pairs:
            continue
        (dx,) = torch.autograd.grad([a for a, _ in pairs], xd, [b for _, b in pairs], retain_graph=True)
        hard = targets != -100 if targets is not None else torch.zeros(r, dtype=torch.bool)
        a = torch.where(some, gk.double() * temp, 0.0) if gk is not None else zero
        b = torch.where(hard, gn.double(), 0.0) if gn is not None else zero
        onehot = torch.zeros(r, v, dtype=torch.float64)
        if targets is not None:
            onehot.scatter_(-1, targets.clamp(0, v - 1)[:, None], 1.0)
        want = a[:, None] * (q - soft) + b[:, None] * (q1 - onehot)
        mag = a.abs()[:, None] * (q + soft) + b.abs()[:, None] * (q1 + onehot)
        rel1 = bounds(x.double(), 1.0)[0]
        tol = (torch.maximum(rel, rel1)[:, None] + tol_w[:, None] + (k + 8) * EPS) * mag
        tol = tol + want.abs() * 2 * type_step(x.dtype) + FLUSH * (2 * a.abs() + 2 * b.abs() + 1)[:, None]
        live = torch.zeros(r, dtype=torch.bool)
        if gk is not None:
            live |= some
            want[bad] = math.nan
        if gn is not None:
            live |= hard
            want[hard & ((targets < 0) | (targets >= v))] = math.nan
        want[nan] = math.nan
        want[~live | empty] = 0.0
        same(dx, want, tol.nan_to_num(1.0), f"dlogits of {which}")


def teacher_of(x, k, gen, dtype):
    noisy = x.float().nan_to_num(0.0, 0.0, -30.0) * 0.8 + torch.randn(x.shape, generator=gen)
    top, ids = torch.topk(noisy, k, dim=-1)
    return ids, top.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k,temp,tdt,idt", [
    (3, 1, 1, 1.0, torch.float32, torch.int64), (5, 9, 3, 2.0, torch.float32, torch.int32),
    (40, 256, 16, 2.0, torch.float32, torch.int64), (7, 257, 64, 1.0, torch.bfloat16, torch.int64),
    (4, 1000, 100, 0.5, torch.float32, torch.int32), (3, 5003, 256, 4.0, torch.float32, torch.int64),
    (2, 50001, 32, 2.0, torch.bfloat16, torch.int32), (300, 130, 7, 1.0, torch.float32, torch.int64),
    (4500, 131, 16, 2.0, torch.float32, torch.int64), (4100, 999, 64, 1.0, torch.bfloat16, torch.int32),
    (4100, 300, 65, 2.0, torch.float32, torch.int64), (1200, 2050, 9, 3.0, torch.float32, torch.int64)])
def test_distillation_and_gradients(m3, dev, dtype, rows, vocab, k, temp, tdt, idt):
    gen = torch.Generator().manual_seed(rows * 31 + vocab)
    x = make_logits((rows, vocab), dtype, gen)
    ids, teacher = teacher_of(x, k, gen, tdt)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    check_distill(m3, dev, x, ids.to(idt), teacher, targets, temp)
    check_distill(m3, dev, x, ids.to(idt), teacher, None, temp)


@pytest.mark.parametrize("vocab,repeat", [(50, 1), (3001, 1), (20011, 1), (61, 300), (1003, 260), (2055, 70)])
def test_distillation_of_hard_rows(m3, dev, vocab, repeat):
    """Rows without entries, entries of weight zero, ids named twice, ids and targets outside the
    vocabulary, ignored targets, empty student rows, NaN and infinities on either side, and garbage
    logits where there is nothing to learn."""
    gen = torch.Generator().manual_seed(vocab)
    rows, k = 16, 12
    x = make_logits((rows, vocab), torch.float32, gen)
    ids, teacher = teacher_of(x, k, gen, torch.float32)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    ids[0] = -1                                   # no entry, hard target alone
    ids[1], targets[1] = -1, -100                 # nothing
    x[1] = math.nan
    ids[2, ::2] = -1                              # half of the entries
    teacher[3, 2:] = -INF
    teacher[4] = -INF                             # entries of no weight at all
    ids[5] = ids[5, 0]                            # one token, twelve times
    ids[6, 1], targets[6] = ids[6, 0], ids[6, 0]  # twice, and the target
    ids[7, 3] = vocab
    targets[8] = -100
    targets[9] = vocab + 5
    x[10] = -INF
    x[11, vocab // 3] = math.nan
    teacher[12, 1] = math.nan
    teacher[13, 1] = INF
    x[14, ids[14, 0]] = -INF                      # the student rules the teacher's best out
    x[15, 0] = INF
    # as often as it takes for the calls of many rows
    x, ids, teacher, targets = (t.repeat(repeat, *[1] * (t.dim() - 1)) for t in (x, ids, teacher, targets))
    for temp in (1.0, 3.0):
        check_distill(m3, dev, x, ids, teacher, targets, temp)
        check_distill(m3, dev, x, ids, teacher, None, temp)


def test_offsets_past_31_bits(m3, dev):
    """The last rows of logits with more than 2^31 entries equal the same rows on their own."""
    gen = torch.Generator().manual_seed(3)
    rows, v = 68000, 32000
    x = torch.zeros(rows, v, device=dev, dtype=torch.bfloat16)
    last = make_logits((8, v), torch.bfloat16, gen).to(dev)
    x[-8:] = last
    t = torch.randint(0, v, (rows,), generator=gen).to(dev)
    t[:-8] = -100
    ids = torch.randint(0, v, (rows, 4), generator=gen).to(dev)
    ids[:-8] = -1
    u = torch.randn(rows, 4, generator=gen).to(dev)
    g = torch.randn(rows, generator=gen).to(dev)
    K = m3.kernels
    for part, whole in zip(K.logprob_forward(last, t[-8:], top=5), K.logprob_forward(x, t, top=5)):
        # whole rows and cut ones sum in another order
        assert (part.double() - whole[-8:].double()).abs().max().item() <= 1e-4 * part.double().abs().max().item()
    stats = K.logprob_forward(x, t)[4]
    dx = K.logprob_backward(x, t, stats, dlogp=g, dentropy=g)
    assert torch.equal(dx[-8:], K.logprob_backward(last, t[-8:], stats[-8:], dlogp=g[-8:], dentropy=g[-8:]))
    assert not dx[:64].any()
    kd, nll, stats = K.distill_forward(x, ids, u, t, 2.0)
    assert kd[-8:].isfinite().all() and (kd[-8:] != 0).all() and not kd[:-8].any()
    dx = K.distill_backward(x, ids, u, t, stats, g, g, 2.0)
    assert torch.equal(dx[-8:], K.distill_backward(last, ids[-8:], u[-8:], t[-8:], stats[-8:], g[-8:], g[-8:], 2.0))


def test_more_rows_than_one_grid_axis(m3, dev):
    """Rows past the workgroups of a grid's first axis (2^27 rows by 16 lanes): the last ones as if
    they were alone."""
    K, rows, last = m3.kernels, (1 << 27) + 37, 8192
    x = torch.randn(rows, 2, device=dev, dtype=torch.bfloat16)
    t = torch.randint(0, 2, (rows,), device=dev)
    ids = torch.randint(0, 2, (rows, 1), device=dev, dtype=torch.int32)
    u = torch.randn(rows, 1, device=dev)
    for part in (slice(rows - last, None), slice(0, last), slice((1 << 27) - last, 1 << 27)):
        got = [a[part] for a in K.logprob_forward(x, t, top=1)]
        want = K.logprob_forward(x[part], t[part], top=1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    kd, nll, kstats = K.distill_forward(x, ids, u, t, 2.0)
    stats = K.logprob_forward(x, t)[4]
    ones = torch.ones(rows, device=dev)
    dx = K.logprob_backward(x, t, stats, None, ones, ones)
    dk = K.distill_backward(x, ids, u, t, kstats, ones, ones, 2.0)
    for part in (slice(rows - last, None), slice(0, last)):
        one = ones[part]
        want = K.distill_forward(x[part], ids[part], u[part], t[part], 2.0)
        assert torch.equal(kd[part], want[0]) and torch.equal(nll[part], want[1])
        assert torch.equal(dk[part], K.distill_backward(x[part], ids[part], u[part], t[part], want[2], one, one, 2.0))
        assert torch.equal(dx[part], K.logprob_backward(x[part], t[part], stats[part], None, one, one))


def test_gradients_match_differences(m3, dev):
    """Central differences of float64-accumulated sums of the kernels' own outputs: a step h leaves
    h^2 of the third derivative and 2^-24 |f| / h of rounding."""
    gen = torch.Generator().manual_seed(12)
    x = make_logits((4, 300), torch.float32, gen).to(dev)
    t = torch.randint(0, 300, (4,), generator=gen).to(dev)
    ids, teacher = (a.to(dev) for a in teacher_of(x.cpu(), 8, gen, torch.float32))

    def f(z):
        lp = m3.token_logprobs(z, t, top=4, temperature=1.5)
        kd = m3.distill_loss(z, ids, teacher, temperature=2.0, targets=t)
        return lp.logp.sum() + 0.5 * lp.entropy.sum() + lp.top_logp.sum() + kd.kd.sum() + kd.nll.sum()

    xg = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(f(xg), xg)
    step = torch.randn(x.shape, generator=gen).to(dev)
    with torch.no_grad():
        slope = (f(x + 1e-2 * step).double() - f(x - 1e-2 * step).double()) / 2e-2
    want = (dx.double() * step.double()).sum()
    assert abs(slope.item() - want.item()) <= 2e-3 * (dx.double() * step.double()).abs().sum().item()


def test_chain_from_the_teacher_to_the_embedding(m3, dev):
    """Together, as they are used: a teacher's scores leave its best tokens, the student learns from
    them and from the text, and the gradient ends in its embedding. Padded positions take no part,
    whatever their logits hold."""
    gen = torch.Generator().manual_seed(5)
    b, l, v, d, k = 3, 20, 97, 24, 6
    tokens = torch.randint(0, v, (b, l + 1), generator=gen)
    tokens[1, 12:], tokens[2, 5:] = v - 1, v - 1
    targets = torch.where(tokens[:, 1:] == v - 1, -100, tokens[:, 1:])
    teacher_logits = make_logits((b, l, v), torch.float32, gen)
    teacher_logits[targets == -100] = math.nan
    table0, head = 0.3 * torch.randn(v, d, generator=gen), torch.randn(d, v, generator=gen) / 4
    t = m3.token_logprobs(teacher_logits.to(dev), targets.to(dev), top=k)
    assert (t.top_ids[(targets == -100).to(dev)] == -1).all()
    table = table0.to(dev).requires_grad_(True)
    x = m3.embed_tokens(table, tokens[:, :-1].to(dev), scale=4.0, padding_idx=v - 1) @ head.to(dev)
    out = m3.distill_loss(x, t.top_ids, t.top_logp, temperature=2.0, targets=targets.to(dev))
    n = (targets != -100).sum().item()
    loss = (0.7 * out.kd.sum() + 0.3 * out.nll.sum()) / n
    loss.backward()

    w = table0.double().requires_grad_(True)
    z = (4.0 * w[tokens[:, :-1]]) @ head.double()
    live = targets != -100
    top, ids = torch.topk(teacher_logits.double().nan_to_num(0.0), k, dim=-1)
    p = torch.softmax(top / 2.0, -1)
    kd = 4.0 * (p * (p.log() - torch.log_softmax(z / 2.0, -1).gather(-1, ids))).sum(-1)
    nll = -torch.log_softmax(z, -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    ref = (0.7 * kd[live].sum() + 0.3 * nll[live].sum()) / n
    (gw,) = torch.autograd.grad(ref, w)
    gw[v - 1] = 0.0
    assert abs(loss.item() - ref.item()) <= 1e-5 * abs(ref.item())
    assert ((table.grad.cpu().double() - gw).abs().max() / gw.abs().max()).item() <= 1e-5


def test_captured_calls_replay_on_new_inputs(m3, dev):
    """Forward and backward launches inside a recorded graph, replayed on changed logits with eager
    work between the replays."""
    gen = torch.Generator().manual_seed(7)
    K = m3.kernels
    for rows, v in ((1, 70000), (64, 256)):
        x = torch.zeros(rows, v, device=dev)
        t = torch.zeros(rows, dtype=torch.int64, device=dev)
        ids = torch.zeros(rows, 8, dtype=torch.int64, device=dev)
        u = torch.zeros(rows, 8, device=dev)
        g = torch.randn(rows, generator=gen).to(dev)

        def step():
            lp = K.logprob_forward(x, t, top=8)
            dx = K.logprob_backward(x, t, lp[4], lp[3], g, g)
            kd = K.distill_forward(x, ids, u, t, 2.0)
            return (*lp[:4], dx, *kd[:2], K.distill_backward(x, ids, u, t, kd[2], g, g, 2.0))

        side = torch.cuda.Stream(dev)
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            x.copy_(make_logits((rows, v), torch.float32, gen))
            t.copy_(torch.randint(0, v, (rows,), generator=gen))
            ids.copy_(torch.randint(0, v, (rows, 8), generator=gen))
            u.copy_(torch.randn(rows, 8, generator=gen))
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))
            torch.cuda.synchronize()


def test_runs_are_bit_reproducible(m3, dev):
    gen = torch.Generator().manual_seed(1)
    for shape in ((700, 256), (30, 50001), (2, 131072)):
        x = make_logits(shape, torch.bfloat16, gen, "ties").to(dev)
        t = torch.randint(0, shape[1], shape[:1], generator=gen).to(dev)
        a, b = (m3.token_logprobs(x, t, top=20) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_backward_of_saved_tensors_elsewhere_and_twice(m3, dev):
    """Saved operands that come back at other addresses (kept in host memory meanwhile), operands
    that the forward read as copies, a graph kept for a second backward, and broadcast cotangents:
    the same gradients as the bare calls."""
    gen = torch.Generator().manual_seed(21)
    x = make_logits((6, 300), torch.float32, gen).to(dev)
    t = torch.randint(0, 300, (6,), generator=gen).to(dev)
    ids, u = (a.to(dev) for a in teacher_of(x.cpu(), 8, gen, torch.float32))
    table = torch.randn(40, 16, generator=gen).to(dev)
    tokens = torch.randint(0, 40, (30, 6), generator=gen).to(dev)
    K = m3.kernels
    one = torch.ones(6, device=dev)
    stats, kstats = K.logprob_forward(x, t, top=4), K.distill_forward(x, ids, u, t, 2.0)[2]
    want = (K.logprob_backward(x, t, stats[4], stats[3], one, one, torch.ones(6, 4, device=dev)),
            K.distill_backward(x, ids, u, t, kstats, one, one, 2.0),
            K.embedding_backward(tokens, torch.ones(30, 6, 16, device=dev), 40, 3.0))

    def sums(x, w, ids=ids, u=u, t=t, tokens=tokens):
        lp = m3.token_logprobs(x, t, top=4)
        kd = m3.distill_loss(x, ids, u, temperature=2.0, targets=t)
        return (lp.logp.sum() + lp.entropy.sum() + lp.top_logp.sum(), kd.kd.sum() + kd.nll.sum(),
                m3.embed_tokens(w, tokens, scale=3.0).sum())

    def check(outs, xg, wg, **kw):
        grads = [torch.autograd.grad(o, v, **kw)[0] for o, v in zip(outs, (xg, xg, wg))]
        assert all(torch.equal(a, b) for a, b in zip(grads, want))

    xg, wg = x.clone().requires_grad_(True), table.clone().requires_grad_(True)
    outs = sums(xg, wg)
    check(outs, xg, wg, retain_graph=True)
    check(outs, xg, wg)
    with torch.autograd.graph.save_on_cpu():
        outs = sums(xg, wg)
    check(outs, xg, wg)
    # read as copies: another axis order, int32 targets, strided teacher and tokens
    xt = x.t().contiguous().requires_grad_(True)
    outs = sums(xt.t(), wg, ids.t().contiguous().t(), u.t().contiguous().t(), t.int(), tokens.t().contiguous().t())
    for o, v, w in zip(outs, (xt, xt, wg), want):
        g = torch.autograd.grad(o, v, retain_graph=True)[0]
        assert torch.equal(g.t() if v is xt else g, w)
    outs = sums(xg, wg)
    with torch.no_grad():
        xg.mul_(1.0)   # autograd sees that the saved logits changed
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(outs[0], xg)


def test_backward_of_saved_logits_with_other_strides(m3, dev):
    """A view's logits that come back from a hook as a compact copy, at the address that the view had:
    the same gradients as without the hook."""
    gen = torch.Generator().manual_seed(23)
    leaf = make_logits((2, 6, 300), torch.float32, gen).to(dev).requires_grad_(True)
    t = torch.randint(0, 300, (2, 5), generator=gen).to(dev)
    ids, u = (a.to(dev) for a in teacher_of(leaf.detach().cpu()[:, :-1], 8, gen, torch.float32))

    def losses(full):
        lp = m3.token_logprobs(full[:, :-1], t, top=4)
        kd = m3.distill_loss(full[:, :-1], ids, u, temperature=2.0, targets=t)
        return lp.logp.sum() + lp.entropy.sum() + lp.top_logp.sum(), kd.kd.sum() + kd.nll.sum()

    want = [torch.autograd.grad(losses(leaf * 1.0)[i], leaf)[0] for i in (0, 1)]
    for i in (0, 1):
        full = leaf * 1.0

        def unpack(held):
            if held.shape != (2, 5, 300):
                return held
            place = full.detach().reshape(-1)[:held.numel()].view(held.shape)
            assert place.data_ptr() == full.data_ptr()
            return place.copy_(held)

        def pack(saved):   # the small operands stay where they are
            return saved.detach().cpu().contiguous() if saved.shape == (2, 5, 300) else saved.detach()

        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = losses(full)[i]
        assert torch.equal(torch.autograd.grad(out, leaf)[0], want[i])


def test_nodes_refuse_what_they_cannot_do(m3, dev):
    x = torch.randn(3, 10, device=dev, requires_grad=True)
    t = torch.tensor([1, 2, 3], device=dev)
    lp = m3.token_logprobs(x, t).logp.sum()
    (dx,) = torch.autograd.grad(lp, x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level():
        dual = fwad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: m3.token_logprobs(dual, t),
                     lambda: m3.distill_loss(dual, t[:, None], x.detach()[:, :1])):
            with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError)):
                call()
    with pytest.raises(ValueError, match="must not require a gradient"):
        m3.distill_loss(x, t[:, None], x[:, :1])


def test_model_scores_and_distillation_step(m3, dev):
    """`model.lm_logprobs`, `model.lm_distill_loss` and `train.make_distill_step` on small models: the
    losses against float64 formulas of the same logits, the logits' part of the gradient through the
    whole model, and the step against its pieces (equal: the same launches)."""
    M, TR = m3.model, m3.train
    siso = m3.SISOConfig(d_model=64, d_state=16, headdim=16, expand=1, chunk=64, policy_name="f32")
    cfg = M.LMConfig(vocab_size=40, n_layers=2, siso=siso)
    big = M.LMConfig(vocab_size=40, n_layers=3, siso=siso, d_intermediate=48)
    student, teacher = M.init_lm(cfg, 1, device=dev), M.init_lm(big, 2, device=dev)
    gen = torch.Generator().manual_seed(3)
    xs = torch.randint(0, 40, (2, 128), generator=gen).to(dev)
    ys = torch.randint(0, 40, (2, 128), generator=gen).to(dev)
    ys[1, 70:] = -100
    with torch.no_grad():
        best = M.lm_logprobs(teacher, xs, ys, big, top=8)
        logits = M.lm_forward(teacher, xs, big)
    logp, h, top_lp, ids, _, _ = logprob_ref(logits.cpu().reshape(-1, 40), ys.cpu().reshape(-1), 8, 1.0)
    assert torch.equal(best.top_ids.cpu().reshape(-1, 8), ids)
    same(best.logp.reshape(-1), logp, bounds(logits.cpu().double().reshape(-1, 40), 1.0)[1], "logp")

    def grads(p):
        loss = M.lm_distill_loss(p, xs, ys, best.top_ids, best.top_logp, cfg, 2.0, 0.3)
        return loss.detach(), torch.autograd.grad(loss, M.lm_leaves(p))

    p = TR.train_params(student)
    loss, got = grads(p)
    x = M.lm_forward(p, xs, cfg)
    live = ys != -100
    w = torch.softmax(best.top_logp[live] / 2.0, -1)
    kd = 4.0 * (w * (w.log() - torch.log_softmax(x[live] / 2.0, -1).gather(-1, best.top_ids[live]))).sum(-1)
    ref = 0.7 * kd.mean() + 0.3 * torch.nn.functional.cross_entropy(x[live], ys[live])
    want = torch.autograd.grad(ref, M.lm_leaves(p))
    assert abs(loss.item() - ref.item()) <= 1e-5 * abs(ref.item())
    for a, b in zip(got, want):
        assert ((a - b).abs().max() / b.abs().max().clamp_min(1e-20)).item() <= 1e-4
    opt = TR.make_optimizer(p, lr=1e-3, warmup=1, steps=10)
    step = TR.make_distill_step(cfg, opt, teacher, big, k=8, temperature=2.0, hard_weight=0.3)
    q = TR.train_params(student)
    opt2 = TR.make_optimizer(q, lr=1e-3, warmup=1, steps=10)
    first = [t.detach().clone() for t in M.lm_leaves(q)]
    got_loss, _, _ = step(p, opt, xs, ys)
    ref_loss, ref_grads = grads(q)
    opt2.step(list(ref_grads))
    assert torch.equal(got_loss, ref_loss)
    assert all(torch.equal(a, b) for a, b in zip(M.lm_leaves(p), M.lm_leaves(q)))
    assert any(not torch.equal(a, b) for a, b in zip(M.lm_leaves(p), first))
    # a part of weight 0 is not there at all, as where the student rules a teacher's token out
    for weight, part in ((0.0, kd.mean()), (1.0, torch.nn.functional.cross_entropy(x[live], ys[live]))):
        only = M.lm_distill_loss(TR.train_params(student), xs, ys, best.top_ids, best.top_logp, cfg, 2.0, weight)
        assert abs(only.item() - part.item()) <= 1e-5 * abs(part.item())
    with pytest.raises(ValueError, match="vocabulary"):
        TR.make_distill_step(cfg, opt, teacher, M.LMConfig(vocab_size=41, n_layers=1, siso=siso))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(300, 32000), (1100, 4000)])
def test_small_terms_beside_a_likely_token(m3, dev, dtype, rows, vocab):
    """A row of one logit 0 and the rest at -16.75: their terms e^-16.75 = 0.89 eps (eps = 2^-24) are
    below half of a step of 1, so a running sum that starts with the likely token takes none of them,
    and the row's sum is short of one for each that the token's thread meets (124 of 32000, 61 of
    4000: 110 and 54 eps). Summed batch by batch, the 15 terms beside the likely one are lost at most, 13.4
    eps; each of the sums that are added to it, of up to 7 batches, 4 pieces and a rest, and the 8 joins
    across lanes and waves, round by at most half a step of a number below 2, one eps each: 34 eps. The
    terms' own errors (exp2's, their argument's and their sums', under 100 eps of the 0.0017 that they sum
    to), the logarithm of 1 + 0.0017 and the result's roundings are under one eps together. log s
    is off by no more than s: 35 eps."""
    term = math.exp(-16.75)
    x = torch.full((rows, vocab), -16.75).to(dtype)
    x[:, 0] = 0.0
    targets = torch.zeros(rows, dtype=torch.int64)
    want = -math.log1p((vocab - 1) * term)
    xd, t = x.to(dev), targets.to(dev)
    ids = torch.zeros(rows, 1, dtype=torch.int64, device=dev)
    u = torch.zeros(rows, 1, device=dev)
    K = m3.kernels
    calls = {"logp": K.logprob_forward(xd, t)[0], "top": K.logprob_forward(xd, t, top=2)[2][:, 0],
             "nll": -K.distill_forward(xd, ids, u, t)[1], "kd": -K.distill_forward(xd, ids, u)[0],
             "nll beside another temperature": -K.distill_forward(xd, ids, u, t, 1.5)[1]}
    for what, got in calls.items():
        assert (got.double() - want).abs().max().item() <= 35 * EPS, what


@pytest.mark.parametrize("weight", [0.0, 0.3, 1.0])
def test_distillation_of_padding_alone(m3, dev, weight):
    """A batch in which every position is padding has nothing to learn: a loss of 0 and gradients of
    zeros, and a step leaves finite parameters."""
    M, TR = m3.model, m3.train
    siso = m3.SISOConfig(d_model=64, d_state=16, headdim=16, expand=1, chunk=64, policy_name="f32")
    cfg = M.LMConfig(vocab_size=40, n_layers=1, siso=siso)
    params = TR.train_params(M.init_lm(cfg, 1, device=dev))
    gen = torch.Generator().manual_seed(3)
    xs = torch.randint(0, 40, (2, 64), generator=gen).to(dev)
    ys = torch.full((2, 64), -100, device=dev)
    ids, u = torch.zeros(2, 64, 4, dtype=torch.int64, device=dev), torch.randn(2, 64, 4, generator=gen).to(dev)
    loss = M.lm_distill_loss(params, xs, ys, ids, u, cfg, 2.0, weight)
    assert loss.item() == 0.0
    for g in torch.autograd.grad(loss, M.lm_leaves(params)):
        assert not g.any()
    opt = TR.make_optimizer(params, lr=1e-3, warmup=1, steps=10)
    step = TR.make_distill_step(cfg, opt, M.init_lm(cfg, 2, device=dev), cfg, k=4, hard_weight=weight)
    got, _, _ = step(params, opt, xs, ys)
    assert got.item() == 0.0 and all(p.isfinite().all() for p in M.lm_leaves(params))


def test_alternatives_past_31_bits(m3, dev):
    """The alternatives of the last rows of logits with more than 2^31 entries: their ids equal those of the
    rows on their own, and everything else is the formulas'."""
    gen = torch.Generator().manual_seed(13)
    rows, v, temp = 68000, 32000, 1.5
    x = torch.zeros(rows, v, device=dev, dtype=torch.bfloat16)
    last = make_logits((8, v), torch.bfloat16, gen)
    x[-8:] = last.to(dev)
    t = torch.full((rows,), -100, device=dev)
    t[-8:] = torch.randint(0, v, (8,), generator=gen).to(dev)
    logp, h, top_lp, ids, _, _ = logprob_ref(last, t[-8:].cpu(), 20, temp)
    _, tol_lp, tol_h = bounds(last.double(), temp)
    out = m3.kernels.logprob_forward(x, t, 20, temp)
    assert torch.equal(out[3][-8:].cpu(), ids) and (out[3][:-8] == -1).all()
    assert torch.equal(out[3][-8:], m3.kernels.logprob_forward(last.to(dev), t[-8:], 20, temp)[3])
    same(out[0][-8:], logp, tol_lp, "logp")
    same(out[1][-8:], h, tol_h, "entropy")
    same(out[2][-8:], top_lp, tol_lp[:, None], "top_logp")
