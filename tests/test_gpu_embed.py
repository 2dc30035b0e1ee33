"""GPU parity of the embedding lookup and its gradient (`m3s_embed_fwd` / `m3s_embed_bwd`)
against float64 sums on the CPU.

Tolerances:
  * forward: the scale is a float32 (22.7 is not one: half a step), one float32 product (half a
    step), and for bf16 one rounding to that type: 2 2^-24 relative in float32, and 2^-8 more in
    bf16 (second-order terms are covered by a factor 1 + 2^-8); with scale 1 bit-identical.
  * gradient: a row that sums n values of magnitude at most m in float32, in pieces, is off by at
    most n 2^-24 times the sum of the magnitudes (n additions, each of a partial sum no larger),
    then the scale's two roundings and the type's, as above.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24


def scaled_step(dtype):
    """The relative error of one product with the scale, rounded to ``dtype``."""
    return 2 * EPS32 if dtype == torch.float32 else (2 * EPS32 + 2.0 ** -8) * (1 + 2.0 ** -8)


def reference(tokens, dy, vocab, scale, pad):
    """The gradient in float64 and the bound on the float32 sums' error, element by element."""
    ids = tokens.reshape(-1).cpu().long()
    rows = dy.reshape(-1, dy.shape[-1]).cpu().double()
    ok = (ids >= 0) & (ids < vocab)
    if pad is not None:
        ok &= ids != pad % vocab
    ids, rows = ids[ok], rows[ok]
    want = torch.zeros(vocab, rows.shape[-1], dtype=torch.float64).index_add_(0, ids, rows)
    mag = torch.zeros_like(want).index_add_(0, ids, rows.abs())
    n = torch.bincount(ids, minlength=vocab).double().unsqueeze(1)
    return want * scale, n * EPS32 * mag * abs(scale)


def check_grad(got, tokens, dy, scale, pad):
    want, err = reference(tokens, dy, got.shape[0], scale, pad)
    tol = err * (1 + 2.0 ** -7) + want.abs() * scaled_step(got.dtype) + 1e-38
    over = ((got.cpu().double() - want).abs() / tol).max().item()
    assert over <= 1.0


def skewed(vocab, shape, gen, dtype=torch.int64):
    u = torch.rand(shape, generator=gen, dtype=torch.float64)
    return ((vocab + 1.0) ** u - 1).floor().clamp(0, vocab - 1).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("vocab,d,shape,scale", [
    (1, 1, (1,), 1.0), (7, 3, (5, 2), 1.0), (40, 5, (64,), 2.5), (256, 768, (3, 700), 1.0),
    (257, 260, (4097,), 0.5), (511, 64, (2, 2500), 1.0), (512, 17, (33, 3), 1.0),
    (5003, 515, (4, 1025), 22.7), (300, 1100, (2000,), 1.0), (70001, 36, (9000,), 6.0), (300007, 8, (3001,), 1.0)])
def test_lookup_and_gradient(m3, dev, dtype, ids, vocab, d, shape, scale):
    gen = torch.Generator().manual_seed(vocab + d)
    table = torch.randn(vocab, d, generator=gen).to(dtype)
    tokens = skewed(vocab, shape, gen, ids)
    dy = torch.randn(*shape, d, generator=gen).to(dtype)
    w = table.to(dev).requires_grad_(True)
    y = m3.embed_tokens(w, tokens.to(dev), scale=scale)
    want = table[tokens.long()].double() * scale
    assert y.dtype == dtype and y.shape == (*shape, d)
    if scale == 1.0:
        assert torch.equal(y.detach().cpu(), table[tokens.long()])
    over = (y.detach().cpu().double() - want).abs() / (want.abs() * scaled_step(dtype) + 1e-38)
    assert over.max().item() <= 1.0
    (dw,) = torch.autograd.grad(y, w, dy.to(dev))
    assert dw.dtype == dtype and dw.shape == (vocab, d)
    check_grad(dw, tokens, dy, scale, None)
    with torch.no_grad():
        assert torch.equal(m3.embed_tokens(w, tokens.to(dev), scale=scale), y)


@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 64, 1023, 1024, 1025, 4095, 4096, 4097, 8192, 40000])
def test_sort_sizes_and_single_ids(m3, dev, n):
    """Lengths around the pieces, the workgroups and the switch of the sort; every token the same
    id, ids in order, and ids against the order."""
    gen = torch.Generator().manual_seed(n)
    d, vocab = 12, 1000
    dy = torch.randn(n, d, generator=gen)
    for tokens in (torch.full((n,), 999), torch.arange(n) % vocab, (n - 1 - torch.arange(n)) * vocab // max(n, 1),
                   skewed(vocab, (n,), gen)):
        got = m3.kernels.embedding_backward(tokens.to(dev), dy.to(dev), vocab)
        check_grad(got, tokens, dy, 1.0, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,d", [(1, 6), (3, 700), (1023, 40), (1024, 515), (1025, 260), (2049, 9), (70001, 300),
                                     (1100003, 8)])
def test_few_tokens(m3, dev, dtype, vocab, d):
    """Up to 1024 tokens, which are listed and not sorted: rows of one token, of the most that one wave
    adds, of more, and of all; tables whose rows end inside a stride; ids one stride apart."""
    gen = torch.Generator().manual_seed(vocab + d)
    for n in (1, 16, 17, 63, 65, 500, 1000, 1024):
        dy = torch.randn(n, d, generator=gen).to(dtype)
        hot = skewed(vocab, (n,), gen)
        hot[torch.rand(n, generator=gen) < 0.3] = vocab - 1
        pairs = torch.arange(n) // 16 % vocab
        strides = torch.arange(n) * 1024 % vocab
        for tokens in (torch.full((n,), vocab // 2), hot, pairs, strides, torch.randperm(n, generator=gen) % vocab):
            got = m3.kernels.embedding_backward(tokens.to(dev), dy.to(dev), vocab, 0.5)
            check_grad(got, tokens, dy, 0.5, None)
        holes = hot.clone()
        holes[::3] = torch.tensor([-1, vocab, 1 << 40])[torch.arange(len(holes[::3])) % 3]
        dy[::3] = float("nan")   # read by nobody
        for pad in (None, vocab - 1):
            got = m3.kernels.embedding_backward(holes.to(dev), dy.to(dev), vocab, 0.5, padding_idx=pad)
            check_grad(got, holes, dy, 0.5, pad)


def test_few_tokens_of_a_large_table(m3, dev):
    """Past 2^26 entries few tokens are sorted too."""
    gen = torch.Generator().manual_seed(5)
    vocab, d = 70001, 961
    tokens, dy = skewed(vocab, (900,), gen), torch.randn(900, d, generator=gen)
    check_grad(m3.kernels.embedding_backward(tokens.to(dev), dy.to(dev), vocab, 0.5), tokens, dy, 0.5, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_and_ids_outside_the_table(m3, dev, dtype):
    """The padding id's row is looked up and gets zeros back; an id outside the table gives NaN and
    adds to no row, whatever its cotangent holds."""
    gen = torch.Generator().manual_seed(3)
    vocab, d = 300, 96
    table = torch.randn(vocab, d, generator=gen).to(dtype)
    tokens = skewed(vocab, (5, 400), gen)
    tokens[1, 100:] = vocab - 1
    dy = torch.randn(5, 400, d, generator=gen).to(dtype)
    for pad in (vocab - 1, -1, 0, None):
        w = table.to(dev).requires_grad_(True)
        y = m3.embed_tokens(w, tokens.to(dev), padding_idx=pad)
        assert torch.equal(y.detach().cpu(), table[tokens])
        (dw,) = torch.autograd.grad(y, w, dy.to(dev))
        check_grad(dw, tokens, dy, 1.0, pad)
    bad = tokens.clone()
    outside = torch.rand(bad.shape, generator=gen) < 0.1
    bad[outside] = torch.tensor([-1, -100, vocab, 1 << 40])[torch.arange(int(outside.sum())) % 4]
    w = table.to(dev).requires_grad_(True)
    y = m3.embed_tokens(w, bad.to(dev))
    assert y[outside.to(dev)].isnan().all() and not y[~outside.to(dev)].isnan().any()
    dy[outside] = float("nan")
    (dw,) = torch.autograd.grad(y, w, dy.to(dev))
    check_grad(dw, bad, dy, 1.0, None)


def test_gradient_is_bit_reproducible_and_matches_differences(m3, dev):
    gen = torch.Generator().manual_seed(8)
    tokens = skewed(256, (6, 2048), gen).to(dev)
    dy = torch.randn(6, 2048, 100, generator=gen).to(dev)
    first = m3.kernels.embedding_backward(tokens, dy, 256)
    for _ in range(3):
        assert torch.equal(m3.kernels.embedding_backward(tokens, dy, 256), first)
    # the lookup is linear: a step h of one entry moves <y, dy> by h times that gradient entry
    table = torch.randn(256, 100, generator=gen).to(dev)
    step = torch.zeros_like(table)
    step[0, 7] = 0.5
    f = lambda t: (m3.embed_tokens(t, tokens, scale=3.0).double() * dy.double()).sum()  # noqa: E731
    slope = (f(table + step) - f(table - step)).item()
    want = m3.kernels.embedding_backward(tokens, dy, 256, 3.0)[0, 7].item()
    assert abs(slope - want) <= 1e-4 * abs(want) + 1e-3


def test_offsets_past_31_bits(m3, dev):
    """The last rows of a table, and the last tokens, with more than 2^31 entries before them."""
    gen = torch.Generator().manual_seed(2)
    vocab, d = 2200000, 1024
    table = torch.zeros(vocab, d, device=dev, dtype=torch.bfloat16)
    last = torch.randn(16, d, generator=gen).to(torch.bfloat16).to(dev)
    table[-16:] = last
    tokens = (vocab - 16 + torch.arange(16)).to(dev)
    assert torch.equal(m3.embed_tokens(table, tokens), last)
    dw = m3.kernels.embedding_backward(tokens, last, vocab)
    assert torch.equal(dw[-16:], last) and not dw[:1000].any() and not dw[-1000:-16].any()
    del table, dw
    tokens = torch.zeros(vocab, dtype=torch.int32, device=dev)
    tokens[-16:] = 1 + torch.arange(16, device=dev)
    y = m3.embed_tokens(last.repeat(2, 1)[:17].contiguous(), tokens)
    assert torch.equal(y[-16:], last.repeat(2, 1)[1:17]) and torch.equal(y[0], last[0])
    dw = m3.kernels.embedding_backward(tokens, y, 17, padding_idx=0)
    assert not dw[0].any() and torch.equal(dw[1:], y[-16:])


def test_strides_broadcast_cotangents_and_views(m3, dev):
    """A table that is a slice of a wider one, tokens that are a strided view, and a cotangent
    that is broadcast."""
    gen = torch.Generator().manual_seed(4)
    wide = torch.randn(90, 48, generator=gen).to(dev)
    table = wide[:, 7:40]
    tokens = torch.randint(0, 90, (6, 50), generator=gen).to(dev).t()[::2]
    assert torch.equal(m3.embed_tokens(table, tokens), table[tokens])
    assert torch.equal(m3.embed_tokens(wide.t(), tokens % 48), wide.t()[tokens % 48])
    dy = torch.randn(33, generator=gen).to(dev).expand(*tokens.shape, 33)
    check_grad(m3.kernels.embedding_backward(tokens, dy, 90), tokens.cpu(), dy.cpu(), 1.0, None)
    w = table.detach().requires_grad_(True)
    m3.embed_tokens(w, tokens).sum().backward()
    check_grad(w.grad, tokens.cpu(), torch.ones(*tokens.shape, 33), 1.0, None)
    one = m3.embed_tokens(table, tokens[0, 0])   # a single id without axes
    assert one.shape == (33,) and torch.equal(one, table[tokens[0, 0]])


def test_captured_calls_replay_on_new_inputs(m3, dev):
    """Lookup and gradient inside a recorded graph, replayed on changed ids and cotangents with
    other work between the replays."""
    gen = torch.Generator().manual_seed(6)
    vocab, d = 700, 64
    table = torch.randn(vocab, d, generator=gen).to(dev)
    for n in (50, 6000):
        tokens = torch.zeros(n, dtype=torch.int64, device=dev)
        dy = torch.zeros(n, d, device=dev)
        side = torch.cuda.Stream(dev)
        with torch.cuda.stream(side):
            m3.kernels.embedding_forward(table, tokens), m3.kernels.embedding_backward(tokens, dy, vocab)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m3.kernels.embedding_forward(table, tokens, 2.0)
            dw = m3.kernels.embedding_backward(tokens, dy, vocab, 2.0, padding_idx=3)
        for _ in range(3):
            tokens.copy_(skewed(vocab, (n,), gen))
            dy.copy_(torch.randn(n, d, generator=gen))
            graph.replay()
            assert torch.equal(y, m3.kernels.embedding_forward(table, tokens, 2.0))
            assert torch.equal(dw, m3.kernels.embedding_backward(tokens, dy, vocab, 2.0, padding_idx=3))
            torch.cuda.synchronize()


def test_calls_on_another_stream_and_two_at_once(m3, dev):
    gen = torch.Generator().manual_seed(9)
    a, b = (skewed(400, (5000,), gen).to(dev) for _ in range(2))
    dy = torch.randn(5000, 32, generator=gen).to(dev)
    want = [m3.kernels.embedding_backward(t, dy, 400) for t in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for s, t in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(m3.kernels.embedding_backward(t, dy, 400))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_model_lookup_keeps_what_it_took(m3, dev):
    """`model._embed` still takes tables and modes that the kernels do not."""
    table = torch.randn(11, 6, device=dev, dtype=torch.float64, requires_grad=True)
    tokens = torch.tensor([[1, 2], [10, 0]], device=dev)
    y = m3.model._embed(table, tokens)
    assert torch.equal(y, table[tokens])
    y.sum().backward()
    assert table.grad[1, 0] == 1 and table.grad[3, 0] == 0
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level():
        dual = fwad.make_dual(table.detach().float(), torch.ones(11, 6, device=dev))
        assert (fwad.unpack_dual(m3.model._embed(dual, tokens)).tangent == 1).all()
        with pytest.raises((NotImplementedError, RuntimeError)):
            m3.embed_tokens(dual, tokens)


def test_lookup_node_is_in_cpp(m3, dev):
    """A small training step's embedding is the host's to pay for: the node of ordinary operands runs
    without the interpreter, through the entry point and through the model, in any shape and type."""
    python_node = torch.autograd.function.BackwardCFunction
    for dtype in (torch.float32, torch.bfloat16):
        for ids in (torch.int32, torch.int64):
            w = torch.randn(300, 24, device=dev).to(dtype).requires_grad_(True)
            tokens = torch.randint(0, 300, (4, 9), device=dev, dtype=ids)
            for y in (m3.embed_tokens(w, tokens), m3.embed_tokens(w[:, 3:19], tokens[0]), m3.model._embed(w, tokens)):
                assert y.requires_grad and not isinstance(y.grad_fn, python_node)
            with torch.no_grad():
                assert not m3.embed_tokens(w, tokens).requires_grad
    strided = m3.embed_tokens(w.t(), tokens.t() % 24)   # copied first, by the node in Python
    assert isinstance(strided.grad_fn, python_node)
    assert torch.equal(strided, w.t()[tokens.t() % 24])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [0, 1, 40, 3000, 30000])
def test_node_gradients_are_the_bare_calls(m3, dev, dtype, n):
    """Through the graph and by `kernels.embedding_backward`: the same bits, with a cotangent that is
    dense, broadcast, strided or absent, twice from one graph, and into slices of a wider table."""
    gen = torch.Generator().manual_seed(n)
    K, vocab, d = m3.kernels, 200, 40
    w = torch.randn(vocab, d, generator=gen).to(dtype).to(dev).requires_grad_(True)
    tokens = skewed(vocab, (n,), gen).to(dev)
    dys = [torch.randn(n, d, generator=gen).to(dtype).to(dev), torch.ones(1, 1, dtype=dtype, device=dev).expand(n, d),
           torch.randn(d, n, generator=gen).to(dtype).to(dev).t()]
    y = m3.embed_tokens(w, tokens, scale=1.5, padding_idx=-1)
    assert torch.equal(y, K.embedding_forward(w.detach(), tokens, 1.5))
    for dy in dys:
        (dw,) = torch.autograd.grad(y, w, dy, retain_graph=True)
        assert torch.equal(dw, K.embedding_backward(tokens, dy, vocab, 1.5, vocab - 1))
    y.backward(dys[0])
    assert torch.equal(w.grad, K.embedding_backward(tokens, dys[0], vocab, 1.5, vocab - 1))
    with pytest.raises(RuntimeError, match="second time"):
        y.backward(dys[0])
    part = m3.embed_tokens(w[:, 8:24], tokens)
    (dw,) = torch.autograd.grad(part, w, dys[0][:, :16])
    assert torch.equal(dw[:, 8:24], K.embedding_backward(tokens, dys[0][:, :16], vocab))
    assert not dw[:, :8].any() and not dw[:, 24:].any()


def test_node_refusals_and_saved_tokens(m3, dev):
    """No second derivative, no use of ids that changed in between, and ids that a hook kept elsewhere."""
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(50, 8, generator=gen).to(dev).requires_grad_(True)
    tokens = skewed(50, (30,), gen).to(dev)
    dy = torch.randn(30, 8, generator=gen).to(dev).requires_grad_(True)
    (dw,) = torch.autograd.grad(m3.embed_tokens(w, tokens), w, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(dw.sum(), dy)
    want = m3.kernels.embedding_backward(tokens, dy.detach(), 50)
    assert torch.equal(dw, want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.repeat(2).to(dev)[::2][:30]):
        y = m3.embed_tokens(w, torch.arange(30, device=dev))   # comes back strided, other ids
    (got,) = torch.autograd.grad(y, w, dy.detach())
    assert torch.equal(got, m3.kernels.embedding_backward(torch.arange(30).repeat(2)[::2][:30].to(dev), dy.detach(), 50))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:7]):
        y = m3.embed_tokens(w, tokens)
    with pytest.raises(ValueError, match="another kind"):
        torch.autograd.grad(y, w, dy.detach())
    y = m3.embed_tokens(w, tokens)
    tokens.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, w, dy.detach())


def test_captured_training_pass_replays_on_new_inputs(m3, dev):
    """Lookup and gradient through autograd inside a recorded graph, replayed on changed tables, ids and
    cotangents, every replay against the bare calls."""
    gen = torch.Generator().manual_seed(16)
    vocab, d, K = 300, 64, m3.kernels
    for n in (50, 6000):
        table = torch.zeros(vocab, d, device=dev)
        tokens = torch.zeros(n, dtype=torch.int64, device=dev)
        dy = torch.zeros(n, d, device=dev)

        def step():
            w = table.detach().requires_grad_(True)   # a leaf of its own: no eager graph shares it
            y = m3.embed_tokens(w, tokens, scale=2.0, padding_idx=3)
            return y.detach(), torch.autograd.grad(y, w, dy)[0]

        side = torch.cuda.Stream(dev)
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            table.copy_(torch.randn(vocab, d, generator=gen))
            tokens.copy_(skewed(vocab, (n,), gen))
            dy.copy_(torch.randn(n, d, generator=gen))
            graph.replay()
            assert torch.equal(out[0], K.embedding_forward(table, tokens, 2.0))
            assert torch.equal(out[1], K.embedding_backward(tokens, dy, vocab, 2.0, padding_idx=3))
            torch.cuda.synchronize()


def test_node_runs_on_the_streams_of_its_forward(m3, dev):
    """Two training passes on streams of their own at once, backward called from the default stream."""
    gen = torch.Generator().manual_seed(19)
    ws = [torch.randn(400, 32, generator=gen).to(dev).requires_grad_(True) for _ in range(2)]
    ids = [skewed(400, (5000,), gen).to(dev) for _ in range(2)]
    dy = torch.randn(5000, 32, generator=gen).to(dev)
    want = [m3.kernels.embedding_backward(t, dy, 400) for t in ids]
    torch.cuda.synchronize()
    ys = []
    for w, t in zip(ws, ids):
        with torch.cuda.stream(torch.cuda.Stream(dev)):
            ys.append(m3.embed_tokens(w, t))
    torch.cuda.synchronize()
    got = [torch.autograd.grad(y, w, dy)[0] for y, w in zip(ys, ws)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, x) for g, x in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,d", [(22003, 256, 768), (33000, 256, 1030), (70001, 300, 20), (40000, 1000, 12),
                                       (14001, 256, 700), (9000, 300007, 8), (5000, 1 << 18, 5), (66000, 262143, 9)])
def test_gradient_of_training_batches(m3, dev, dtype, n, vocab, d):
    """Long batches: pieces of 32 and of 16 sorted rows (65536 and 32768 rows times column tiles of 256
    on) in one and in several tiles, ids in every piece and in hundreds of them, and sorts of two and three
    passes by several workgroups."""
    gen = torch.Generator().manual_seed(n)
    dy = torch.randn(n, d, generator=gen).to(dtype)
    dyd = dy.to(dev)
    one = torch.full((n,), vocab - 2)
    one[::7001] = 1
    for tokens, pad in ((skewed(vocab, (n,), gen), None), (one, None), (skewed(vocab, (n,), gen), 0)):
        got = m3.kernels.embedding_backward(tokens.to(dev), dyd, vocab, 0.5, pad)
        check_grad(got, tokens, dy, 0.5, pad)
        assert torch.equal(got, m3.kernels.embedding_backward(tokens.to(dev).int(), dyd, vocab, 0.5, pad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 8, 65, 129, 515, 768, 1100, 4092, 4095, 4096, 4097, 8191, 8192, 8195, 40003])
def test_lookup_of_every_row_form(m3, dev, dtype, d):
    """Rows narrower than 16 bytes, of lanes that divide them evenly or not, and of 16 KB and more, dense
    and as slices of wider ones; ids outside the table among them. A product in float32, rounded once:
    the same bits as torch's."""
    gen = torch.Generator().manual_seed(d)
    wide = torch.randn(37, d + 5, generator=gen).to(dtype).to(dev)
    for n in (1, 2, 700, 1031):
        tokens = torch.randint(0, 37, (n,), generator=gen)
        tokens[3::50] = torch.tensor([-1, 37, 1 << 40])[torch.arange(len(tokens[3::50])) % 3]
        tokens = tokens.to(dev)
        bad = (tokens < 0) | (tokens >= 37)
        for table in (wide[:, :d].contiguous(), wide[:, 3:3 + d]):
            for scale in (1.0, 22.7):
                y = m3.embed_tokens(table, tokens, scale=scale)
                want = (table[tokens.clamp(0, 36)].float() * scale).to(dtype)
                assert torch.equal(y[~bad], want[~bad]) and y[bad].isnan().all()
