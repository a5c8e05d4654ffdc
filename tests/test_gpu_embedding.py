"""ops.embedding and ops.embedding_grad against their definitions in 64 bits.

Tolerances. The lookup rounds the scale and the product to fp32 and the result to its type: off by at most
2^-23 + eps/2 of the value. The gradient of a token that occurs c times adds c terms in fp32, in whatever grouping:
off by at most (c + 2) 2^-24 of the sum of their magnitudes (c - 1 additions, the scale, the product), and eps/2 of the
value for the store; fp16 results below its normal range by half of its smallest step, 2^-25."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_tokens(kind, n, vocab, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "text":
        t = (float(vocab) ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, vocab - 1) * 7919 % vocab
    elif kind == "same":
        t = torch.full((n,), vocab - 1)
    elif kind == "distinct":
        t = torch.randperm(max(n, vocab), generator=g)[:n] % vocab
    elif kind == "falling":
        t = torch.arange(n).flip(0) % vocab
    else:  # outside: some below, some above the table
        t = torch.randint(-3, vocab + 3, (n,), generator=g)
    return t.to(dtype)


def exact_grad(grad, tokens, vocab, scale, padding):
    """(the gradient, the sum of magnitudes, how often the token occurs), in 64 bits on the CPU."""
    dim = grad.shape[-1]
    t, g = tokens.reshape(-1).cpu().long(), grad.reshape(-1, dim).cpu().double()
    keep = (t >= 0) & (t < vocab) & (t != (-1 if padding is None else padding % vocab))
    t, g = t[keep], g[keep]
    out, mag, count = torch.zeros(vocab, dim, dtype=torch.float64), torch.zeros(vocab, dim, dtype=torch.float64), torch.zeros(vocab, dtype=torch.float64)
    out.index_add_(0, t, g * scale)
    mag.index_add_(0, t, g.abs() * abs(scale))
    count.index_add_(0, t, torch.ones(len(t), dtype=torch.float64))
    return out, mag, count


def check_grad(got, grad, tokens, vocab, scale=1.0, padding=None):
    want, mag, count = exact_grad(grad, tokens, vocab, scale, padding)
    err = (got.cpu().double() - want).abs()
    allowed = (count[:, None] + 2) * 2.0 ** -24 * mag + half_step(got.dtype) * want.abs() * (1 + 2.0 ** -10)
    if got.dtype == torch.float16:
        allowed += 2.0 ** -25
    assert torch.isfinite(err).all()
    assert (err <= allowed).all(), f"off by {float((err - allowed).max()):.3g} more than allowed"
    assert (got.cpu()[count == 0] == 0).all()


LOOKUPS = [  # vocab, dim, tokens' shape, dtype, index, scale
    (256, 768, (4, 128), "fp32", torch.int64, 1.0),
    (256, 768, (16, 512), "bf16", torch.int64, 27.7128),
    (32000, 4096, (8, 1), "bf16", torch.int32, 64.0),
    (50021, 999, (1, 333), "fp16", torch.int32, 1.0),
    (7, 1, (3,), "fp16", torch.int64, 0.5),
    (5, 3, (1,), "fp32", torch.int32, -2.0),
    (1, 4100, (2, 2), "bf16", torch.int64, 1.0),
    (100, 62, (0,), "fp32", torch.int64, 1.0),
    (1000, 20, (70001,), "fp32", torch.int32, 3.0),
]


@pytest.mark.parametrize("vocab,dim,shape,dtype,index,scale", LOOKUPS)
def test_lookup(vocab, dim, shape, dtype, index, scale):
    from tandem_amd import ops

    dtype = DT[dtype]
    w = torch.randn(vocab, dim, generator=torch.Generator().manual_seed(1)).to(dtype)
    tokens = make_tokens("text", int(np.prod(shape)), vocab, 2, index).view(shape)
    got = ops.embedding(tokens.to(DEV), w.to(DEV), scale=scale)
    assert got.shape == (*shape, dim) and got.dtype == dtype
    want = w.double()[tokens.long()] * scale
    assert ((got.cpu().double() - want).abs() <= (2.0 ** -23 + half_step(dtype)) * want.abs()).all()


def test_lookup_from_a_table_off_the_vector_grid():
    from tandem_amd import ops

    store = torch.randn(100 * 24 + 3, device=DEV, dtype=torch.bfloat16)
    w = store[3:].view(100, 24)
    tokens = torch.arange(99, -1, -1, device=DEV)
    assert torch.equal(ops.embedding(tokens, w), w.flip(0))


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_tokens_outside_the_table(index):
    from tandem_amd import ops

    vocab, dim = 33, 40
    w = torch.randn(vocab, dim, device=DEV)
    tokens = make_tokens("outside", 500, vocab, 3, index)
    tokens[0], tokens[1] = torch.iinfo(index).max, torch.iinfo(index).min
    got = ops.embedding(tokens.to(DEV), w).cpu()
    inside = (tokens >= 0) & (tokens < vocab)
    assert torch.isnan(got[~inside]).all() and torch.equal(got[inside], w.cpu()[tokens[inside].long()])
    g = torch.randn(500, dim, device=DEV)
    check_grad(ops.embedding_grad(g, tokens.to(DEV), vocab), g, tokens, vocab)
    nothing = torch.full((77,), -1, dtype=index, device=DEV)  # no token takes a gradient
    assert (ops.embedding_grad(g[:77], nothing, vocab) == 0).all()


GRADS = [  # vocab, dim, n, tokens, dtype, index, scale, padding
    (256, 768, 8192, "text", "fp32", torch.int64, 1.0, None),
    (256, 96, 8191, "text", "bf16", torch.int32, 2.0, 0),
    (511, 64, 8193, "text", "fp16", torch.int64, 1.0, -1),
    (512, 64, 1000, "falling", "fp32", torch.int64, 1.0, None),
    (513, 64, 1000, "distinct", "fp32", torch.int32, 1.0, 7),
    (1, 33, 5000, "same", "fp32", torch.int64, 1.0, None),
    (2, 8, 20000, "text", "bf16", torch.int64, 1.0, None),
    (1000, 17, 1, "text", "bf16", torch.int64, 4.0, None),
    (1000, 16, 2, "same", "fp16", torch.int64, 4.0, None),
    (300, 130, 15, "same", "fp32", torch.int64, 1.0, None),
    (300, 130, 16, "same", "fp32", torch.int64, 1.0, None),
    (300, 130, 17, "same", "fp32", torch.int64, 1.0, None),
    (50021, 999, 4099, "text", "fp16", torch.int32, 1.0, 7),
    (70000, 4, 70001, "text", "fp32", torch.int64, 1.0, None),
    (131072, 8, 65536, "distinct", "bf16", torch.int64, 1.0, None),
    (300000, 5, 66000, "text", "fp32", torch.int64, 1.0, None),
    (4000, 12, 66000, "same", "fp32", torch.int64, 1.0, None),
    (2000, 2048, 300, "text", "bf16", torch.int64, 45.25, None),
    (64, 1, 600, "text", "fp32", torch.int64, 1.0, None),
    (97, 5000, 40, "text", "bf16", torch.int64, 1.0, None),
]


@pytest.mark.parametrize("vocab,dim,n,kind,dtype,index,scale,padding", GRADS)
def test_gradient(vocab, dim, n, kind, dtype, index, scale, padding):
    from tandem_amd import ops

    tokens = make_tokens(kind, n, vocab, 4, index)
    grad = torch.randn(n, dim, generator=torch.Generator().manual_seed(5)).to(DT[dtype]).to(DEV)
    got = ops.embedding_grad(grad, tokens.to(DEV), vocab, scale=scale, padding_idx=padding)
    assert got.shape == (vocab, dim) and got.dtype == DT[dtype]
    check_grad(got, grad, tokens, vocab, scale, padding)
    again = ops.embedding_grad(grad, tokens.to(DEV), vocab, scale=scale, padding_idx=padding)
    assert torch.equal(got, again)


def test_gradient_of_more_tokens_than_one_merge_takes():
    """Past 8 tiles the runs are merged twice; past 64, three times. Few columns: the order is what is tested."""
    from tandem_amd import ops

    for n in (65537, 530001):
        tokens = make_tokens("text", n, 5000, 6)
        grad = torch.randn(n, 2, generator=torch.Generator().manual_seed(7))
        check_grad(ops.embedding_grad(grad.to(DEV), tokens.to(DEV), 5000), grad, tokens, 5000)


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 511, 512, 513, 32768, 32769, 131072, 262144, 262145])
@pytest.mark.parametrize("n,kind", [(8192, "text"), (8193, "text"), (8193, "same"), (12288, "outside"), (12289, "distinct"), (20000, "same"), (41000, "text")])
def test_every_way_of_sorting(vocab, n, kind):
    """Both sides of the sizes where the sort takes another form: 8192 tokens, 262144 rows; whole and ragged tiles, one token for all, few tokens,
    as many as there are. Counts and sums of small whole numbers are exact in fp32 below 2^24."""
    from tandem_amd import ops

    tokens = make_tokens(kind, n, vocab, 12)
    g = torch.Generator().manual_seed(13)
    grad = torch.stack([torch.ones(n), torch.arange(n) % 97.0, torch.randn(n, generator=g)], 1)
    got = ops.embedding_grad(grad.to(DEV), tokens.to(DEV), vocab)
    check_grad(got, grad, tokens, vocab)
    want, _, count = exact_grad(grad, tokens, vocab, 1.0, None)
    assert torch.equal(got[:, :2].cpu().double(), want[:, :2])  # whole numbers below 2^24
    assert torch.equal(got, ops.embedding_grad(grad.to(DEV), tokens.to(DEV), vocab))


@pytest.mark.parametrize("vocab,dim,dtype", [(1024, 128, torch.float32), (1025, 128, torch.float32), (256, 512, torch.float32), (341, 384, torch.float16),
                                             (512, 512, torch.bfloat16), (513, 512, torch.bfloat16), (97, 511, torch.bfloat16), (300, 33, torch.float32),
                                             (5, 6, torch.float16), (1, 1, torch.float32)])
@pytest.mark.parametrize("n,kind", [(1, "text"), (63, "same"), (64, "distinct"), (513, "outside"), (4095, "same"), (4096, "text"), (4097, "text")])
def test_small_tables(vocab, dim, dtype, n, kind):
    """Both sides of the sizes where one launch does it all: 4096 tokens, 1024 rows of 512 bytes; narrow and wide accesses, a padding row."""
    from tandem_amd import ops

    tokens = make_tokens(kind, n, vocab, 14)
    grad = torch.randn(n, dim, generator=torch.Generator().manual_seed(15)).to(dtype)
    for padding, index in ((None, torch.int64), (int(tokens[0]) if 0 <= int(tokens[0]) < vocab else 0, torch.int32)):
        got = ops.embedding_grad(grad.to(DEV), tokens.to(index).to(DEV), vocab, scale=0.5, padding_idx=padding)
        check_grad(got, grad, tokens, vocab, 0.5, padding)
        assert torch.equal(got, ops.embedding_grad(grad.to(DEV), tokens.to(index).to(DEV), vocab, scale=0.5, padding_idx=padding))


def test_more_tokens_than_the_tiles_of_a_split():
    from tandem_amd import ops

    n = (1 << 22) + 4097
    tokens = make_tokens("text", n, 3000, 14)
    grad = torch.ones(n, 1)
    got = ops.embedding_grad(grad.to(DEV), tokens.to(DEV), 3000)
    assert torch.equal(got[:, 0].cpu().long(), torch.bincount(tokens, minlength=3000))


def test_no_tokens_at_all():
    from tandem_amd import ops

    got = ops.embedding_grad(torch.empty(0, 48, device=DEV), torch.empty(0, device=DEV, dtype=torch.int64), 77)
    assert got.shape == (77, 48) and (got == 0).all()


def test_non_finite_rows_stay_with_their_token():
    from tandem_amd import ops

    grad = torch.zeros(64, 16, device=DEV)
    grad[10], grad[20] = float("inf"), float("nan")
    tokens = torch.arange(64, device=DEV) % 32
    got = ops.embedding_grad(grad, tokens, 32)
    assert torch.isinf(got[10]).all() and torch.isnan(got[20]).all()
    assert (got[torch.arange(32, device=DEV).remainder(10) != 0] == 0).all()


def test_autograd_with_views_and_expanded_gradients():
    from tandem_amd import ops

    w = torch.randn(100, 24, device=DEV, requires_grad=True)
    tokens = torch.randint(0, 100, (6, 11), generator=torch.Generator().manual_seed(8)).to(DEV)[:, :10]  # strided
    ops.embedding(tokens, w, scale=3.0, padding_idx=4).sum().backward()  # an expanded gradient
    check_grad(w.grad, torch.ones(6, 10, 24), tokens, 100, 3.0, 4)
    frozen = torch.randn(100, 24, device=DEV)
    assert not ops.embedding(tokens, frozen).requires_grad
    with torch.no_grad():
        assert not ops.embedding(tokens, w).requires_grad


def test_gradient_against_differences():
    """The loss sum(g * embedding(W)) is linear in W: a step h in one element moves it by h dW exactly. In fp32 the
    outputs are off by 2^-23 of themselves, so with |W|, |g| < 4, h = 1 and c uses of the row the quotient is off by less than
    2 c 16 2^-22."""
    from tandem_amd import ops

    vocab, dim = 9, 12
    w = torch.randn(vocab, dim, generator=torch.Generator().manual_seed(9)).clamp(-3, 3)
    tokens = make_tokens("text", 40, vocab, 10)
    g = torch.randn(40, dim, generator=torch.Generator().manual_seed(11)).clamp(-3, 3)
    dw = ops.embedding_grad(g.to(DEV), tokens.to(DEV), vocab, scale=1.5).cpu().double()
    for v in range(vocab):
        uses = int((tokens == v).sum())
        for c in (0, 5, 11):
            up = w.clone()
            up[v, c] += 1.0
            h = float(up[v, c].double() - w[v, c].double())
            losses = [float((ops.embedding(tokens.to(DEV), x.to(DEV), scale=1.5).cpu().double() * g.double()).sum()) for x in (up, w)]
            assert abs((losses[0] - losses[1]) / h - float(dw[v, c])) <= (uses + 1) * 32 * 1.5 * 2.0 ** -22


def test_a_captured_graph_replayed_on_other_tokens():
    from tandem_amd import ops

    vocab, dim, n = 300, 72, 9000
    w = torch.randn(vocab, dim, device=DEV)
    tokens, grad = torch.zeros(n, dtype=torch.int64, device=DEV), torch.zeros(n, dim, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            ops.embedding(tokens, w)
            ops.embedding_grad(grad, tokens, vocab)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding(tokens, w, scale=2.0)
        dw = ops.embedding_grad(grad, tokens, vocab, scale=2.0)
    for seed in (1, 2, 3):
        tokens.copy_(make_tokens("text", n, vocab, seed))
        grad.copy_(torch.randn(n, dim, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.embedding(tokens, w, scale=2.0))
        assert torch.equal(dw, ops.embedding_grad(grad, tokens, vocab, scale=2.0))
        check_grad(dw, grad, tokens, vocab, 2.0)


def test_two_streams_at_once():
    from tandem_amd import ops

    jobs = []
    for seed in range(4):
        tokens = make_tokens("text", 20000, 900, seed).to(DEV)
        grad = torch.randn(20000, 40, generator=torch.Generator().manual_seed(seed)).to(DEV)
        jobs.append((torch.cuda.Stream(), tokens, grad))
    torch.cuda.synchronize()
    got = []
    for stream, tokens, grad in jobs:
        with torch.cuda.stream(stream):
            got.append(ops.embedding_grad(grad, tokens, 900))
    torch.cuda.synchronize()
    for (_, tokens, grad), dw in zip(jobs, got):
        check_grad(dw, grad, tokens, 900)


def test_refusals_on_the_gpu():
    from tandem_amd import ops

    w, t = torch.randn(10, 4, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for call in (lambda: ops.embedding(t.float(), w), lambda: ops.embedding(t, w.double()), lambda: ops.embedding(t, w[0]),
                 lambda: ops.embedding(t, w.t()), lambda: ops.embedding(t.cpu(), w), lambda: ops.embedding(t, w, padding_idx=10),
                 lambda: ops.embedding_grad(torch.zeros(4, 4, device=DEV), t, 10), lambda: ops.embedding_grad(torch.zeros(3, 4, device=DEV), t, 0)):
        with pytest.raises(ValueError):
            call()
