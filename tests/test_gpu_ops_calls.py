"""Calls of the model operators that are allowed and easily forgotten: empty batches, operands that come back moved, graphs that hold half a step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("weight", [1.0, 0.5, 0.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_loss_of_no_rows_with_targets(dtype, weight, reduction):
    from tandem_amd import ops

    x, idx, t = torch.empty(0, 50, device=DEV, dtype=dtype), torch.empty(0, 4, device=DEV, dtype=torch.int64), torch.empty(0, 4, device=DEV)
    how = dict(targets=torch.empty(0, device=DEV, dtype=torch.int64), weight=weight, reduction=reduction, temperature=2.0)
    loss, grad = ops.distill_loss_and_grad(x, idx, t, **how)
    alone = ops.distill_loss(x, idx, t, **how)
    leaf = x.clone().requires_grad_()
    trained = ops.distill_loss(leaf, idx, t, **how)
    trained.sum().backward()
    for got in (loss, alone, trained):
        assert got.shape == ((0,) if reduction == "none" else ()) and (got == 0).all()
    assert grad.shape == leaf.grad.shape == (0, 50)


def distillation(rows, vocab, dtype, lead=0, seed=1):
    """Logits that begin `lead` elements behind an allocation's start, a teacher's columns and logits, targets."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.zeros(lead + rows * vocab, device=DEV, dtype=dtype)[lead:].view(rows, vocab)
    x.copy_(torch.randn(rows, vocab, generator=gen) * 2)
    columns, t = torch.randint(0, vocab, (rows, 4), generator=gen).to(DEV), torch.randn(rows, 4, generator=gen).to(DEV)
    return x, columns, t, torch.randint(0, vocab, (rows,), generator=gen).to(DEV)


@pytest.mark.parametrize("lead", [0, 1, 3])
@pytest.mark.parametrize("vocab", [251, 5003, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_offloaded_logits_that_began_anywhere(dtype, vocab, lead):
    """The copy that comes back begins on an allocation's boundary, the gradient that the forward pass left where the logits did."""
    from tandem_amd import ops

    x, columns, t, y = distillation(6, vocab, dtype, lead)
    for up in (1.0, 0.5):
        leaf = x.detach().requires_grad_()
        assert leaf.data_ptr() == x.data_ptr()
        with torch.autograd.graph.save_on_cpu():
            loss = ops.distill_loss(leaf, columns, t, y, temperature=2.0, weight=0.5)
        loss.backward(torch.tensor(up, device=DEV))
        # a gradient that both times comes from the copy is the same bits; one from rows that begin elsewhere has its sums in another order: off by
        # less than 2^-13 of a value each (4 R + V / 64 + 50 units of 2^-24, R < 16, V < 40002), and a step of the type where a rounding turns the other way
        want = ops.distill_loss_and_grad(x.clone(), columns, t, y, temperature=2.0, weight=0.5, scale=up)[1]
        if lead * x.element_size() % 16 == 0:
            assert torch.equal(leaf.grad, want)
        else:
            assert leaf.grad.shape == want.shape and (leaf.grad.float() - want.float()).abs().max() <= (torch.finfo(dtype).eps + 2.0 ** -12) * want.float().abs().max()


@pytest.mark.parametrize("forward_captured", [False, True])
@pytest.mark.parametrize("vocab,dtype", [(256, torch.float32), (20000, torch.bfloat16)])
def test_a_graph_that_holds_the_backward_pass_alone(vocab, dtype, forward_captured):
    """Replayed without the forward pass, which ran eagerly or is a graph of its own, after the gradient that the last replay gave was changed."""
    from tandem_amd import ops

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # everything on one stream, the leaf's first use too
        x, columns, t, y = distillation(70, vocab, dtype)
        leaf = x.clone().requires_grad_()
        loss_of = lambda: ops.distill_loss(leaf, columns, t, y, temperature=2.0, weight=0.5)  # noqa: E731
        want = torch.autograd.grad(loss_of(), leaf)[0]
        torch.cuda.synchronize()
        fore, back = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        if forward_captured:
            with torch.cuda.graph(fore, stream=s):
                loss = loss_of()
        else:
            loss = loss_of()
        with torch.cuda.graph(back, stream=s, **({"pool": fore.pool()} if forward_captured else {})):
            (grad,) = torch.autograd.grad(loss, leaf)
        if forward_captured:
            fore.replay()
        for _ in range(3):
            back.replay()
            torch.cuda.synchronize()
            assert torch.equal(grad, want)
            grad.mul_(3.0)
            torch.cuda.synchronize()


def test_a_captured_step_hands_out_its_own_forward_pass_s_gradient():
    """Within one capture the number is the same on both threads, and the gradient is computed once."""
    from tandem_amd import _lib, ops

    x, columns, t, y = distillation(70, 20000, torch.bfloat16)
    leaf, ids = x.clone().requires_grad_(), []
    number = lambda: ids.append(_lib.lib().tdm_stream_capture_id(torch.cuda.current_stream().cuda_stream))  # noqa: E731

    class Note(torch.autograd.Function):
        @staticmethod
        def forward(ctx, z):
            number()
            return z.view_as(z)

        @staticmethod
        def backward(ctx, g):
            number()
            return g

    def step():
        loss = ops.distill_loss(Note.apply(leaf), columns, t, y, temperature=2.0, weight=0.5)
        return loss.detach(), *torch.autograd.grad(loss, leaf)  # no graph of the leaf's outlives the step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    assert ids[:2] == [0, 0] and 0 < ids[2] == ids[3] and 0 < ids[4] == ids[5] != ids[2]
    for _ in range(2):
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            out[1].zero_()
            torch.cuda.synchronize()


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("batch,tokens,hq,hk,d,rotary,dtype", [(2, 5, 3, 1, 64, 64, torch.bfloat16), (3, 67, 5, 5, 80, 40, torch.float32), (1, 1, 9, 2, 128, 128, torch.float16),
                                                               (2, 1000, 12, 4, 2, 2, torch.bfloat16), (1, 300, 1, 1, 510, 10, torch.float16)])
def test_heads_that_lie_apart_leave_what_is_between_them(batch, tokens, hq, hk, d, rotary, dtype, interleaved):
    """Results written into the middle of larger heads, tokens and batches: everything around them stays, and they are those of the plain call."""
    from tandem_amd import _lib, ops

    gen = torch.Generator().manual_seed(9)
    q, k = (torch.randn(batch, tokens, h, d, generator=gen).to(dtype).to(DEV) for h in (hq, hk))
    up = [torch.randn(t.shape, generator=gen).to(dtype).to(DEV) for t in (q, k, k)]
    qw, kw = (torch.randn(d, generator=gen).to(DEV) for _ in range(2))
    pos, freq = torch.arange(tokens, device=DEV) + 7, ops.rope_frequencies(rotary)
    code = ops.CODES[dtype]
    shape, at = _lib.QK_SHAPE.pack(batch, tokens, hq, hk, d, rotary, interleaved, code, 0, 4, 1e-6), _lib.POSITIONS.pack(pos.data_ptr(), 0, 1)
    heads = lambda x: _lib.HEADS.pack(x.data_ptr(), *x.stride()[:3])  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    L = _lib.lib()

    def roomy(t):
        around = torch.full((t.shape[0] + 1, t.shape[1] + 2, t.shape[2] + 1, d + 6), 7.0, dtype=dtype, device=DEV)
        return around, around[:t.shape[0], 1:-1, :t.shape[2], 2:2 + d]

    def untouched(around, inside):
        inside.fill_(7.0)
        return bool((around == 7.0).all())

    (qa, qo), (ka, ko) = roomy(q), roomy(k)
    _lib.check(L.tdm_k6_qk_norm_rope(shape, heads(q), heads(k), qw.data_ptr(), kw.data_ptr(), at, freq.data_ptr(), heads(qo), heads(ko), stream))
    want = ops.qk_norm_rope(q, k, qw, kw, pos, freq, interleaved=bool(interleaved))
    # another width of access, so other lanes hold a head: its sum has another order, off by up to d 2^-24 of it, and a rounding may turn the other way
    near = lambda a, b: torch.isfinite(a).all() and ((a.float() - b.float()).abs() <= (torch.finfo(dtype).eps + 2.0 ** -13) * b.float().abs().amax(-1, True)).all()  # noqa: E731
    assert near(qo, want[0]) and near(ko, want[1])
    assert untouched(qa, qo) and untouched(ka, ko)
    (dqa, dq), (dka, dk), (dva, dv) = roomy(q), roomy(k), roomy(k)
    need = L.tdm_k6_qk_norm_rope_grad_workspace(shape)
    work = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    dw = torch.full((2, d + 2), 7.0, device=DEV)
    _lib.check(L.tdm_k6_qk_norm_rope_grad(shape, heads(up[0]), heads(up[1]), heads(up[2]), heads(q), heads(k), qw.data_ptr(), kw.data_ptr(), at, freq.data_ptr(),
                                          heads(dq), heads(dk), heads(dv), dw[0, 1:].data_ptr(), dw[1, 1:].data_ptr(), work.data_ptr(), need, stream))
    want = ops.qk_norm_rope_grad(up[0], up[1], q, k, qw, kw, pos, freq, interleaved=bool(interleaved))
    assert near(dq, want[0]) and near(dk, want[1]) and torch.equal(dv, up[2])
    for got, ref, x, g in zip(dw[:, 1:-1], want[2:], (q, k), up):
        # N terms in two orders, each of at most sqrt(2) times its row's largest upstream value times the normed element; no term passes N additions
        x, terms = x.double(), x[..., 0].numel()
        most = (2 ** 0.5 * g.double().abs().amax(-1, True) * (x * x.square().mean(-1, True).rsqrt()).abs()).sum((0, 1, 2))
        assert ((got - ref).abs() <= 2 * (terms + 16) * 2.0 ** -24 * most).all()
    assert (dw[:, 0] == 7).all() and (dw[:, -1] == 7).all() and (work[need:] == 0xFF).all()
    assert untouched(dqa, dq) and untouched(dka, dk) and untouched(dva, dv)


@pytest.mark.parametrize("vocab,dim,n,dtype,lead", [(50, 999, 37, torch.float16, 1), (50, 64, 1, torch.bfloat16, 0), (7, 3, 1030, torch.float32, 3), (9, 2050, 5, torch.bfloat16, 2)])
def test_a_lookup_writes_its_rows_and_nothing_else(vocab, dim, n, dtype, lead):
    from tandem_amd import _lib, ops

    gen = torch.Generator().manual_seed(10)
    w, tokens = torch.randn(vocab, dim, generator=gen).to(dtype).to(DEV), torch.randint(0, vocab, (n,), generator=gen).to(DEV)
    around = torch.full((64 + lead + n * dim + 64,), 7.0, dtype=dtype, device=DEV)
    out = around[64 + lead:64 + lead + n * dim]
    _lib.check(_lib.lib().tdm_k5_embedding(w.data_ptr(), tokens.data_ptr(), 4, out.data_ptr(), n, vocab, dim, ops.CODES[dtype], 1.0, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out.view(n, dim), w[tokens])
    assert (around[:64 + lead] == 7).all() and (around[64 + lead + n * dim:] == 7).all()


def test_a_compiled_program_calls_the_operators():
    """torch.compile leaves its graph for every launch: same losses and gradients, twice, and with other inputs."""
    from tandem_amd import ops

    gen = torch.Generator().manual_seed(11)
    table, proj, qw, kw = (torch.randn(*s, generator=gen).mul_(0.1).to(DEV).requires_grad_() for s in ((50, 32), (64, 32), (16,), (16,)))
    freq, pos = ops.rope_frequencies(16), torch.arange(6, device=DEV)

    def program(tokens, columns, teacher):
        x = ops.embedding(tokens, table, scale=2.0)
        q, k, v = ops.qkv_norm_rope(x @ proj.t(), 2, 1, qw, kw, pos, freq)
        logits = torch.cat((q.flatten(2), k.flatten(2), v.flatten(2)), -1) * 3
        return ops.distill_loss(logits, columns, teacher, temperature=2.0) / 2

    compiled = torch.compile(program, backend="eager")
    for seed in (1, 2, 3):
        gen.manual_seed(seed)
        inputs = torch.randint(0, 50, (2, 6), generator=gen).to(DEV), torch.randint(0, 64, (2, 6, 3), generator=gen).to(DEV), torch.randn(2, 6, 3, generator=gen).to(DEV)
        leaves = (table, proj, qw, kw)
        want_loss = program(*inputs)
        want = torch.autograd.grad(want_loss, leaves)
        loss = compiled(*inputs)
        assert torch.equal(loss, want_loss) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))


def test_what_is_refused_on_the_gpu_too():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    from tandem_amd import ops

    w, tokens = torch.randn(9, 4, device=DEV), torch.tensor([1, 2], device=DEV)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        ops.embedding(tokens, forward_ad.make_dual(w, torch.ones_like(w)))
    for record in (lambda: torch.jit.trace(lambda w: ops.embedding(tokens, w), (w,)), lambda: make_fx(lambda w: ops.embedding(tokens, w))(w)):
        with pytest.raises(NotImplementedError, match="recorded"):
            record()
    with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
        torch.func.jvp(lambda w: ops.embedding(tokens, w), (w,), (torch.ones_like(w),))
    leaf = w.clone().requires_grad_()
    out = ops.embedding(tokens, leaf)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
    assert torch.equal(ops.embedding(tokens, w), w[tokens])
