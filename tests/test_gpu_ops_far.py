"""The operators where offsets pass 32 bits, and through the C ABI as its header
allows: queries and keys in place, workspaces full of anything, results at any element's alignment."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def test_a_table_of_more_than_four_billion_bytes():
    from tandem_amd import ops

    vocab, dim = (1 << 21) + 5, 1200  # 2.5e9 elements, 5 GB
    w = torch.zeros(vocab, dim, device=DEV, dtype=torch.bfloat16)
    tokens = torch.tensor([0, vocab - 1, 1789569, 1789570, 1 << 20, vocab - 1], device=DEV)  # 1789569 * 1200 elements is 2^31 and a little less
    rows = torch.randn(6, dim, device=DEV, dtype=torch.bfloat16)
    w[tokens[1:]] = rows[1:]
    assert torch.equal(ops.embedding(tokens, w), w[tokens])
    assert w[tokens].abs().sum() > 0
    del w
    g = torch.randn(6, dim, device=DEV, dtype=torch.bfloat16)
    dw = ops.embedding_grad(g, tokens, vocab)
    assert torch.equal(dw[tokens[[0, 2, 3, 4]]], g[[0, 2, 3, 4]])
    assert torch.equal(dw[vocab - 1], (g[1].float() + g[5].float()).bfloat16())
    dw[tokens] = 0
    assert float(dw.abs().max()) == 0.0


def test_logits_of_more_than_four_billion_bytes():
    from tandem_amd import ops

    rows, vocab = 33000, 70001  # 2.3e9 elements; odd, so that the rows start anywhere
    x = torch.empty(rows, vocab, device=DEV, dtype=torch.bfloat16).normal_(generator=torch.Generator(DEV).manual_seed(1))
    idx = torch.randint(0, vocab, (rows, 8), device=DEV, generator=torch.Generator(DEV).manual_seed(2))
    t = torch.randn(rows, 8, device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    loss, grad = ops.distill_loss_and_grad(x, idx, t, reduction="none")
    for part in (slice(0, 3), slice(30676, 30680), slice(rows - 3, rows)):  # row 30677 holds element 2^31
        want = ops.distill_loss_and_grad(x[part].clone(), idx[part], t[part], reduction="none")
        assert torch.equal(loss[part], want[0]) and torch.equal(grad[part], want[1])


def test_heads_further_apart_than_32_bits():
    from tandem_amd import ops

    store = torch.zeros(3 * (1 << 31) + 4096, device=DEV, dtype=torch.bfloat16)  # 13 GB
    q = store.as_strided((2, 3, 2, 64), ((1 << 31) + 64, 256, 128, 1))
    k = store.as_strided((2, 3, 1, 64), ((1 << 31) + 64, 256, 64, 1), 1 << 31)
    gen = torch.Generator().manual_seed(4)
    q.copy_(torch.randn(2, 3, 2, 64, generator=gen))
    k.copy_(torch.randn(2, 3, 1, 64, generator=gen))
    how = dict(positions=torch.arange(3, device=DEV), inv_freq=ops.rope_frequencies(64))
    far, near = ops.qk_norm_rope(q, k, None, None, **how), ops.qk_norm_rope(q.contiguous(), k.contiguous(), None, None, **how)
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    up = [torch.randn(t.shape, generator=gen).bfloat16().to(DEV) for t in (q, k)]
    far, near = ops.qk_norm_rope_grad(*up, q, k, None, None, **how), ops.qk_norm_rope_grad(*up, q.contiguous(), k.contiguous(), None, None, **how)
    assert all(torch.equal(a, b) for a, b in zip(far[:2], near[:2]))


@pytest.mark.parametrize("interleaved", [0, 1])
def test_queries_and_keys_in_place(interleaved):
    from tandem_amd import _lib, ops

    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(2, 333, (6 + 2 * 3) * 96, generator=gen).bfloat16().to(DEV)
    w = [torch.randn(96, generator=gen).bfloat16().to(DEV) for _ in range(2)]
    pos, freq = torch.arange(333, device=DEV), ops.rope_frequencies(48)
    q, k, v = ops.qkv_norm_rope(qkv, 6, 3, *w, pos, freq, interleaved=bool(interleaved))
    lead = qkv.stride()[:2]
    heads = [_lib.HEADS.pack(qkv.data_ptr() + 2 * 96 * first, *lead, 96) for first in (0, 6)]
    shape = _lib.QK_SHAPE.pack(2, 333, 6, 3, 96, 48, interleaved, 3, 3, 4, 1e-6)
    at = _lib.POSITIONS.pack(pos.data_ptr(), 0, 1)
    _lib.check(_lib.lib().tdm_k6_qk_norm_rope(shape, *heads, w[0].data_ptr(), w[1].data_ptr(), at, freq.data_ptr(), *heads, stream()))
    got = qkv.unflatten(-1, (12, 96))
    assert torch.equal(got[:, :, :6], q) and torch.equal(got[:, :, 6:9], k) and torch.equal(got[:, :, 9:], v)


def test_workspaces_full_of_anything_and_results_at_any_alignment():
    from tandem_amd import _lib, ops

    L = _lib.lib()
    tokens = torch.randint(0, 700, (9000,), generator=torch.Generator().manual_seed(6)).to(DEV)
    for dim, lead in ((40, 0), (40, 3), (33, 1)):
        grad = torch.randn(9000, dim, device=DEV).half()
        want = ops.embedding_grad(grad, tokens, 700, scale=2.0)
        need = L.tdm_k5_embedding_grad_workspace(9000, 700, dim)
        for fill in (0xFF, 0x01):
            work = torch.full((need,), fill, dtype=torch.uint8, device=DEV)
            guard = torch.full((700 * dim + lead + 64,), 7.0, dtype=torch.float16, device=DEV)
            out = guard[lead:lead + 700 * dim]
            _lib.check(L.tdm_k5_embedding_grad(grad.data_ptr(), tokens.data_ptr(), 4, out.data_ptr(), work.data_ptr(), need, 9000, 700, dim, 2, 2.0, -1, stream()))
            assert torch.equal(out.view(700, dim), want)
            assert (guard[:lead] == 7).all() and (guard[lead + 700 * dim:] == 7).all()
    x, idx, t = torch.randn(20, 40000, device=DEV), torch.zeros(20, 3, dtype=torch.int64, device=DEV), torch.randn(20, 3, device=DEV)
    for fill in (0xFF, 0x01):
        how = _lib.DISTILL_HOW.pack(20, 40000, -100, 3, 0, 4, 0, 4, 1, 1.0, 1.0, 1.0)
        need = L.tdm_k7_distill_workspace(how)
        for grad in (None, torch.empty_like(x)):
            work = torch.full((need + 64,), fill, dtype=torch.uint8, device=DEV)
            loss = torch.empty((), device=DEV)
            _lib.check(L.tdm_k7_distill(how, x.data_ptr(), idx.data_ptr(), t.data_ptr(), None, loss.data_ptr(), None if grad is None else grad.data_ptr(), None, 0,
                                        work.data_ptr(), need, stream()))
            want = ops.distill_loss(x, idx, t) if grad is None else ops.distill_loss_and_grad(x, idx, t)
            assert torch.equal(loss, want if grad is None else want[0]) and (work[need:] == fill).all()
            assert grad is None or torch.equal(grad, want[1])


def test_the_gradient_of_the_norms_does_not_depend_on_what_its_workspace_holds():
    from tandem_amd import _lib, ops

    L = _lib.lib()
    gen = torch.Generator().manual_seed(7)
    q, k = (torch.randn(1, 50, h, 64, generator=gen).to(DEV) for h in (3, 1))
    up = [torch.randn(t.shape, generator=gen).to(DEV) for t in (q, k)]
    w = [torch.randn(64, generator=gen).to(DEV) for _ in range(2)]
    pos, freq = torch.arange(50, device=DEV), ops.rope_frequencies(64)
    want = ops.qk_norm_rope_grad(*up, q, k, *w, pos, freq)
    heads = lambda x: _lib.HEADS.pack(x.data_ptr(), *x.stride()[:3])  # noqa: E731
    shape, at = _lib.QK_SHAPE.pack(1, 50, 3, 1, 64, 64, 0, 0, 0, 4, 1e-6), _lib.POSITIONS.pack(pos.data_ptr(), 0, 1)
    need = L.tdm_k6_qk_norm_rope_grad_workspace(shape)
    work = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    dq, dk, dw = torch.empty_like(q), torch.empty_like(k), [torch.empty_like(x) for x in w]
    _lib.check(L.tdm_k6_qk_norm_rope_grad(shape, heads(up[0]), heads(up[1]), None, heads(q), heads(k), w[0].data_ptr(), w[1].data_ptr(), at, freq.data_ptr(),
                                          heads(dq), heads(dk), None, dw[0].data_ptr(), dw[1].data_ptr(), work.data_ptr(), need, stream()))
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, *dw), want)) and (work[need:] == 0xFF).all()
