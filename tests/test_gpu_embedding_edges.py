"""ops.embedding_grad where its sort has nothing to do, or takes another form: no tokens in tables beyond the one launch, tiles of 1024 tokens that
are just full or just begun, the most tokens that are split, the largest vocabulary."""

import pytest
import torch

from test_gpu_embedding import check_grad, exact_grad, make_tokens

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("lead", [0, 1, 4])
@pytest.mark.parametrize("vocab,dim,dtype", [(77, 48, torch.float32), (5000, 48, torch.float32), (5000, 33, torch.bfloat16), (70001, 512, torch.float32),
                                             (600001, 9, torch.float16)])
def test_no_tokens(vocab, dim, dtype, lead):
    """Every row is zeros, also where the sort's launch clears them all (up to 48 MiB), a part, or none (a result off the 16-byte grid)."""
    from tandem_amd import _lib, ops

    if lead == 0:
        got = ops.embedding_grad(torch.empty(0, dim, device=DEV, dtype=dtype), torch.empty(0, device=DEV, dtype=torch.int64), vocab)
        assert got.shape == (vocab, dim) and (got == 0).all()
    L = _lib.lib()
    need = L.tdm_k5_embedding_grad_workspace(0, vocab, dim)
    work = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device=DEV)
    guard = torch.full((64 + vocab * dim + 64,), 7.0, dtype=dtype, device=DEV)
    out = guard[64 + lead:64 + lead + vocab * dim - 64]
    rows = (vocab * dim - 64) // dim  # whole rows that fit between the guards at any lead
    need = L.tdm_k5_embedding_grad_workspace(0, rows, dim)
    _lib.check(L.tdm_k5_embedding_grad(None, None, 4, out.data_ptr(), work.data_ptr(), need, 0, rows, dim, ops.CODES[dtype], 1.0, -1,
                                       torch.cuda.current_stream().cuda_stream))
    assert (out[:rows * dim] == 0).all() and (guard[:64 + lead] == 7).all() and (guard[64 + lead + rows * dim:] == 7).all()


@pytest.mark.parametrize("vocab", [300, 40000])
@pytest.mark.parametrize("n", [8193, 9215, 9216, 9217, 16384, 16385, (1 << 20) - 1, 1 << 20, (1 << 20) + 1])
def test_tiles_that_are_just_full_or_just_begun(n, vocab):
    from tandem_amd import ops

    tokens = make_tokens("text", n, vocab, 21)
    grad = torch.stack([torch.ones(n), torch.arange(n) % 5.0 - 2.0], 1)
    got = ops.embedding_grad(grad.to(DEV), tokens.to(DEV), vocab)
    assert torch.equal(got.cpu().double(), exact_grad(grad, tokens, vocab, 1.0, None)[0])  # whole numbers below 2^24


@pytest.mark.parametrize("vocab", [(1 << 24) - 1, 1 << 24])
def test_the_largest_vocabulary(vocab):
    from tandem_amd import ops

    tokens = torch.cat([torch.tensor([0, vocab - 1, vocab - 1, vocab // 2, vocab, -1]), make_tokens("outside", 300, vocab, 22)])
    grad = torch.randn(len(tokens), 2, generator=torch.Generator().manual_seed(23))
    check_grad(ops.embedding_grad(grad.to(DEV), tokens.to(DEV), vocab, padding_idx=vocab // 2), grad, tokens, vocab, padding=vocab // 2)


def test_a_vocabulary_beyond_the_largest_is_refused():
    from tandem_amd import ops

    with pytest.raises(ValueError, match="2\\^24"):
        ops.embedding_grad(torch.zeros(1, 2, device=DEV), torch.zeros(1, device=DEV, dtype=torch.int64), (1 << 24) + 1)
