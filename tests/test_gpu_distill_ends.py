"""tdm_k7_distill writes its rows and nothing else: bytes before the first row and behind the last stay as they were."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
GUARD = 1 << 18  # elements on either side: more than a workgroup's held vectors span

# rows, vocab, dtype: every form that holds a row in registers, by rows that fill little of it
FORMS = [(5, 601, torch.bfloat16), (1100, 2103, torch.bfloat16), (1100, 4201, torch.float16), (9, 2101, torch.float16), (1100, 9001, torch.bfloat16), (9, 9003, torch.bfloat16),
         (9, 17001, torch.float16), (9, 33001, torch.bfloat16), (9, 66003, torch.bfloat16), (9, 33001, torch.float32), (300, 260, torch.float32), (9, 140001, torch.bfloat16)]


@pytest.mark.parametrize("last", ["counts", "ignored"])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0])
@pytest.mark.parametrize("rows,vocab,dtype", FORMS)
def test_what_lies_beside_the_rows_stays(rows, vocab, dtype, temperature, last):
    from tandem_amd import _lib, ops

    gen = torch.Generator().manual_seed(3)
    around = torch.full((GUARD * 2 + rows * vocab,), float("nan"), dtype=dtype, device=DEV)
    x = around[GUARD:GUARD + rows * vocab].view(rows, vocab)
    x.copy_(torch.randn(rows, vocab, generator=gen) * 2)
    idx, t = torch.randint(0, vocab, (rows, 5), generator=gen).to(DEV), torch.randn(rows, 5, generator=gen).to(DEV)
    y = torch.randint(0, vocab, (rows,), generator=gen)
    if last == "ignored":
        y[-1] = -100
    y = y.to(DEV)
    want = ops.distill_loss_and_grad(x.clone(), idx, t, targets=y, temperature=temperature, weight=0.5)
    how = _lib.DISTILL_HOW.pack(rows, vocab, -100, 5, ops.CODES[dtype], 4, 0, 4, 1, temperature, 0.5, 1.0)
    L = _lib.lib()
    need = L.tdm_k7_distill_workspace(how)
    guard = torch.full((GUARD * 2 + rows * vocab,), 7.0, dtype=dtype, device=DEV)
    grad, work, loss = guard[GUARD:GUARD + rows * vocab], torch.empty(need, dtype=torch.uint8, device=DEV), torch.empty((), device=DEV)
    _lib.check(L.tdm_k7_distill(how, x.data_ptr(), idx.data_ptr(), t.data_ptr(), y.data_ptr(), loss.data_ptr(), grad.data_ptr(), None, 0, work.data_ptr(), need,
                                torch.cuda.current_stream().cuda_stream))
    assert (guard[:GUARD] == 7).all() and (guard[GUARD + rows * vocab:] == 7).all()
    assert torch.equal(loss, want[0]) and torch.equal(grad.view(rows, vocab), want[1]) and torch.isfinite(grad).all()
