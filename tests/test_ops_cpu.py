"""What the model operators refuse before they touch the GPU: through Python and through the C ABI."""

import ctypes

import pytest
import torch


def _lib():
    from tandem_amd import _lib

    return _lib


def refused(status, *words):
    message = _lib().lib().tdm_last_error().decode()
    assert status == 1 and all(w in message for w in words), (status, message)


def test_embedding_refuses_cpu_tensors():
    from tandem_amd import ops

    with pytest.raises(ValueError, match="no CPU path"):
        ops.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 4))
    with pytest.raises(ValueError, match="no CPU path"):
        ops.embedding_grad(torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64), 4)


def test_embedding_argument_errors_need_no_gpu():
    L = _lib().lib()
    p = ctypes.c_void_p(4096)  # never read: every call below is refused first
    f32, i64 = 0, 4
    refused(L.tdm_k5_embedding(p, p, i64, p, 1, 4, 4, 1, 1.0, None), "dtype")
    refused(L.tdm_k5_embedding(p, p, 0, p, 1, 4, 4, f32, 1.0, None), "int64")
    refused(L.tdm_k5_embedding(p, p, i64, p, -1, 4, 4, f32, 1.0, None), "tokens")
    refused(L.tdm_k5_embedding(p, p, i64, p, 1, 0, 4, f32, 1.0, None), "vocabulary")
    refused(L.tdm_k5_embedding(p, p, i64, p, 1, 4, 0, f32, 1.0, None), "rows of")
    refused(L.tdm_k5_embedding(p, None, i64, p, 1, 4, 4, f32, 1.0, None), "null")
    assert L.tdm_k5_embedding(None, None, i64, None, 0, 4, 4, f32, 1.0, None) == 0  # nothing to do
    assert L.tdm_k5_embedding_grad_workspace(-1, 4, 4) == -1 and L.tdm_k5_embedding_grad_workspace(1 << 29, 4, 4) == -1
    need = L.tdm_k5_embedding_grad_workspace(10_000, 4, 4)
    assert need >= 10_000 * 8
    grad = lambda *a: L.tdm_k5_embedding_grad(*a, None)  # noqa: E731
    refused(grad(p, p, i64, p, p, need - 1, 10_000, 4, 4, f32, 1.0, -1), "workspace")
    refused(grad(p, p, i64, p, ctypes.c_void_p(4100), need, 10_000, 4, 4, f32, 1.0, -1), "16 bytes")
    refused(grad(p, p, i64, None, p, need, 10_000, 4, 4, f32, 1.0, -1), "null")
    refused(grad(p, p, 7, p, p, need, 10_000, 4, 4, f32, 1.0, -1), "int64")
