"""The operators of the model that torch has no single pass for, as HIP kernels: the embedding lookup with a scale and its
gradient by sorted tokens.

Functions on tensors in GPU memory, differentiable, launched on the current stream of the tensors' device; float32,
float16 and bfloat16, sums in fp32, one rounding at the end. Each has its gradient beside it (`*_grad`) for programs that
run their backward pass by hand. Nothing here waits for the GPU, every result is the same bits every time, and all of it can be
captured into a graph. The reference has no counterpart: its model (tandem/model.py:14-120 there) is made of torch's own
operators.
"""

import ctypes

import torch

from ._lib import check, dtype_code, lib, require_device_tensor, stream_ptr

DTYPES = (torch.float32, torch.float16, torch.bfloat16)
INDEX_DTYPES = (torch.int64, torch.int32)


def _floating(t, what):
    require_device_tensor(t, what)
    if t.dtype not in DTYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16, not {t.dtype}")


def _indices(t, what):
    """`t` as contiguous indices in GPU memory (slices of a batch are copied)."""
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{what}: needs a tensor in GPU memory (got {getattr(t, 'device', type(t))}); tandem_amd has no CPU path")
    if t.dtype not in INDEX_DTYPES:
        raise ValueError(f"{what}: int64 or int32, not {t.dtype}")
    return t.contiguous()


def _same_device(first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}")


def _call(device, entry, *args):
    """entry(*args, stream) on `device`'s current stream: the launch goes to the current device, which may be another."""
    if device.index == torch.cuda.current_device():
        check(entry(*args, stream_ptr(device)))
    else:
        with torch.cuda.device(device):
            check(entry(*args, stream_ptr(device)))


# ---- embedding


def _padding(padding_idx, vocab):
    if padding_idx is None:
        return -1
    if not -vocab <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} outside a vocabulary of {vocab}")
    return padding_idx % vocab


def embedding(tokens, weight, scale=1.0, padding_idx=None):
    """scale * weight[tokens]: tokens of any shape (int64 or int32), weight [vocab, dim] contiguous; the result has the tokens'
    shape and dim behind it, in weight's dtype. `padding_idx`: a token whose row takes no gradient. A token outside
    [0, vocab) reads nothing: its row comes out as NaN, and takes no gradient.

    The gradient of weight is dense and written in one pass over the upstream gradient, its rows added in the order of
    the tokens (see embedding_grad)."""
    padding = _check_embedding(tokens, weight, padding_idx)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(tokens, weight, float(scale), padding)
    return _embedding(tokens, weight, float(scale))


def _check_embedding(tokens, weight, padding_idx):
    _floating(weight, "embedding(weight)")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"embedding(weight): [vocab, dim], not {list(weight.shape)}")
    return _padding(padding_idx, weight.shape[0])


def _embedding(tokens, weight, scale):
    tokens = _indices(tokens, "embedding(tokens)")
    _same_device(weight, tokens)
    vocab, dim = weight.shape
    out = torch.empty(*tokens.shape, dim, device=weight.device, dtype=weight.dtype)
    _call(weight.device, lib().tdm_k5_embedding, weight.data_ptr(), tokens.data_ptr(), dtype_code(tokens.dtype), out.data_ptr(),
          tokens.numel(), vocab, dim, dtype_code(weight.dtype), scale)
    return out


def embedding_grad(grad, tokens, vocab, scale=1.0, padding_idx=None):
    """The gradient [vocab, dim] of embedding()'s weight for the upstream gradient `grad` (the tokens' shape and dim behind it):
    row v is scale times the sum of the rows of `grad` whose token is v, added in fp32 in the order of the tokens, and
    rounded once; zero for tokens that do not occur, and for `padding_idx`."""
    _floating(grad, "embedding_grad(grad)")
    vocab = int(vocab)
    if vocab < 1:
        raise ValueError(f"a vocabulary of {vocab}")
    return _embedding_grad(grad, tokens, vocab, float(scale), _padding(padding_idx, vocab))


def _embedding_grad(grad, tokens, vocab, scale, padding):
    tokens = _indices(tokens, "embedding_grad(tokens)")
    _same_device(grad, tokens)
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape or grad.shape[-1] == 0:
        raise ValueError(f"embedding_grad: a gradient of {list(grad.shape)} for tokens of {list(tokens.shape)}")
    n, dim = tokens.numel(), grad.shape[-1]
    out = torch.empty(vocab, dim, device=grad.device, dtype=grad.dtype)
    L = lib()
    need = L.tdm_k5_embedding_grad_workspace(n, vocab, dim)
    if need < 0:
        raise ValueError(L.tdm_last_error().decode(errors="replace"))
    work = torch.empty(need, device=grad.device, dtype=torch.uint8)
    _call(grad.device, L.tdm_k5_embedding_grad, grad.data_ptr(), tokens.data_ptr(), dtype_code(tokens.dtype), out.data_ptr(),
          work.data_ptr(), need, n, vocab, dim, dtype_code(grad.dtype), scale, padding)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        tokens = _indices(tokens, "embedding(tokens)")
        ctx.save_for_backward(tokens)
        ctx.how = weight.shape[0], scale, padding
        return _embedding(tokens, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return None, _embedding_grad(grad.contiguous(), tokens, *ctx.how), None, None
