"""The operators of the model that torch has no single pass for, as HIP kernels: the embedding lookup with a scale and its
gradient by sorted tokens; the norms of queries and keys per head with the position rotation in the same pass;
the distillation loss from a teacher's top logits with its gradient.

Functions on tensors in GPU memory, differentiable (in reverse mode, once), launched on the current stream of the tensors' device; float32,
float16 and bfloat16, sums in fp32, one rounding at the end. Each has its gradient beside it (`*_grad`) for programs that
run their backward pass by hand. Nothing here waits for the GPU, every result is the same bits every time, and all of it can be
captured into a graph. The reference has no counterpart: its model (tandem/model.py:14-120 there) is made of torch's own
operators.
"""

import struct

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from ._lib import DISTILL_HOW, DTYPES as CODES, HEADS, POSITIONS, QK_SHAPE, check, lib, require_device_tensor

DTYPES = (torch.float32, torch.float16, torch.bfloat16)
INDEX_DTYPES = (torch.int64, torch.int32)


def _on_gpu(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: needs a tensor in GPU memory (got {getattr(t, 'device', type(t))}); tandem_amd has no CPU path")


def _no_tangent(*tensors):
    """Refuses operands that carry a tangent of forward-mode differentiation: the kernels would drop it, and the result's derivative be zero.
    For where a level is open (forward_ad._current_level >= 0): no tensor has one otherwise."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("tandem_amd.ops has no derivatives in forward mode")


def _tensor(t, what):
    _on_gpu(t, what)
    if t.dtype not in DTYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16, not {t.dtype}")
    if forward_ad._current_level >= 0:
        _no_tangent(t)


def _floating(t, what):
    _on_gpu(t, what)
    if t.dtype not in DTYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16, not {t.dtype}")
    if forward_ad._current_level >= 0:
        _no_tangent(t)
    if not t.is_contiguous():
        raise ValueError(f"{what}: needs a contiguous tensor")


def _indices(t, what):
    """`t` as contiguous indices in GPU memory (slices of a batch are copied)."""
    _on_gpu(t, what)
    if t.dtype not in INDEX_DTYPES:
        raise ValueError(f"{what}: int64 or int32, not {t.dtype}")
    return t.contiguous()


def _same_device(first, *others):
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"tensors on {first.device} and {t.device}")


# A call's own queries of torch, bound once: they are most of what a small call costs the host.
_PRE_DISPATCH = torch._C.DispatchKey.PreDispatch
_compiling, _tracing, _modes, _has_key = (torch.compiler.is_dynamo_compiling, torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack,
                                          torch._C._dispatch_tls_is_dispatch_key_included)
_current_device, _current_stream = (getattr(torch._C, name, None) for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"))  # None: torch without a GPU


def _recorded():
    """Whether a trace is being made: a launch leaves nothing in it but the empty tensor that it fills. (torch.compile leaves its graph for
    a launch, and is no such trace.)"""
    return _tracing() is not None or get_proxy_mode() is not None


def _call(t, entry, *args):
    """entry(*args, stream) on the current stream of `t`'s device: the launch goes to the current device, which may be another."""
    # a mode of any kind shows on the stack or, before dispatch, as a key; asking which one takes longer, and there hardly ever is one
    if not _compiling() and (_tracing() is not None or _modes() or _has_key(_PRE_DISPATCH)) and _recorded():
        raise NotImplementedError("tandem_amd.ops can't be recorded by torch.jit.trace, make_fx or torch.export")
    device = t.get_device()
    if device == _current_device():
        status = entry(*args, _current_stream(device))
    else:
        with torch.cuda.device(device):
            status = entry(*args, _current_stream(device))
    if status:
        check(status)


def _ptr(t):
    """The address of an operand that may be missing. One whose storage has been given back (a sharded weight's between its uses) has the address
    zero, which says "missing" to the library; so has an empty one, which may be."""
    if t is None:
        return None
    at = t.data_ptr()
    if at == 0 and t.numel() > 0:
        raise ValueError(f"an operand of {list(t.shape)} has no memory")
    return at


def _workspace(bytes_needed, like):
    if bytes_needed < 0:
        raise ValueError(lib().tdm_last_error().decode(errors="replace"))
    return like.new_empty(bytes_needed, dtype=torch.uint8) if bytes_needed else None


def _once(backward):
    """torch's once_differentiable, which runs the backward pass without gradients and refuses a second one, where a second one was asked for
    (only then do gradients flow in a backward pass): its own bookkeeping costs more than most launches."""
    checked = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


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
    [0, vocab) comes out as a row of NaN, and takes no gradient.

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
    if tokens.get_device() != weight.get_device():
        _same_device(weight, tokens)
    vocab, dim = weight.shape
    out = weight.new_empty((*tokens.shape, dim))
    _call(weight, lib().tdm_k5_embedding, weight.data_ptr(), tokens.data_ptr(), CODES[tokens.dtype], out.data_ptr(), tokens.numel(), vocab, dim,
          CODES[weight.dtype], scale)
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
    need = lib().tdm_k5_embedding_grad_workspace(tokens.numel(), vocab, grad.shape[-1])
    return _embedding_backward(grad, tokens, vocab, grad.shape[-1], scale, padding, need)


def _embedding_backward(grad, tokens, vocab, dim, scale, padding, need):
    if forward_ad._current_level >= 0:
        _no_tangent(grad)
    out = grad.new_empty((vocab, dim))
    work = _workspace(need, grad)
    _call(grad, lib().tdm_k5_embedding_grad, grad.data_ptr(), tokens.data_ptr(), CODES[tokens.dtype], out.data_ptr(), _ptr(work), need,
          tokens.numel(), vocab, dim, CODES[grad.dtype], scale, padding)
    return out


# A backward pass runs on a thread of autograd's, where Python is slow to start: what the forward pass knows is kept for it, and what
# autograd sees to (an upstream gradient's shape, dtype and device) is not checked again.


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        tokens = _indices(tokens, "embedding(tokens)")
        ctx.save_for_backward(tokens)
        vocab, dim = weight.shape
        ctx.how = vocab, dim, scale, padding, lib().tdm_k5_embedding_grad_workspace(tokens.numel(), vocab, dim)
        return _embedding(tokens, weight, scale)

    @staticmethod
    @_once
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return None, _embedding_backward(grad if grad.is_contiguous() else grad.contiguous(), tokens, *ctx.how), None, None


# ---- norms of queries and keys, with the rotation


def rope_frequencies(rotary_dim, base=10000.0, device="cuda"):
    """The rotation's angles per position: base ** (-2 i / rotary_dim) for i < rotary_dim / 2, float64."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"an even number of rotated elements, not {rotary_dim}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cpu")
    return (base ** (-i / rotary_dim)).to(device)


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """Every head of q [batch, tokens, q_heads, dim] and k [batch, tokens, kv_heads, dim] (or both without batch) divided by the
    root of its mean square (+ eps), times its weight [dim] (None: ones), and rotated by its token's position: the pairs
    (a, b) of its first 2 * len(inv_freq) elements become (a cos - b sin, b cos + a sin) of position * inv_freq[i]. A pair is
    elements i and i + len(inv_freq); with `interleaved` 2i and 2i + 1. Returns (q, k) of the same shapes, contiguous.

    q and k may be views of any strides whose last dimension is contiguous; float32, float16 or bfloat16, the weights of the
    same dtype or float32. positions: int64 or int32, of a shape that expands to [batch, tokens]; inv_freq: float64
    (rope_frequencies), it takes no gradient. Angles are computed in float64, so far positions keep their precision. Single tokens are a
    batch of one token each."""
    x = _separate(q, k)
    how = _check_qk(x, q, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or _wants_grad(q_weight) or _wants_grad(k_weight)):
        return _QkNormRope.apply(q, k, q_weight, k_weight, x, how)
    return _qk_forward(q, q_weight, k_weight, x, how)


def qk_norm_rope_grad(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """The gradients (dq, dk, dq_weight, dk_weight) of qk_norm_rope for the upstream gradients dq_out, dk_out (None: zeros); a
    weight that is None has none. The weights' gradients are summed in fp32 over all tokens and heads in a fixed order."""
    x = _separate(q, k)
    how = _check_qk(x, q, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    _check_upstream(q, x, dq_out, dk_out)
    return _separate_backward(dq_out, dk_out, q, k, q_weight, k_weight, x, how, _qk_need(how))


def qkv_norm_rope(qkv, q_heads, kv_heads, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """qk_norm_rope on a packed projection: qkv [batch, tokens, (q_heads + 2 kv_heads) * dim] (or without batch) holds the
    queries' heads, the keys' and the values'. Returns (q, k, v): q and k as qk_norm_rope does, v a view of qkv. Its gradient
    is one pass that writes the gradient of qkv whole, the values' part included."""
    x = _packed(qkv, q_heads, kv_heads)
    how = _check_qk(x, qkv, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    if torch.is_grad_enabled() and (qkv.requires_grad or _wants_grad(q_weight) or _wants_grad(k_weight)):
        return _QkvNormRope.apply(qkv, q_weight, k_weight, x, how)
    return (*_qk_forward(qkv, q_weight, k_weight, x, how), _values(qkv, x))


def qkv_norm_rope_grad(dq_out, dk_out, dv_out, qkv, q_heads, kv_heads, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """The gradients (dqkv, dq_weight, dk_weight) of qkv_norm_rope for the upstream gradients dq_out, dk_out, dv_out (None: zeros)."""
    x = _packed(qkv, q_heads, kv_heads)
    how = _check_qk(x, qkv, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    _check_upstream(qkv, x, dq_out, dk_out, dv_out)
    return _packed_backward(dq_out, dk_out, dv_out, qkv, q_weight, k_weight, x, how, _qk_need(how))


class _Heads:
    """Where a call's heads lie: tokens ((batch, tokens) or (tokens,)), heads and their size, and q, k and, packed, v as tdm_heads."""

    __slots__ = ("tokens", "q_heads", "kv_heads", "dim", "q", "k", "v")

    def alike(self):
        """Heads of the same number and size, yet to be placed."""
        x = _Heads()
        x.tokens, x.q_heads, x.kv_heads, x.dim = self.tokens, self.q_heads, self.kv_heads, self.dim
        return x


def _packed(qkv, q_heads, kv_heads):
    _tensor(qkv, "qkv")
    *tokens, width = qkv.shape
    if len(tokens) not in (1, 2) or qkv.stride(-1) != 1:
        raise ValueError(f"qkv {list(qkv.shape)}: [batch, tokens, width] or [tokens, width], the last dimension contiguous")
    heads = q_heads + 2 * kv_heads
    if q_heads < 1 or kv_heads < 1 or width == 0 or width % heads:
        raise ValueError(f"qkv: a width of {width} for {q_heads} query heads and {kv_heads} key and value heads")
    x = _Heads()
    x.tokens, x.q_heads, x.kv_heads, x.dim = tokens, q_heads, kv_heads, width // heads
    _place_packed(x, qkv)
    return x


def _place_packed(x, qkv):
    strides = qkv.stride()
    lead = strides[:-1] if len(strides) == 3 else (0, strides[0])
    at, step = qkv.data_ptr(), x.dim * qkv.element_size()
    x.q = HEADS.pack(at, *lead, x.dim)
    x.k = HEADS.pack(at + x.q_heads * step, *lead, x.dim)
    x.v = HEADS.pack(at + (x.q_heads + x.kv_heads) * step, *lead, x.dim)


def _values(qkv, x):
    """The values' heads, a view."""
    return qkv.as_strided((*x.tokens, x.kv_heads, x.dim), (*qkv.stride()[:-1], x.dim, 1),
                          qkv.storage_offset() + (x.q_heads + x.kv_heads) * x.dim)


def _separate(q, k):
    _tensor(q, "q")
    _tensor(k, "k")
    *tokens, q_heads, dim = q.shape
    *k_tokens, kv_heads, k_dim = k.shape
    if q.dtype != k.dtype or tokens != k_tokens or dim != k_dim:
        raise ValueError(f"q {list(q.shape)} {q.dtype} and k {list(k.shape)} {k.dtype} differ in dtype, tokens or head size")
    if len(tokens) not in (1, 2) or 0 in (q_heads, kv_heads, dim) or q.stride(-1) != 1 or k.stride(-1) != 1:
        raise ValueError(f"q {list(q.shape)}, k {list(k.shape)}: [batch, tokens, heads, dim] or [tokens, heads, dim], the last dimension contiguous")
    _same_device(q, k)
    x = _Heads()
    x.tokens, x.q_heads, x.kv_heads, x.dim, x.q, x.k, x.v = tokens, q_heads, kv_heads, dim, _view(q), _view(k), None
    return x


def _view(t):
    """t [batch, tokens, heads, dim] or [tokens, heads, dim] as tdm_heads; None: no data."""
    if t is None:
        return HEADS.pack(0, 0, 0, 0)
    strides = t.stride()
    return HEADS.pack(_ptr(t), *strides[:-1]) if len(strides) == 4 else HEADS.pack(_ptr(t), 0, *strides[:-1])


def _wants_grad(w):
    return w is not None and w.requires_grad


class _QkHow:
    """What a call and its gradient share besides the tensors they differentiate."""

    __slots__ = ("shape", "positions", "inv_freq")

    def at(self):
        """The positions as tdm_positions."""
        strides = self.positions.stride()
        return POSITIONS.pack(self.positions.data_ptr(), *(strides if len(strides) == 2 else (0, strides[0])))

    def of(self, positions, inv_freq):
        """The same call on the tensors that the backward pass got back: hooks on saved tensors may have moved them."""
        how = _QkHow()
        how.shape, how.positions, how.inv_freq = self.shape, positions, inv_freq
        return how


def _check_qk(x, like, q_weight, k_weight, positions, inv_freq, eps, interleaved):
    dtype = weight_dtype = like.dtype
    for w in (q_weight, k_weight):
        if w is not None:
            _floating(w, "qk_norm_rope(weight)")
            weight_dtype = w.dtype
            if w.shape != (x.dim,) or weight_dtype not in (dtype, torch.float32):
                raise ValueError(f"a weight of {list(w.shape)} {w.dtype} for heads of {x.dim} {dtype}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight differ in dtype")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in INDEX_DTYPES:
        raise ValueError("positions: an int64 or int32 tensor")
    require_device_tensor(inv_freq, "qk_norm_rope(inv_freq)")
    if forward_ad._current_level >= 0:
        _no_tangent(inv_freq)
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise ValueError("inv_freq takes no gradient")
    rotary = 2 * inv_freq.numel()
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or rotary > x.dim:
        raise ValueError(f"inv_freq: at most {x.dim // 2} float64 values")
    _same_device(like, q_weight, k_weight, positions, inv_freq)
    tokens = x.tokens
    if list(positions.shape) != tokens:
        try:
            positions = positions.expand(tokens)
        except RuntimeError:
            raise ValueError(f"positions of {list(positions.shape)} for tokens of {tokens}") from None
    how = _QkHow()
    how.positions, how.inv_freq = positions, inv_freq
    try:
        how.shape = QK_SHAPE.pack(tokens[0] if len(tokens) == 2 else 1, tokens[-1], x.q_heads, x.kv_heads, x.dim, rotary, int(interleaved), CODES[dtype],
                                  CODES[weight_dtype], CODES[positions.dtype], eps)
    except struct.error as e:
        raise ValueError(f"qk_norm_rope: {e}") from None
    return how


def _qk_forward(like, q_weight, k_weight, x, how):
    q_out, k_out = like.new_empty((*x.tokens, x.q_heads, x.dim)), like.new_empty((*x.tokens, x.kv_heads, x.dim))
    _call(like, lib().tdm_k6_qk_norm_rope, how.shape, x.q, x.k, _ptr(q_weight), _ptr(k_weight), how.at(), how.inv_freq.data_ptr(), _view(q_out), _view(k_out))
    return q_out, k_out


def _check_upstream(like, x, dq_out, dk_out, dv_out=None):
    for g, heads, what in ((dq_out, x.q_heads, "dq_out"), (dk_out, x.kv_heads, "dk_out"), (dv_out, x.kv_heads, "dv_out")):
        if g is not None and (g.dtype != like.dtype or list(g.shape) != [*x.tokens, heads, x.dim] or g.get_device() != like.get_device()):
            raise ValueError(f"{what}: a gradient of {list(g.shape)} {g.dtype} on {g.device} for {[*x.tokens, heads, x.dim]} {like.dtype} on {like.device}")


def _rows(g):
    """An upstream gradient as the kernel reads it: of any strides, the last dimension contiguous."""
    return g if g is None or g.stride(-1) == 1 else g.contiguous()


def _qk_need(how):
    return lib().tdm_k6_qk_norm_rope_grad_workspace(how.shape)


def _qk_backward(dq_out, dk_out, dv_out, like, q_weight, k_weight, x, how, dx, need):
    if forward_ad._current_level >= 0:
        _no_tangent(dq_out, dk_out, dv_out)
    dq_out, dk_out, dv_out = _rows(dq_out), _rows(dk_out), _rows(dv_out)
    work = _workspace(need, like)
    dqw, dkw = None if q_weight is None else torch.empty_like(q_weight), None if k_weight is None else torch.empty_like(k_weight)
    _call(like, lib().tdm_k6_qk_norm_rope_grad, how.shape, _view(dq_out), _view(dk_out), _view(dv_out), x.q, x.k, _ptr(q_weight), _ptr(k_weight),
          how.at(), how.inv_freq.data_ptr(), dx.q, dx.k, dx.v, _ptr(dqw), _ptr(dkw), _ptr(work), need)
    return dqw, dkw


def _separate_backward(dq_out, dk_out, q, k, q_weight, k_weight, x, how, need):
    dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
    dx = _Heads()
    dx.q, dx.k, dx.v = _view(dq), _view(dk), None
    return (dq, dk, *_qk_backward(dq_out, dk_out, None, q, q_weight, k_weight, x, how, dx, need))


def _packed_backward(dq_out, dk_out, dv_out, qkv, q_weight, k_weight, x, how, need):
    dqkv = qkv.new_empty(qkv.shape)
    dx = x.alike()
    _place_packed(dx, dqkv)
    return (dqkv, *_qk_backward(dq_out, dk_out, dv_out, qkv, q_weight, k_weight, x, how, dx, need))


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, x, how):
        ctx.save_for_backward(q, k, q_weight, k_weight, how.positions, how.inv_freq)
        ctx.how, ctx.need = how.of(None, None), _qk_need(how)
        ctx.set_materialize_grads(False)
        return _qk_forward(q, q_weight, k_weight, x, how)

    @staticmethod
    @_once
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, positions, inv_freq = ctx.saved_tensors
        x = _Heads()  # placed anew: hooks on saved tensors may have moved them
        x.q, x.k = _view(q), _view(k)
        return (*_separate_backward(dq_out, dk_out, q, k, q_weight, k_weight, x, ctx.how.of(positions, inv_freq), ctx.need), None, None)


class _QkvNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, x, how):
        ctx.save_for_backward(qkv, q_weight, k_weight, how.positions, how.inv_freq)
        ctx.heads, ctx.how, ctx.need = x.alike(), how.of(None, None), _qk_need(how)
        ctx.set_materialize_grads(False)
        return (*_qk_forward(qkv, q_weight, k_weight, x, how), _values(qkv, x))

    @staticmethod
    @_once
    def backward(ctx, dq_out, dk_out, dv_out):
        qkv, q_weight, k_weight, positions, inv_freq = ctx.saved_tensors
        x = ctx.heads.alike()
        _place_packed(x, qkv)
        return (*_packed_backward(dq_out, dk_out, dv_out, qkv, q_weight, k_weight, x, ctx.how.of(positions, inv_freq), ctx.need), None, None)


# ---- distillation from a teacher's top logits

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def distill_loss(logits, teacher_index, teacher_logits, targets=None, temperature=1.0, weight=1.0, ignore_index=-100, reduction="mean"):
    """The loss of a student's logits [..., vocab] against a teacher's k top logits teacher_logits [..., k] at the columns
    teacher_index [..., k], mixed with the cross-entropy of hard targets [...]. For a row x, T the temperature, a the weight:

        p = softmax(teacher_logits / T)
        a T^2 sum_k p_k (log p_k - log softmax(x / T)[index_k]) + (1 - a) (-log softmax(x)[target])

    averaged ("mean") or added up ("sum") over the rows that count, or one value per row ("none"), in fp32. A row whose target is
    ignore_index does not count: its loss and gradient are zero, whatever its logits are; without any row that counts the mean is
    zero. Targets may be given with weight 1 to say which rows count. An entry with a negative column or a teacher's logit of
    -inf says nothing; a row without another takes no part in the first term; a column named twice has the sum of its
    entries. A column, or a target that is used, outside the vocabulary and a NaN among the teacher's logits show: the row's loss
    and gradient are NaN.

    logits contiguous, float32, float16 or bfloat16; the teacher's logits any of these, they take no gradient; k at most 1024. Where
    the gradient of float32 or bfloat16 logits is needed it is computed with the loss, from one reading of the logits, and kept until
    the backward pass hands it out; an upstream gradient other than one (a loss that is scaled or divided afterwards) makes the
    backward pass compute it again. Of float16 logits, whose loss is scaled as a rule, the backward pass computes it."""
    how, operands = _check_distill(logits, teacher_index, teacher_logits, targets, temperature, weight, ignore_index, reduction, 1.0)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Distill.apply(logits, *operands, how, reduction == "none")
    return _distill(logits, *operands, how, reduction == "none", True, None, None, False)


def distill_loss_and_grad(logits, teacher_index, teacher_logits, targets=None, temperature=1.0, weight=1.0, ignore_index=-100, reduction="mean",
                          scale=1.0):
    """(loss, gradient of scale * loss with respect to logits), for programs that run their backward pass by hand; the arguments are
    distill_loss's. `scale`: what the loss is multiplied with before the gradient is rounded to the logits' type (loss scaling);
    the loss that is returned is not scaled. With reduction "none" the gradient is that of the sum."""
    how, operands = _check_distill(logits, teacher_index, teacher_logits, targets, temperature, weight, ignore_index, reduction, scale)
    grad = _empty_at_phase_of(logits)
    return _distill(logits, *operands, how, reduction == "none", True, grad, None, False), grad


def _empty_at_phase_of(t):
    """An uninitialised contiguous tensor like `t` that starts at the same distance from a 16-byte boundary."""
    lead = t.data_ptr() % 16 // t.element_size()
    if lead == 0:
        return t.new_empty(t.shape)
    return t.new_empty(t.numel() + lead)[lead:].view(t.shape)


def _check_distill(logits, index, teacher, targets, temperature, weight, ignore_index, reduction, scale):
    _floating(logits, "distill_loss(logits)")
    _floating(teacher, "distill_loss(teacher_logits)")
    index = _indices(index, "distill_loss(teacher_index)")
    if logits.dim() < 1 or logits.shape[-1] == 0 or teacher.dim() < 1 or teacher.shape[-1] == 0:
        raise ValueError(f"logits {list(logits.shape)}, teacher_logits {list(teacher.shape)}: [..., vocab] and [..., k]")
    if teacher.shape[:-1] != logits.shape[:-1] or index.shape != teacher.shape:
        raise ValueError(f"logits {list(logits.shape)}, teacher_index {list(index.shape)}, teacher_logits {list(teacher.shape)}: rows differ")
    if reduction not in REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction}")
    if targets is not None:
        targets = _indices(targets, "distill_loss(targets)")
        if targets.shape != logits.shape[:-1]:
            raise ValueError(f"targets {list(targets.shape)} for logits {list(logits.shape)}")
    elif weight != 1.0:
        raise ValueError("a weight below 1 needs targets")
    _same_device(logits, index, teacher, targets)
    vocab = logits.shape[-1]
    try:
        how = DISTILL_HOW.pack(logits.numel() // vocab, vocab, ignore_index, teacher.shape[-1], CODES[logits.dtype], CODES[index.dtype],
                               CODES[teacher.dtype], CODES[torch.int64 if targets is None else targets.dtype], REDUCTIONS[reduction], temperature,
                               weight, scale)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"distill_loss: {e}") from None
    return how, (index, teacher, targets)


def _distill(logits, index, teacher, targets, how, each_row, want_loss, grad, upstream, keep_ones, need=None):
    L = lib()
    if need is None:
        need = L.tdm_k7_distill_workspace(how)
    work = _workspace(need, logits)
    loss = logits.new_empty(logits.shape[:-1] if each_row else (), dtype=torch.float32) if want_loss else None
    _call(logits, L.tdm_k7_distill, how, logits.data_ptr(), index.data_ptr(), teacher.data_ptr(), _ptr(targets), _ptr(loss), _ptr(grad),
          _ptr(upstream), int(keep_ones), _ptr(work), need)
    return loss


def _capture_of(t):
    """The number of the graph capture that `t`'s current stream is part of (0: none, negative: unknown)."""
    return lib().tdm_stream_capture_id(_current_stream(t.get_device()))


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, targets, how, each_row):
        ctx.save_for_backward(logits, index, teacher, targets)
        ctx.how, ctx.each_row, ctx.need = how, each_row, lib().tdm_k7_distill_workspace(how)
        # float16 is trained with a scaled loss: a gradient computed here would be for nothing
        ctx.grad, ctx.capture = (None, 0) if logits.dtype == torch.float16 else (_empty_at_phase_of(logits), _capture_of(logits))
        return _distill(logits, index, teacher, targets, how, each_row, True, ctx.grad, None, False, ctx.need)

    @staticmethod
    @_once
    def backward(ctx, upstream):
        if forward_ad._current_level >= 0:
            _no_tangent(upstream)
        # The gradient for an upstream of one is there: the kernel leaves the rows alone for which it is one. It is handed out once; a second
        # backward pass through the same graph computes its own. So does one whose logits hooks on saved tensors gave back at another distance from a
        # 16-byte boundary (the kernel takes both at one), and one that is captured apart from its forward pass: replayed without it, it would
        # hand out what the last replay's user made of the gradient.
        logits, *operands = ctx.saved_tensors
        grad, ctx.grad = ctx.grad, None
        first = grad is not None and (grad.data_ptr() - logits.data_ptr()) % 16 == 0 and 0 <= ctx.capture == _capture_of(logits)
        if not first:
            grad = _empty_at_phase_of(logits)
        _distill(logits, *operands, ctx.how, ctx.each_row, False, grad, upstream if upstream.is_contiguous() else upstream.contiguous(), first, ctx.need)
        return grad, None, None, None, None, None
