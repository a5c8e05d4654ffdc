"""ops.qk_norm_rope / qkv_norm_rope and their gradients against the formulas in 64 bits.

Tolerances, u = 2^-24, D the head's size. The mean square adds D squares in fp32 (each rounded): relative error at most
(D + 2) u, half of that in its root; with the reciprocal root (2 u), the two products of the norm and the rotation's products and sum
(4 u) a rotated element (a c - b s) is off by at most (|a| + |b|) ((D/2 + 8) u + e), e = 2^-22 the error of a sine or cosine
(a quarter turn's rest rounded to fp32, then the library's sine: 2 u each, and the float's own step). A result is rounded
once more, half a step of its type. The gradients chain the same errors once more: with G = |ga| + |gb| the magnitude of a
rotated upstream pair, the terms w G and u mean(w G u) of dx are each off by at most K = (2 D + 16) u + 2 e of themselves, and
a sum over n heads adds n u of the sum of magnitudes."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U, E = 2.0 ** -24, 2.0 ** -22


def turn(x, c, s, interleaved, mag=False):
    """The pairs of x's first 2 * c.shape[-1] elements rotated; mag: the magnitudes that went in."""
    half = c.shape[-1]
    t = x[..., :2 * half]
    a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :half], t[..., half:])
    a, b = (a.abs() + b.abs(), a.abs() + b.abs()) if mag else (a * c - b * s, b * c + a * s)
    t = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    rest = x[..., 2 * half:]
    return torch.cat((t, rest.abs() if mag else rest), -1)


def reference(x, w, g, positions, inv_freq, eps, interleaved):
    """(y, its allowed error, dx, its allowed error, dw, its allowed error), before the rounding to the type, in 64 bits on the CPU."""
    x, g, d = x.detach().double().cpu(), g.detach().double().cpu(), x.shape[-1]
    w = torch.ones(d, dtype=torch.float64) if w is None else w.detach().double().cpu()
    angle = (positions.double().cpu().expand(x.shape[:-2])[..., None] * inv_freq.cpu())[..., None, :]
    c, s = angle.cos(), angle.sin()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r
    y = turn(u * w, c, s, interleaved)
    y_err = turn(u * w, c, s, interleaved, True) * ((d / 2 + 8) * U + E)
    k = (2 * d + 16) * U + 2 * E
    back, mag = turn(g, c, -s, interleaved), turn(g, c, s, interleaved, True)
    dx = r * (w * back - u * (w * back * u).mean(-1, keepdim=True))
    dx_err = r * k * (w.abs() * mag + u.abs() * (w.abs() * mag * u.abs()).mean(-1, keepdim=True))
    over = tuple(range(x.dim() - 1))
    n = x.numel() // max(d, 1)
    dw, dw_err = (back * u).sum(over), (n * U + k) * (mag * u.abs()).sum(over)
    return y, y_err, dx, dx_err, dw, dw_err


def near(got, want, err, what):
    assert got.shape == want.shape, what
    allowed = err + torch.finfo(got.dtype).eps / 2 * (want.abs() + err) * (1 + 2.0 ** -10)
    if got.dtype == torch.float16:
        allowed = allowed + 2.0 ** -25
    off = (got.detach().cpu().double() - want).abs()
    assert torch.isfinite(off).all(), what
    assert (off <= allowed).all(), f"{what}: off by {float((off - allowed).max()):.3g} more than allowed"


def inputs(batch, tokens, hq, hk, d, dtype, seed, packed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(DT[dtype]).to(DEV)  # noqa: E731
    lead = (batch, tokens) if batch else (tokens,)
    x = make(*lead, (hq + 2 * hk) * d) if packed else (make(*lead, hq, d), make(*lead, hk, d))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(DT[dtype]).to(DEV) for _ in range(2)]
    up = [make(*lead, h, d) for h in ((hq, hk, hk) if packed else (hq, hk))]
    return x, w, up


CASES = [  # batch (0: none), tokens, q heads, k heads, head, rotated, dtype, interleaved, first position, weights
    (2, 33, 12, 12, 64, 64, "bf16", False, 0, "same"),
    (0, 5, 32, 8, 128, 128, "bf16", False, 150_000, "same"),
    (1, 1, 1, 1, 2, 2, "fp32", False, 3, "same"),
    (3, 17, 10, 5, 80, 40, "fp32", True, 0, "same"),
    (1, 9, 3, 1, 6, 4, "fp16", False, 70, "fp32"),
    (2, 7, 4, 2, 130, 130, "fp32", False, 10, "none"),
    (2, 7, 4, 2, 130, 66, "bf16", True, 10, "fp32"),
    (1, 40, 2, 2, 256, 64, "fp16", False, 1_000_000, "same"),
    (1, 12, 2, 1, 512, 512, "bf16", False, 0, "same"),
    (1, 12, 2, 1, 512, 512, "fp32", True, 0, "same"),
    (1, 12, 1, 2, 510, 254, "fp32", False, 0, "same"),
    (2, 30, 4, 4, 96, 0, "bf16", False, 0, "same"),
    (1, 11, 8, 2, 72, 36, "bf16", False, 5, "same"),
    (1, 6000, 3, 1, 64, 32, "bf16", True, 0, "same"),
    (4, 2049, 2, 2, 32, 32, "fp32", False, 0, "same"),
]


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("batch,tokens,hq,hk,d,rotary,dtype,il,first,weights", CASES)
def test_forward_and_gradient(batch, tokens, hq, hk, d, rotary, dtype, il, first, weights, packed):
    from tandem_amd import ops

    x, w, up = inputs(batch, tokens, hq, hk, d, dtype, 1, packed)
    w = [None, None] if weights == "none" else [t.float() for t in w] if weights == "fp32" else w
    freq = ops.rope_frequencies(rotary) if rotary else torch.empty(0, dtype=torch.float64, device=DEV)
    pos = first + torch.arange(tokens, device=DEV)
    if batch:
        pos = pos + 1000 * torch.arange(batch, device=DEV)[:, None]
    how = dict(positions=pos, inv_freq=freq, eps=1e-5, interleaved=il)
    leaves = [t.requires_grad_() for t in ((x,) if packed else x)] + [t.requires_grad_() for t in w if t is not None]
    if packed:
        outs = ops.qkv_norm_rope(x, hq, hk, *w, **how)
        q, k, v = x.detach().unflatten(-1, (hq + 2 * hk, d)).split((hq, hk, hk), dim=-2)
        assert torch.equal(outs[2], v)
        direct = ops.qkv_norm_rope_grad(*up, x.detach(), hq, hk, *w, **how)
    else:
        outs = ops.qk_norm_rope(*x, *w, **how)
        q, k = x
        direct = ops.qk_norm_rope_grad(*up, *(t.detach() for t in x), *w, **how)
    grads = torch.autograd.grad(outs, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(grads, [t for t in direct if t is not None]))
    if packed:
        dq, dk, dv = grads[0].unflatten(-1, (hq + 2 * hk, d)).split((hq, hk, hk), dim=-2)
        assert torch.equal(dv, up[2])
    else:
        dq, dk = grads[:2]
    grads = (*grads, None, None) if weights == "none" else grads
    for name, xx, ww, gg, got, dgot, dwgot in (("q", q, w[0], up[0], outs[0], dq, grads[-2]), ("k", k, w[1], up[1], outs[1], dk, grads[-1])):
        y, y_err, dx, dx_err, dw, dw_err = reference(xx, ww, gg, pos, freq, 1e-5, il)
        near(got, y, y_err, name)
        near(dgot, dx, dx_err, "d" + name)
        if ww is not None:
            near(dwgot, dw, dw_err, f"d{name}_weight")


def test_views_of_any_strides_and_alignment():
    """q lies [batch, heads, tokens, dim], k starts one element off the 16-byte grid in wider rows; the upstream gradients are transposed and
    expanded."""
    from tandem_amd import ops

    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 6, 19, 64, generator=g).bfloat16().to(DEV).transpose(1, 2)
    k = torch.randn(2, 19, 3, 71, generator=g).bfloat16().to(DEV)[..., 1:65]
    w = [torch.randn(64, generator=g).bfloat16().to(DEV) for _ in range(2)]
    pos = torch.randint(0, 5000, (19, 2), generator=g, dtype=torch.int32).to(DEV).t()
    how = dict(positions=pos, inv_freq=ops.rope_frequencies(32), eps=1e-6)
    up = (torch.randn(2, 6, 19, 64, generator=g).bfloat16().to(DEV).transpose(1, 2), torch.full((), 0.25, device=DEV, dtype=torch.bfloat16).expand(2, 19, 3, 64))
    outs = ops.qk_norm_rope(q, k, *w, **how)
    grads = ops.qk_norm_rope_grad(*up, q, k, *w, **how)
    for i, x in enumerate((q, k)):
        y, y_err, dx, dx_err, dw, dw_err = reference(x, w[i], up[i], pos, how["inv_freq"], 1e-6, False)
        assert outs[i].is_contiguous()
        near(outs[i], y, y_err, "y")
        near(grads[i], dx, dx_err, "dx")
        near(grads[2 + i], dw, dw_err, "dw")


def test_missing_upstream_gradients_are_zeros():
    from tandem_amd import ops

    x, w, up = inputs(2, 9, 4, 2, 64, "fp32", 4, True)
    how = dict(positions=torch.arange(9, device=DEV), inv_freq=ops.rope_frequencies(64))
    x.requires_grad_()
    q, k, v = ops.qkv_norm_rope(x, 4, 2, *w, **how)
    (dx,) = torch.autograd.grad(k, x, up[1])
    zero = [torch.zeros_like(t) for t in up]
    want, *_ = ops.qkv_norm_rope_grad(zero[0], up[1], zero[2], x.detach(), 4, 2, *w, **how)
    assert torch.equal(dx, want) and (dx[..., 6 * 64:] == 0).all() and (dx[..., :4 * 64] == 0).all()
    none = ops.qkv_norm_rope_grad(None, None, None, x.detach(), 4, 2, *w, **how)
    assert all((t == 0).all() for t in none)


def test_no_tokens():
    from tandem_amd import ops

    x, w, up = inputs(2, 0, 4, 2, 64, "bf16", 4, True)
    how = dict(positions=torch.empty(0, device=DEV, dtype=torch.int64), inv_freq=ops.rope_frequencies(64))
    q, k, v = ops.qkv_norm_rope(x, 4, 2, *w, **how)
    assert q.shape == (2, 0, 4, 64) and v.shape == (2, 0, 2, 64)
    dx, dqw, dkw = ops.qkv_norm_rope_grad(*up, x, 4, 2, *w, **how)
    assert dx.shape == x.shape and (dqw == 0).all() and (dkw == 0).all()


def test_rows_of_zeros_and_non_finite_rows_stay_alone():
    from tandem_amd import ops

    x, w, _ = inputs(1, 6, 2, 2, 64, "fp32", 5, False)
    q, k = x
    q[0, 1, 0], q[0, 2, 1, 5], k[0, 3, 0, 7] = 0.0, float("nan"), float("inf")
    yq, yk = ops.qk_norm_rope(q, k, *w, torch.arange(6, device=DEV), ops.rope_frequencies(64))
    assert (yq[0, 1, 0] == 0).all() and torch.isnan(yq[0, 2, 1]).all()
    fine = torch.ones(1, 6, 2, dtype=torch.bool, device=DEV)
    fine[0, 2, 1] = False
    assert torch.isfinite(yq[fine]).all()
    fine[0, 2, 1], fine[0, 3, 0] = True, False
    assert torch.isfinite(yk[fine]).all() and not torch.isfinite(yk[0, 3, 0]).all()


def test_position_zero_is_the_norm_alone_and_distance_is_what_counts():
    """The product of a rotated query and key depends on the distance of their positions only: also far out, where an fp32 angle
    would be off by radians. Unit rows: each product is off by at most 64 * 2 ((32 + 8) u + e) < 64 * 2^-20."""
    from tandem_amd import ops

    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, 4, 1, 64, generator=g).to(DEV)
    freq = ops.rope_frequencies(64)
    at = lambda p: torch.tensor([p, p + 3, p + 10, p + 500], device=DEV)  # noqa: E731
    still, _ = ops.qk_norm_rope(x, x, None, None, torch.zeros(4, device=DEV, dtype=torch.int64), freq, eps=0.0)
    assert torch.allclose(still.cpu().double().square().mean(-1), torch.ones(1, 4, 1, dtype=torch.float64), atol=1e-5)
    dots = []
    for p in (0, 77, 1 << 20, (1 << 40) + 12345):
        q, _ = ops.qk_norm_rope(x, x, None, None, at(p), freq, eps=0.0)
        q = q.cpu().double()[0, :, 0]
        dots.append(q @ q.t())
    for d in dots[1:3]:
        assert (d - dots[0]).abs().max() < 64 * 2.0 ** -19
    assert (dots[3] - dots[0]).abs().max() < 64 * 2.0 ** -10  # 2^40 positions: a double's angle holds 2^-13 of a turn


def test_gradient_against_differences():
    """Central differences of sum(g y) in fp32 with step 2^-6 on elements of order 1: the third-order term is below 2^-12 |g| times a
    constant under 64 for 64 elements, the rounding of y (2^-20 relative, 128 terms) below 2^-7 after division by the step's 2^-5."""
    from tandem_amd import ops

    x, w, up = inputs(1, 2, 1, 1, 64, "fp32", 7, False)
    how = dict(positions=torch.tensor([[5, 900]], device=DEV), inv_freq=ops.rope_frequencies(64))
    dq, dk, dqw, dkw = (t.cpu().double() for t in ops.qk_norm_rope_grad(*up, *x, *w, **how))

    def loss(q, wq):
        y, _ = ops.qk_norm_rope(q, x[1], wq, w[1], **how)
        return float((y.cpu().double() * up[0].cpu().double()).sum())

    h = 2.0 ** -6
    for e in (0, 17, 40, 63):
        step = torch.zeros_like(x[0])
        step[0, 1, 0, e] = h
        assert abs((loss(x[0] + step, w[0]) - loss(x[0] - step, w[0])) / (2 * h) - float(dq[0, 1, 0, e])) < 0.02
        step = torch.zeros_like(w[0])
        step[e] = h
        assert abs((loss(x[0], w[0] + step) - loss(x[0], w[0] - step)) / (2 * h) - float(dqw[e])) < 0.02


def test_a_captured_graph_replayed():
    from tandem_amd import ops

    x, w, up = inputs(2, 300, 8, 4, 64, "bf16", 8, True)
    pos, freq = torch.zeros(2, 300, dtype=torch.int64, device=DEV), ops.rope_frequencies(64)

    def call():
        return (*ops.qkv_norm_rope(x, 8, 4, *w, pos, freq), *ops.qkv_norm_rope_grad(*up, x, 8, 4, *w, pos, freq))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for seed in (1, 2, 3):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=g))
        pos.copy_(torch.randint(0, 9999, pos.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, call()))


def test_refusals_on_the_gpu():
    from tandem_amd import ops

    x, w, up = inputs(1, 3, 4, 2, 64, "bf16", 9, True)
    pos, freq = torch.arange(3, device=DEV), ops.rope_frequencies(64)
    q, k = torch.zeros(1, 3, 4, 64, device=DEV), torch.zeros(1, 3, 2, 64, device=DEV)
    for call in (lambda: ops.qkv_norm_rope(x, 5, 2, *w, pos, freq), lambda: ops.qkv_norm_rope(x, 4, 2, w[0].double(), w[1], pos, freq),
                 lambda: ops.qkv_norm_rope(x, 4, 2, w[0].float(), w[1], pos, freq), lambda: ops.qkv_norm_rope(x, 4, 2, *w, pos.float(), freq),
                 lambda: ops.qkv_norm_rope(x, 4, 2, *w, pos[:2], freq), lambda: ops.qkv_norm_rope(x, 4, 2, *w, pos, freq.float()),
                 lambda: ops.qkv_norm_rope(x, 4, 2, *w, pos, ops.rope_frequencies(66)), lambda: ops.qkv_norm_rope(x, 4, 2, *w, pos.cpu(), freq),
                 lambda: ops.qk_norm_rope(q, k.bfloat16(), None, None, pos, freq), lambda: ops.qk_norm_rope(q, k[:, :2], None, None, pos, freq),
                 lambda: ops.qk_norm_rope(q.transpose(2, 3), k, None, None, pos, freq), lambda: ops.qk_norm_rope(q.double(), k.double(), None, None, pos, freq),
                 lambda: ops.qk_norm_rope(q[..., :63], k[..., :63], None, None, pos, freq[:31]),
                 lambda: ops.qkv_norm_rope_grad(up[0][..., :32], up[1], up[2], x, 4, 2, *w, pos, freq)):
        with pytest.raises(ValueError):
            call()
