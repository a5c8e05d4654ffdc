"""The operators together, as the GPT runs them: embedding with a scale, normed and rotated queries and keys, the distillation
loss, forward and backward, against the same model written out in 64 bits; then under DDP, ZeRO and FSDP, in a captured step, with
activations recomputed, and in bfloat16.

Tolerance of the fp32 model against 64 bits: some 30 roundings in a row from the tokens to the loss and as many back, each of sums of at
most 256 terms: 60 * 256 * 2^-24 of the norm, 1e-3, is what they could add up to; 2e-3 is asked of every gradient's 2-norm."""

import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DEV = "cuda"
TIMEOUT = 90.0


def config():
    from tandem_amd.model import Config

    return Config(vocab=259, seq=40, layers=2, heads=4, dim=64, rotary=True, embed_scale=8.0)


def batch(cfg, seed, rows=3, steps=37, k=7, device=DEV):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, cfg.vocab, (rows, steps), generator=g)
    targets = torch.randint(0, cfg.vocab, (rows, steps), generator=g)
    targets[0, 20:] = -100  # a padded row
    columns = torch.rand(rows, steps, cfg.vocab, generator=g).argsort(-1)[..., :k]
    logits = torch.randn(rows, steps, k, generator=g) * 2
    return [t.to(device) for t in (idx, targets, columns, logits)]


def loss_of(model, idx, targets, columns, logits):
    return model(idx, targets, teacher=(columns, logits), temperature=2.0, teacher_weight=0.7)


def written_out(cfg, p, idx, targets, columns, logits):
    """The model's loss from its parameters `p` (by name), in plain operations of p's dtype."""
    def norm(x, name):
        return F.layer_norm(x, (cfg.dim,), p[name + ".weight"], p[name + ".bias"])

    def linear(x, name):
        return x @ p[name + ".weight"].t() + p[name + ".bias"]

    per = cfg.dim // cfg.heads
    half = per // 2
    angle = torch.arange(idx.shape[1], dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, per, 2, dtype=torch.float64) / per)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x, w):
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    x = p["embed.tok.weight"][idx] * cfg.embed_scale
    rows, steps = idx.shape
    future = torch.ones(steps, steps, dtype=torch.bool).triu(1)
    for i in range(cfg.layers):
        at = f"blocks.{i}."
        q, k, v = (part.view(rows, steps, cfg.heads, per) for part in linear(norm(x, at + "ln1"), at + "attn.qkv").split(cfg.dim, -1))
        q, k = turn(q, p[at + "attn.q_norm"]), turn(k, p[at + "attn.k_norm"])
        scores = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(-1, -2) / math.sqrt(per)).masked_fill(future, -math.inf)
        x = x + linear((scores.softmax(-1) @ v.transpose(1, 2)).transpose(1, 2).reshape(rows, steps, cfg.dim), at + "attn.proj")
        x = x + linear(F.gelu(linear(norm(x, at + "ln2"), at + "fc")), at + "out")
    z = norm(x, "head.ln") @ p["head.lm.weight"].t()
    t = (logits.to(z.dtype) / 2.0).log_softmax(-1)
    soft = (t.exp() * (t - (z / 2.0).log_softmax(-1).gather(-1, columns))).sum(-1) * 4.0
    counted = targets != -100
    hard = -z.log_softmax(-1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    return ((0.7 * soft + 0.3 * hard) * counted).sum() / counted.sum()


def model_on_gpu(seed=0, dtype=torch.float32):
    from tandem_amd.model import GPT

    torch.manual_seed(seed)
    model = GPT(config())
    with torch.no_grad():  # weights of the norms that matter
        for name, p in model.named_parameters():
            if name.endswith("_norm"):
                p.add_(torch.randn(p.shape) * 0.1)
    return model.to(DEV, dtype)


def no_library_attention():
    torch.backends.cuda.enable_flash_sdp(False)
    torch.backends.cuda.enable_mem_efficient_sdp(False)


def test_loss_and_every_gradient_against_the_model_written_out():
    no_library_attention()
    model, cfg = model_on_gpu(), config()
    data = batch(cfg, 1)
    loss = loss_of(model, *data)
    loss.backward()
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in model.named_parameters()}
    assert "embed.pos.weight" not in p
    want = written_out(cfg, p, *(t.cpu() for t in data))
    grads = dict(zip(p, torch.autograd.grad(want, list(p.values()))))
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-3 * abs(float(want.detach()))
    for n, t in model.named_parameters():
        off = (t.grad.double().cpu() - grads[n]).norm()
        assert off <= 2e-3 * grads[n].norm() + 1e-9, (n, float(off), float(grads[n].norm()))


def test_a_first_call_in_inference_mode_leaves_training_as_it_is():
    no_library_attention()
    data = batch(config(), 4)
    model, fresh = model_on_gpu(), model_on_gpu()
    with torch.inference_mode():
        seen = loss_of(model, *data)
    loss = loss_of(model, *data)
    loss.backward()
    want = loss_of(fresh, *data)
    want.backward()
    assert float(seen) == float(loss.detach()) == float(want.detach())
    for (n, p), q in zip(model.named_parameters(), fresh.parameters()):
        assert torch.allclose(p.grad, q.grad, rtol=1e-5, atol=1e-7), n


def test_the_plain_model_learns_from_a_teacher_too():
    from tandem_amd import ops
    from tandem_amd.model import GPT, Config

    torch.manual_seed(0)
    model = GPT(Config(seq=32, layers=1, heads=2, dim=32)).to(DEV)
    idx, targets, columns, logits = batch(model.config, 2, steps=30)
    loss = model(idx, teacher=(columns, logits), temperature=2.0)
    assert torch.equal(loss, ops.distill_loss(model(idx), columns, logits, temperature=2.0))
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)


def test_bfloat16_follows_the_fp32_model():
    """bfloat16 keeps 8 bits: each of some 30 roundings in a row is off by 2^-9; 30 * 2^-9 of the loss."""
    model = model_on_gpu()
    data = batch(config(), 3)
    want = float(loss_of(model, *data))
    half = model.bfloat16()
    loss = loss_of(half, *data)
    loss.backward()
    assert loss.dtype == torch.float32 and abs(float(loss) - want) <= 30 * 2.0 ** -9 * abs(want)
    assert all(p.grad.dtype == torch.bfloat16 and torch.isfinite(p.grad).all() for p in half.parameters())


def test_recomputed_and_offloaded_activations_give_the_same_gradients():
    """What the operators save may come back as other tensors: recomputed (checkpointing) or from host memory."""
    from torch.utils.checkpoint import checkpoint

    no_library_attention()
    model, data = model_on_gpu(), batch(config(), 4)
    params = list(model.parameters())
    want = torch.autograd.grad(loss_of(model, *data), params)

    class Recomputed(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            return checkpoint(self.inner, x, use_reentrant=False)

    blocks = model.blocks
    model.blocks = torch.nn.ModuleList(Recomputed(b) for b in blocks)
    junk = []
    loss = loss_of(model, *data)
    junk.append(torch.randn(1 << 20, device=DEV))  # memory that forward has given back is used for something else
    got = torch.autograd.grad(loss, params)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    model.blocks = blocks
    with torch.autograd.graph.save_on_cpu():
        loss = loss_of(model, *data)
    junk.append(torch.randn(1 << 20, device=DEV))
    got = torch.autograd.grad(loss, params)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_training_step_replayed():
    no_library_attention()
    model, cfg = model_on_gpu(), config()
    data = batch(cfg, 5)
    params = list(model.parameters())

    def step():
        loss = loss_of(model, *data)
        return loss, torch.autograd.grad(loss, params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    for seed in (6, 7, 8):
        for old, new in zip(data, batch(cfg, seed)):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want_loss, want = step()
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss)
        for a, b in zip(grads, want):  # the matrix products may pick another kernel outside the graph
            assert (a - b).norm() <= 1e-4 * b.norm() + 1e-9


def train_rank(g, strategy, steps):
    from tandem_amd import ShardedAdamW
    from tandem_amd.ddp import DDP
    from tandem_amd.model import GPT
    from tandem_amd.zero import FSDP, ZeRO

    no_library_attention()
    torch.manual_seed(0)
    model = GPT(config()).to(g.device)
    if strategy == "ddp":
        z = DDP(model, g, bucket_bytes=1 << 16)
        opt = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.1, foreach=False, fused=False)
    else:
        sopt = ShardedAdamW(lr=3e-3, weight_decay=0.1, order="device")
        z = ZeRO(model, g, 2, sopt, 1 << 16) if strategy == "zero2" else FSDP(model, g, sopt)
    losses = []
    for step in range(steps):
        loss = loss_of(z, *batch(config(), 100 + 2 * step + g.rank, device=g.device))
        loss.backward()
        losses.append(loss.item())
        if strategy == "ddp":
            opt.step()
            opt.zero_grad()
        else:
            z.step()
            z.zero_grad()
    w = z.full_parameters() if strategy == "zero3" else torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    return losses, w.cpu()


def test_the_strategies_agree_on_the_rotary_model():
    """Two processes: the average is (a + b) / 2 in any order, so DDP, ZeRO-2 and FSDP agree bit for bit, and so do the ranks."""
    from tandem_amd import launch

    runs = {s: launch(train_rank, 2, s, 3, gpus=[0, 0], timeout=TIMEOUT) for s in ("ddp", "zero2", "zero3")}
    losses, weights = [r[0] for r in runs["ddp"]], runs["ddp"][0][1]
    assert all(math.isfinite(v) for rank in losses for v in rank)
    for ranks in runs.values():
        assert [r[0] for r in ranks] == losses
        assert all(torch.equal(r[1], weights) for r in ranks)


def test_a_second_derivative_is_refused():
    from tandem_amd import ops

    w = torch.randn(10, 16, device=DEV, requires_grad=True)
    x = torch.randn(4, 30, device=DEV, requires_grad=True)
    columns, logits = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.randn(4, 2, device=DEV)
    qkv = torch.randn(5, 48, device=DEV, requires_grad=True)
    q, _, _ = ops.qkv_norm_rope(qkv, 1, 1, None, None, torch.arange(5, device=DEV), ops.rope_frequencies(16))
    for out, leaf in ((ops.embedding(torch.arange(4, device=DEV), w), w), (ops.distill_loss(x, columns, logits), x), (q, qkv)):
        (first,) = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()
