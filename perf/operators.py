"""The language-model operators of tandem_amd.ops at the sizes they are used at: the embedding with its
gradient, the norms of queries and keys with the rotation, the distillation loss with its gradient.

`own` false: each operator in plain torch operations, in 32 bits (angles in 64), rounded once at the end.
`own` true: the calls that a training or serving program makes.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
INDEX = {"int64": torch.int64, "int32": torch.int32}
IGNORE = -100
EPS = 1e-6


def listed():
    return [
        # the medium preset's token gradient: bytes, so every row of the table is hit many times
        dict(name="embed bytes grad", op="embedding", **{"pass": "grad"}, dtype="fp32", index="int64", vocab=256, dim=768, batch=16, seq=512,
             scale=1.0, padding=-1),
        # answering: one new token for each of eight sequences
        dict(name="embed one token", op="embedding", **{"pass": "forward"}, dtype="bf16", index="int32", vocab=32000, dim=4096, batch=8, seq=1,
             scale=64.0, padding=-1),
        # pretraining with a large vocabulary: the dense gradient is mostly rows that no token names
        dict(name="embed large train", op="embedding", **{"pass": "train"}, dtype="bf16", index="int64", vocab=131072, dim=2048, batch=8, seq=4096,
             scale=45.25, padding=-1),
        # fine-tuning on ragged text: rows of 999 halves start anywhere, padding takes no gradient
        dict(name="embed odd grad", op="embedding", **{"pass": "grad"}, dtype="fp16", index="int32", vocab=50021, dim=999, batch=1, seq=4099,
             scale=1.0, padding=7),
        # the medium preset's attention, packed as its qkv projection writes it, forward and backward
        dict(name="qk medium train", op="qk_norm_rope", **{"pass": "train"}, form="packed", dtype="bf16", batch=16, seq=512, q_heads=12,
             kv_heads=12, head_dim=64, rotary=64, interleaved=False, last=0),
        # answering: one new token for each of sixteen sequences, far into their contexts
        dict(name="qk one token", op="qk_norm_rope", **{"pass": "forward"}, form="packed", dtype="bf16", batch=16, seq=1, q_heads=32,
             kv_heads=8, head_dim=128, rotary=128, interleaved=False, last=100000),
        # one long sequence with shared key heads
        dict(name="qk long train", op="qk_norm_rope", **{"pass": "train"}, form="packed", dtype="bf16", batch=1, seq=32768, q_heads=32,
             kv_heads=8, head_dim=128, rotary=128, interleaved=False, last=0),
        # queries and keys from projections of their own, half of each head rotated in neighbouring pairs
        dict(name="qk odd grad", op="qk_norm_rope", **{"pass": "grad"}, form="separate", dtype="fp32", batch=3, seq=1021, q_heads=10,
             kv_heads=5, head_dim=80, rotary=40, interleaved=True, last=0),
        # the medium preset's loss: bytes, mixed with the hard targets
        dict(name="distill bytes grads", op="distill", **{"pass": "grads"}, dtype="fp32", rows=8192, vocab=256, k=16, temperature=2.0, weight=0.5,
             ignored=0.0, scale=1.0),
        # the loss alone on the last tokens of a few sequences (evaluation)
        dict(name="distill few rows", op="distill", **{"pass": "loss"}, dtype="bf16", rows=4, vocab=131072, k=64, temperature=1.0, weight=1.0,
             ignored=0.0, scale=1.0),
        # the largest training step: a large vocabulary, the teacher's top 64, no hard targets
        dict(name="distill large train", op="distill", **{"pass": "train"}, dtype="bf16", rows=8192, vocab=131072, k=64, temperature=1.0,
             weight=1.0, ignored=0.0, scale=1.0),
        # a padded batch in halves, its loss scaled: rows without a target, an odd vocabulary, two temperatures at once
        dict(name="distill odd grads", op="distill", **{"pass": "grads"}, dtype="fp16", rows=1031, vocab=50021, k=33, temperature=1.5, weight=0.7,
             ignored=0.2, scale=4096.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embedding", "qk_norm_rope", "distill"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "embedding":
        what = rng.choice(["forward", "grad", "train"])
        vocab, dim = _log(rng, 200, 131072), _log(rng, 64, 4096)
        dim = dim if rng.random() < 0.3 else max(64, dim // 64 * 64)
        vocab = min(vocab, (1 << 28) // dim)
        batch = _log(rng, 1, 16)
        seq = max(1, min(_log(rng, 1, 8192), (1 << 26) // (dim * batch)))
        return dict(op=op, **{"pass": what}, dtype=dtype, index=rng.choice(["int64", "int32"]), vocab=vocab, dim=dim, batch=batch, seq=seq,
                    scale=rng.choice([1.0, round(math.sqrt(dim), 2)]), padding=rng.choice([-1, 0, 7]))
    if op == "qk_norm_rope":
        what, form = rng.choice(["forward", "grad", "train"]), rng.choice(["packed", "packed", "separate"])
        head_dim = rng.choice([32, 64, 80, 96, 128, 128, 160, 256])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
        q_heads = kv_heads * rng.choice([1, 1, 2, 4])
        batch = _log(rng, 1, 64)
        seq = max(1, min(_log(rng, 1, 32768), (1 << 27) // (batch * (q_heads + 2 * kv_heads) * head_dim)))
        return dict(op=op, **{"pass": what}, form=form, dtype=dtype, batch=batch, seq=seq, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2]), interleaved=rng.random() < 0.3, last=rng.choice([0, 4000, 200000]))
    vocab = _log(rng, 200, 131072)
    rows = max(1, min(_log(rng, 1, 16384), (1 << 29) // vocab))
    return dict(op=op, **{"pass": rng.choice(["loss", "grads", "train"])}, dtype=dtype, rows=rows, vocab=vocab, k=_log(rng, 1, 128),
                temperature=rng.choice([1.0, 1.5, 2.0]), weight=rng.choice([1.0, 0.5, 0.9]), ignored=rng.choice([0.0, 0.0, 0.3]),
                scale=4096.0 if dtype == "fp16" else 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype, std=1.0):
        return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=gen)

    def uniform(*shape, dtype=torch.float32):
        return torch.rand(*shape, device="cuda", dtype=dtype, generator=gen)

    s = {"case": case}
    if case["op"] == "embedding":
        vocab, dim, shape = case["vocab"], case["dim"], (case["batch"], case["seq"])
        # how often a token occurs falls with one over its rank, as in text; the ranks are strewn over the table
        rank = (torch.pow(float(vocab), uniform(*shape, dtype=torch.float64)) - 1).long().clamp_(0, vocab - 1)
        step = next(p for p in (7919, 104729, 1299709) if vocab % p)
        s["tokens"] = (rank * step % vocab).to(INDEX[case["index"]])
        s["padding"] = None if case["padding"] < 0 else case["padding"]
        s["weight"] = normal(vocab, dim, std=0.02).requires_grad_(case["pass"] == "train")
        if case["pass"] != "forward":
            s["grad"] = normal(*shape, dim, std=1e-2)
    elif case["op"] == "qk_norm_rope":
        b, t, hq, hk, d = (case[n] for n in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
        train = case["pass"] == "train"
        if case["form"] == "packed":
            s["qkv"] = normal(b, t, (hq + 2 * hk) * d).requires_grad_(train)
        else:
            s["q"], s["k"] = normal(b, t, hq, d).requires_grad_(train), normal(b, t, hk, d).requires_grad_(train)
        s["q_weight"] = (1 + normal(d, dtype=torch.float32, std=0.1)).to(dtype).requires_grad_(train)
        s["k_weight"] = (1 + normal(d, dtype=torch.float32, std=0.1)).to(dtype).requires_grad_(train)
        first = torch.randint(0, case["last"] + 1, (b, 1), device="cuda", generator=gen)
        s["positions"] = first + torch.arange(t, device="cuda")
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
        if case["pass"] != "forward":
            s["dq"], s["dk"] = normal(b, t, hq, d, std=1e-2), normal(b, t, hk, d, std=1e-2)
            if case["form"] == "packed":
                s["dv"] = normal(b, t, hk, d, std=1e-2)
    else:
        rows, vocab, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
        first = torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen)
        s["index"] = (first + torch.arange(k, device="cuda") * (vocab // k)) % vocab
        s["teacher"] = normal(rows, k, dtype=torch.float32, std=2.0).sort(dim=1, descending=True).values
        logits = normal(rows, vocab, std=2.0)
        logits.scatter_add_(1, s["index"], (s["teacher"] + 5.0).to(dtype))  # a student that has learnt something
        s["logits"] = logits.requires_grad_(case["pass"] == "train")
        s["upstream"] = torch.tensor(case["scale"], device="cuda")
        s["targets"] = None
        if case["weight"] < 1.0 or case["ignored"] > 0.0:
            best = uniform(rows) < 0.7
            s["targets"] = torch.where(best, s["index"][:, 0], torch.randint(0, vocab, (rows,), device="cuda", generator=gen))
            s["targets"][uniform(rows) < case["ignored"]] = IGNORE
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------


def _plain_embedding(s):
    case, tokens, weight = s["case"], s["tokens"].long(), s["weight"].detach()
    out = dw = None
    if case["pass"] != "grad":
        out = (weight[tokens].float() * case["scale"]).to(weight.dtype)
    if case["pass"] != "forward":
        acc = torch.zeros(case["vocab"], case["dim"], device="cuda", dtype=torch.float32)
        acc.index_add_(0, tokens.reshape(-1), s["grad"].reshape(-1, case["dim"]).float())
        if s["padding"] is not None:
            acc[s["padding"]] = 0.0
        dw = (acc * case["scale"]).to(weight.dtype)
    return [x for x in (out, dw) if x is not None]


def _halves(x, rotary, interleaved):
    turned = x[..., :rotary]
    if interleaved:
        return turned[..., 0::2], turned[..., 1::2]
    return turned[..., : rotary // 2], turned[..., rotary // 2:]


def _rotate(x, cos, sin, rotary, interleaved):
    a, b = _halves(x, rotary, interleaved)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, x[..., rotary:]), dim=-1)


def _plain_norm_rope(x, weight, cos, sin, case):
    x32 = x.float()
    r = 1.0 / torch.sqrt((x32 * x32).mean(dim=-1, keepdim=True) + EPS)
    return _rotate(x32 * r * weight.float(), cos, sin, case["rotary"], case["interleaved"]).to(x.dtype)


def _plain_norm_rope_grad(g, x, weight, cos, sin, case):
    x32, w32 = x.float(), weight.float()
    r = 1.0 / torch.sqrt((x32 * x32).mean(dim=-1, keepdim=True) + EPS)
    unit = x32 * r
    g32 = _rotate(g.float(), cos, -sin, case["rotary"], case["interleaved"])
    dw = (g32 * unit).sum(dim=(0, 1, 2)).to(weight.dtype)
    gw = g32 * w32
    return (r * (gw - unit * (gw * unit).mean(dim=-1, keepdim=True))).to(x.dtype), dw


def _plain_qk(s):
    case = s["case"]
    b, t, hq, hk, d = (case[n] for n in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
    if case["form"] == "packed":
        q, k, v = (x.view(b, t, -1, d) for x in s["qkv"].detach().split((hq * d, hk * d, hk * d), dim=-1))
    else:
        q, k, v = s["q"].detach(), s["k"].detach(), None
    qw, kw = s["q_weight"].detach(), s["k_weight"].detach()
    angle = s["positions"].double()[..., None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    if case["pass"] != "grad":
        out["q"], out["k"] = _plain_norm_rope(q, qw, cos, sin, case), _plain_norm_rope(k, kw, cos, sin, case)
        if v is not None:
            out["v"] = v
    if case["pass"] != "forward":
        gq, out["dq_weight"] = _plain_norm_rope_grad(s["dq"], q, qw, cos, sin, case)
        gk, out["dk_weight"] = _plain_norm_rope_grad(s["dk"], k, kw, cos, sin, case)
        if v is not None:
            out["dqkv"] = torch.cat((gq.flatten(2), gk.flatten(2), s["dv"].flatten(2)), dim=-1)
        else:
            out["dq"], out["dk"] = gq, gk
    return out


def _plain_distill(s):
    case, x = s["case"], s["logits"].detach()
    tau, weight, y = case["temperature"], case["weight"], s["targets"]
    x32 = x.float()
    x32 = x32 - x32.amax(dim=1, keepdim=True)
    e = torch.exp(x32 / tau)
    z = e.sum(dim=1, keepdim=True)
    t = s["teacher"].float() / tau
    t = t - t.amax(dim=1, keepdim=True)
    p = torch.exp(t)
    zt = p.sum(dim=1, keepdim=True)
    p = p / zt
    log_p, log_q = t - torch.log(zt), x32.gather(1, s["index"]) / tau - torch.log(z)
    row = weight * tau * tau * (p * (log_p - log_q)).sum(dim=1)
    counted = None
    if y is not None:
        counted = y != IGNORE
        label = torch.where(counted, y, 0)[:, None]
    if weight < 1.0:
        e1 = torch.exp(x32)
        z1 = e1.sum(dim=1, keepdim=True)
        row = row + (1.0 - weight) * (torch.log(z1) - x32.gather(1, label))[:, 0]
    count = float(case["rows"])
    if counted is not None:
        row = torch.where(counted, row, 0.0)
        count = counted.sum().clamp(min=1).float()
    loss = row.sum() / count
    if case["pass"] == "loss":
        return [loss]
    g = e / z * (weight * tau)
    g.scatter_add_(1, s["index"], -weight * tau * p)
    if weight < 1.0:
        e1 = e1 / z1 * (1.0 - weight)
        e1.scatter_add_(1, label, torch.full_like(label, weight - 1.0, dtype=torch.float32))
        g = g + e1
    if counted is not None:
        g = torch.where(counted[:, None], g, 0.0)
    return [loss, (g * (case["scale"] / count)).to(x.dtype)]


# ---- the framework's operators ---------------------------------------------------------------------------------


def _own_embedding(s):
    from tandem_amd import ops

    case, scale, padding = s["case"], s["case"]["scale"], s["padding"]
    if case["pass"] == "grad":
        return [ops.embedding_grad(s["grad"], s["tokens"], case["vocab"], scale=scale, padding_idx=padding)]
    out = ops.embedding(s["tokens"], s["weight"], scale=scale, padding_idx=padding)
    if case["pass"] == "forward":
        return [out]
    return [out, *torch.autograd.grad(out, s["weight"], s["grad"])]


def _own_qk(s):
    from tandem_amd import ops

    case = s["case"]
    how = dict(positions=s["positions"], inv_freq=s["inv_freq"], eps=EPS, interleaved=case["interleaved"])
    weights = (s["q_weight"], s["k_weight"])
    if case["form"] == "packed":
        heads = (case["q_heads"], case["kv_heads"])
        if case["pass"] == "grad":
            d = ops.qkv_norm_rope_grad(s["dq"], s["dk"], s["dv"], s["qkv"], *heads, *weights, **how)
            return dict(zip(("dqkv", "dq_weight", "dk_weight"), d))
        q, k, v = ops.qkv_norm_rope(s["qkv"], *heads, *weights, **how)
        out = {"q": q, "k": k, "v": v}
        if case["pass"] == "train":
            d = torch.autograd.grad((q, k, v), (s["qkv"], *weights), (s["dq"], s["dk"], s["dv"]))
            out.update(zip(("dqkv", "dq_weight", "dk_weight"), d))
        return out
    if case["pass"] == "grad":
        d = ops.qk_norm_rope_grad(s["dq"], s["dk"], s["q"], s["k"], *weights, **how)
        return dict(zip(("dq", "dk", "dq_weight", "dk_weight"), d))
    q, k = ops.qk_norm_rope(s["q"], s["k"], *weights, **how)
    out = {"q": q, "k": k}
    if case["pass"] == "train":
        d = torch.autograd.grad((q, k), (s["q"], s["k"], *weights), (s["dq"], s["dk"]))
        out.update(zip(("dq", "dk", "dq_weight", "dk_weight"), d))
    return out


def _own_distill(s):
    from tandem_amd import ops

    case = s["case"]
    how = dict(targets=s["targets"], temperature=case["temperature"], weight=case["weight"], ignore_index=IGNORE)
    if case["pass"] == "grads":
        return list(ops.distill_loss_and_grad(s["logits"], s["index"], s["teacher"], scale=case["scale"], **how))
    loss = ops.distill_loss(s["logits"], s["index"], s["teacher"], **how)
    if case["pass"] == "loss":
        return [loss]
    return [loss, *torch.autograd.grad(loss, s["logits"], s["upstream"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"embedding": _own_embedding, "qk_norm_rope": _own_qk, "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "qk_norm_rope": _plain_qk, "distill": _plain_distill}[op](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    es, what = SIZE[case["dtype"]], case["pass"]
    forward, backward = what in ("forward", "loss", "train"), what in ("grad", "grads", "train")
    if case["op"] == "embedding":
        n, d, index = case["batch"] * case["seq"], case["dim"], 4 if case["index"] == "int32" else 8
        rows = min(n, case["vocab"])  # rows of the table that a lookup touches, at most
        return {"bytes": forward * (n * index + (rows + n) * d * es) + backward * (n * index + n * d * es + case["vocab"] * d * es),
                "flops": float(forward * n * d + backward * (n + case["vocab"]) * d)}
    if case["op"] == "qk_norm_rope":
        n = case["batch"] * case["seq"]
        x = n * (case["q_heads"] + case["kv_heads"]) * case["head_dim"]
        v = n * case["kv_heads"] * case["head_dim"] if case["form"] == "packed" else 0
        small = n * 8 + case["rotary"] * 4 + 2 * case["head_dim"] * es
        return {"bytes": forward * (2 * x * es + small) + backward * (3 * x * es + 2 * v * es + small + 2 * case["head_dim"] * es),
                "flops": float(forward * 8 * x + backward * 16 * x)}
    # a training pass reads the logits once and writes their gradient once: both come from the same row
    n, x = case["rows"], case["rows"] * case["vocab"]
    small = n * min(case["k"], case["vocab"]) * 12 + n * 8
    return {"bytes": x * es * (2 if backward else 1) + small, "flops": float(x * (8 if backward else 4))}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------


def _exact_embedding(s):
    case = s["case"]
    out = []
    tokens, dim = s["tokens"].reshape(-1).long(), case["dim"]
    if case["pass"] != "grad":
        out.append(case["scale"] * torch.index_select(s["weight"].detach(), 0, tokens).double().view(*s["tokens"].shape, dim))
    if case["pass"] != "forward":
        # sorted by token, the gradient of one is a difference of two running sums
        order = torch.argsort(tokens, stable=True)
        run_sum = torch.cumsum(s["grad"].reshape(-1, dim)[order].double(), dim=0)
        run_sum = torch.cat((torch.zeros_like(run_sum[:1]), run_sum))
        ends = torch.searchsorted(tokens[order], torch.arange(case["vocab"], device="cuda"), right=True)
        begins = torch.cat((torch.zeros_like(ends[:1]), ends[:-1]))
        dw = torch.zeros(case["vocab"], dim, device="cuda", dtype=torch.float64)
        named = (ends > begins).nonzero()[:, 0]
        dw[named] = (run_sum[ends[named]] - run_sum[begins[named]]) * case["scale"]
        if s["padding"] is not None:
            dw[s["padding"]] = 0.0
        out.append(dw)
    return out


def _exact_turn(x, weight, angle, case):
    rotary = case["rotary"]
    y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * weight
    t = y[..., :rotary]
    pairs = t.unflatten(-1, (rotary // 2, 2)) if case["interleaved"] else t.unflatten(-1, (2, rotary // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle)
    pairs = torch.view_as_real(z)
    t = pairs.flatten(-2) if case["interleaved"] else pairs.transpose(-1, -2).flatten(-2)
    return torch.cat((t, y[..., rotary:]), dim=-1)


def _exact_qk(s):
    case = s["case"]
    b, t, hq, hk, d = (case[n] for n in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
    leaves = [x.detach().double().requires_grad_() for x in ((s["qkv"],) if case["form"] == "packed" else (s["q"], s["k"]))]
    qw, kw = (s[n].detach().double().requires_grad_() for n in ("q_weight", "k_weight"))
    if case["form"] == "packed":
        heads = leaves[0].view(b, t, hq + 2 * hk, d)
        q, k, v = heads[:, :, :hq], heads[:, :, hq: hq + hk], heads[:, :, hq + hk:]
    else:
        q, k, v = *leaves, None
    angle = (s["positions"].double()[:, :, None] * s["inv_freq"])[:, :, None, :]
    rq, rk = _exact_turn(q, qw, angle, case), _exact_turn(k, kw, angle, case)
    out = {}
    if case["pass"] != "grad":
        out["q"], out["k"] = rq.detach(), rk.detach()
        if v is not None:
            out["v"] = v.detach()
    if case["pass"] != "forward":
        outs, gs = ((rq, rk, v), (s["dq"], s["dk"], s["dv"])) if v is not None else ((rq, rk), (s["dq"], s["dk"]))
        grads = torch.autograd.grad(outs, (*leaves, qw, kw), [g.double() for g in gs])
        out.update(zip(("dqkv", "dq_weight", "dk_weight") if v is not None else ("dq", "dk", "dq_weight", "dk_weight"), grads))
    return out


def _exact_distill(s):
    case, rows = s["case"], s["case"]["rows"]
    tau, weight = case["temperature"], case["weight"]
    counted = torch.ones(rows, device="cuda", dtype=torch.bool) if s["targets"] is None else s["targets"] != IGNORE
    count = max(1, int(counted.sum()))
    step = max(1, (1 << 26) // case["vocab"])
    loss, grads = 0.0, []
    for a in range(0, rows, step):
        x = s["logits"][a:a + step].detach().double().requires_grad_()
        p = torch.log_softmax(s["teacher"][a:a + step].double() / tau, dim=1)
        q = torch.log_softmax(x / tau, dim=1).gather(1, s["index"][a:a + step])
        row = weight * tau ** 2 * (p.exp() * (p - q)).sum(dim=1)
        if weight < 1.0:
            y = s["targets"][a:a + step].clamp(min=0)
            row = row - (1.0 - weight) * torch.log_softmax(x, dim=1).gather(1, y[:, None])[:, 0]
        part = (row * counted[a:a + step]).sum() / count
        if case["pass"] != "loss":
            grads.append(torch.autograd.grad(part * case["scale"], x)[0])
        loss = loss + part.detach()
    return [loss] if case["pass"] == "loss" else [loss, torch.cat(grads)]


def exact(case, seed):
    return {"embedding": _exact_embedding, "qk_norm_rope": _exact_qk, "distill": _exact_distill}[case["op"]](prepare(case, seed))
