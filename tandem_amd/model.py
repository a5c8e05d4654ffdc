"""The GPT every strategy trains: decoder-only, pre-norm, causal attention, GELU
MLP, LM head not tied to the embedding (so each parameter belongs to exactly
one unit when the model is sharded).

This mirrors the reference's model (tandem/model.py:14-120 there) in everything
the data-parallel path can observe: module names, parameter registration order
and shapes, the seeded initialisation (same draws in the same order), presets
and units(). The kernels here never look inside the model; it defines the shapes
of every gradient, bucket, shard and unit in the benchmarks.

Beyond the reference, and off by default: a model whose queries and keys are normed
per head and rotated by position (Config.rotary, with no position table), whose
token embedding is scaled (Config.embed_scale), and whose loss is a teacher's
(GPT.forward's `teacher`). These run on the kernels of tandem_amd.ops, on the GPU only.
"""

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops

_PRESETS = {
    "tiny": {},
    "small": dict(seq=256, layers=6, heads=6, dim=384),
    "medium": dict(seq=512, layers=12, heads=12, dim=768),  # 85,842,432 parameters
    "large": dict(seq=512, layers=24, heads=16, dim=1024),
}


@dataclass
class Config:
    vocab: int = 256  # bytes: no tokenizer
    seq: int = 128
    layers: int = 4
    heads: int = 4
    dim: int = 128
    rotary: bool = False  # queries and keys normed per head and rotated by position; no position table
    embed_scale: float = 1.0  # of the token embedding; only with rotary

    def __post_init__(self):
        if self.embed_scale != 1.0 and not self.rotary:
            raise ValueError("embed_scale needs rotary=True")

    @staticmethod
    def preset(name):
        return Config(**_PRESETS[name])


class Attention(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.heads = cfg.heads
        self.qkv = nn.Linear(cfg.dim, 3 * cfg.dim)
        self.proj = nn.Linear(cfg.dim, cfg.dim)
        self.rotary = cfg.rotary
        if cfg.rotary:
            self.q_norm = nn.Parameter(torch.ones(cfg.dim // cfg.heads))
            self.k_norm = nn.Parameter(torch.ones(cfg.dim // cfg.heads))
            self._seq, self._turn = cfg.seq, {}

    def _rotation(self, device):
        """(positions 0 .. seq - 1, angles per position) on `device`; not buffers, which a cast of the model would round. Kept for every later
        call: copied from the host, so that they are there for any stream, and no inference tensors, which training could not save."""
        if device not in self._turn:
            per_head = self.q_norm.shape[0]
            with torch.inference_mode(False):
                self._turn[device] = (torch.arange(self._seq, device="cpu").to(device), ops.rope_frequencies(per_head, device=device))
        return self._turn[device]

    def forward(self, x):
        batch, steps, width = x.shape
        if self.rotary:
            if steps > self._seq:  # a single position would be repeated instead
                raise ValueError(f"{steps} tokens for a model of {self._seq} positions")
            positions, inv_freq = self._rotation(x.device)
            heads = ops.qkv_norm_rope(self.qkv(x), self.heads, self.heads, self.q_norm, self.k_norm, positions[:steps], inv_freq)
            mixed = F.scaled_dot_product_attention(*(part.transpose(1, 2) for part in heads), is_causal=True)
            return self.proj(mixed.transpose(1, 2).reshape(batch, steps, width))
        per_head = width // self.heads
        q, k, v = (part.view(batch, steps, self.heads, per_head).transpose(1, 2)
                   for part in self.qkv(x).split(width, dim=2))
        mixed = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.proj(mixed.transpose(1, 2).reshape(batch, steps, width))


class Block(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.ln1 = nn.LayerNorm(cfg.dim)
        self.attn = Attention(cfg)
        self.ln2 = nn.LayerNorm(cfg.dim)
        self.fc = nn.Linear(cfg.dim, 4 * cfg.dim)
        self.out = nn.Linear(4 * cfg.dim, cfg.dim)

    def forward(self, x):
        x = x + self.attn(self.ln1(x))
        return x + self.out(F.gelu(self.fc(self.ln2(x))))


class ScaledEmbedding(nn.Embedding):
    """torch's embedding in everything but its pass: scale * weight[idx] by ops.embedding."""

    def __init__(self, vocab, dim, scale):
        super().__init__(vocab, dim)
        self.scale = scale

    def forward(self, idx):
        return ops.embedding(idx, self.weight, scale=self.scale, padding_idx=self.padding_idx)


class Embed(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.tok = ScaledEmbedding(cfg.vocab, cfg.dim, cfg.embed_scale) if cfg.rotary else nn.Embedding(cfg.vocab, cfg.dim)
        self.pos = None if cfg.rotary else nn.Embedding(cfg.seq, cfg.dim)

    def forward(self, idx):
        if self.pos is None:
            return self.tok(idx)
        where = torch.arange(idx.shape[1], device=idx.device)
        return self.tok(idx) + self.pos(where)


class Head(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.ln = nn.LayerNorm(cfg.dim)
        self.lm = nn.Linear(cfg.dim, cfg.vocab, bias=False)

    def forward(self, x):
        return self.lm(self.ln(x))


def _first_init(module):
    # N(0, 0.02) weights for every Linear and Embedding, zero biases
    if isinstance(module, (nn.Linear, nn.Embedding)):
        nn.init.normal_(module.weight, std=0.02)
    if isinstance(module, nn.Linear) and module.bias is not None:
        nn.init.zeros_(module.bias)


class GPT(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.config = cfg
        self.embed = Embed(cfg)
        self.blocks = nn.ModuleList(Block(cfg) for _ in range(cfg.layers))
        self.head = Head(cfg)
        self.apply(_first_init)
        residual_std = 0.02 / math.sqrt(2 * cfg.layers)  # GPT-2's scaling of the projections that feed the residual stream
        for block in self.blocks:
            nn.init.normal_(block.attn.proj.weight, std=residual_std)
            nn.init.normal_(block.out.weight, std=residual_std)

    def units(self):
        """The model as a sequence of modules: what ZeRO-3 shards one at a time."""
        return [self.embed, *self.blocks, self.head]

    def forward(self, idx, targets=None, teacher=None, temperature=1.0, teacher_weight=1.0):
        """The logits; with `targets` the loss. `teacher`: (columns, logits) of a teacher's top logits, each [batch, tokens, k]; the
        loss is then ops.distill_loss of them at `temperature`, mixed with the targets' share 1 - teacher_weight."""
        x = self.embed(idx)
        for block in self.blocks:
            x = block(x)
        logits = self.head(x)
        if teacher is not None:
            return ops.distill_loss(logits, *teacher, targets=targets, temperature=temperature, weight=teacher_weight)
        return logits if targets is None else loss_fn(logits, targets)


def loss_fn(logits, targets):
    return F.cross_entropy(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1))


def count_params(model):
    return sum(p.numel() for p in model.parameters())
