"""What the model operators refuse before they touch the GPU: through Python and through the C ABI."""

import ctypes

import pytest
import torch


def _lib():
    from tandem_amd import _lib

    return _lib


def test_packed_structures_have_the_sizes_the_header_gives_them(tmp_path):
    import os
    import subprocess

    source = tmp_path / "sizes.c"
    source.write_text('#include "tandem_hip.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu", sizeof(tdm_heads), sizeof(tdm_positions), '
                      'sizeof(tdm_qk_shape), sizeof(tdm_distill_how)); return 0; }\n')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(source), "-o", str(tmp_path / "sizes")], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], stdout=subprocess.PIPE, text=True, check=True).stdout.split()
    L = _lib()
    assert [int(n) for n in got] == [s.size for s in (L.HEADS, L.POSITIONS, L.QK_SHAPE, L.DISTILL_HOW)]


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
    most, wide = 1 << 28, 1 << 20  # refused before the first launch, which would write
    refused(grad(p, p, i64, p, p, L.tdm_k5_embedding_grad_workspace(most, 4, wide), most, 4, wide, f32, 1.0, -1), "one launch")


def test_qk_norm_rope_refuses_cpu_tensors_and_odd_rotations():
    from tandem_amd import ops

    q, freq = torch.zeros(1, 2, 3, 64), torch.zeros(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.qk_norm_rope(q, q, None, None, torch.arange(2), freq)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.qkv_norm_rope(torch.zeros(1, 2, 192), 1, 1, None, None, torch.arange(2), freq)
    with pytest.raises(ValueError, match="even"):
        ops.rope_frequencies(63, device="cpu")
    f = ops.rope_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 10 ** -0.5, 0.1, 10 ** -1.5], dtype=torch.float64), rtol=1e-14)


def test_qk_norm_rope_argument_errors_need_no_gpu():
    lib = _lib()
    L = lib.lib()
    fields = dict(batch=1, tokens=2, q_heads=4, kv_heads=2, head_dim=64, rotary_dim=64, interleaved=0, dtype=3, weight_dtype=3, position_dtype=4, eps=1e-6)
    shape = lambda **change: lib.QK_SHAPE.pack(*{**fields, **change}.values())  # noqa: E731
    no_heads, no_positions = lib.HEADS.pack(0, 0, 0, 0), lib.POSITIONS.pack(0, 0, 0)
    h, at, p = lib.HEADS.pack(4096, 128, 64, 64), lib.POSITIONS.pack(4096, 0, 1), ctypes.c_void_p(4096)  # never read
    call = lambda s, **k: L.tdm_k6_qk_norm_rope(s, k.get("q", h), h, p, p, k.get("at", at), k.get("freq", p), h, h, None)  # noqa: E731
    for change, word in ((dict(dtype=1), "dtype"), (dict(weight_dtype=2), "weights"), (dict(position_dtype=0), "positions"), (dict(tokens=1 << 31), "tokens"),
                         (dict(batch=-1), "tokens"), (dict(q_heads=-1), "heads"), (dict(head_dim=63), "even"), (dict(head_dim=514), "512"),
                         (dict(rotary_dim=66), "rotated"), (dict(rotary_dim=3), "rotated"), (dict(eps=-1.0), "eps")):
        refused(call(shape(**change)), word)
        assert L.tdm_k6_qk_norm_rope_grad_workspace(shape(**change)) == -1
    refused(call(shape(), q=no_heads), "null")
    refused(call(shape(), at=no_positions), "null")
    refused(call(shape(), freq=None), "null")
    assert call(shape(tokens=0), q=no_heads) == 0
    need = L.tdm_k6_qk_norm_rope_grad_workspace(shape())
    assert need >= 2 * 64 * 4
    grad = lambda w, n: L.tdm_k6_qk_norm_rope_grad(shape(), h, h, None, h, h, p, p, at, p, h, h, None, p, p, w, n, None)  # noqa: E731
    refused(grad(p, need - 1), "workspace")
    refused(grad(None, need), "workspace")
    refused(grad(ctypes.c_void_p(4100), need), "workspace")


def test_distill_loss_refuses_cpu_tensors():
    from tandem_amd import ops

    with pytest.raises(ValueError, match="no CPU path"):
        ops.distill_loss(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3))


def test_distill_argument_errors_need_no_gpu():
    lib = _lib()
    L = lib.lib()
    fields = dict(rows=4, vocab=100, ignore_index=-100, k=8, dtype=0, index_dtype=4, teacher_dtype=0, target_dtype=4, reduction=1, temperature=2.0,
                  weight=1.0, scale=1.0)
    how = lambda **change: lib.DISTILL_HOW.pack(*{**fields, **change}.values())  # noqa: E731

    p, off = ctypes.c_void_p(4096), ctypes.c_void_p(4100)  # never read
    need = L.tdm_k7_distill_workspace(how())
    assert need >= 16

    def call(h, logits=p, index=p, targets=p, loss=p, grad=p, work=p, nbytes=need):
        return L.tdm_k7_distill(h, logits, index, p, targets, loss, grad, None, 0, work, nbytes, None)

    for change, word in ((dict(dtype=1), "logits"), (dict(teacher_dtype=4), "teacher"), (dict(index_dtype=0), "columns"), (dict(target_dtype=0), "targets"),
                         (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"), (dict(vocab=0), "logits in a row"), (dict(vocab=1 << 31), "logits in a row"),
                         (dict(k=0), "teacher's logits"), (dict(k=1025), "1024"), (dict(temperature=0.0), "temperature"),
                         (dict(temperature=float("inf")), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(weight=-0.1), "weight"),
                         (dict(weight=1.1), "weight"), (dict(weight=float("nan")), "weight"), (dict(reduction=3), "reduction")):
        refused(call(how(**change)), word)
        assert L.tdm_k7_distill_workspace(how(**change)) == -1
    refused(call(how(weight=0.5), targets=None), "targets")
    refused(call(how(), logits=None), "null")
    refused(call(how(), index=None), "null")
    refused(call(how(), loss=None, grad=None), "wanted")
    refused(call(how(), nbytes=need - 1), "workspace")
    refused(call(how(), work=off), "workspace")
    refused(call(how(), grad=off), "16-byte")


def test_the_rotary_model_s_parameters_and_refusals():
    from tandem_amd.model import GPT, Config

    cfg = Config(seq=16, layers=1, heads=2, dim=16, rotary=True, embed_scale=4.0)
    model = GPT(cfg)
    names = [n for n, _ in model.named_parameters()]
    assert "embed.pos.weight" not in names and "blocks.0.attn.q_norm" in names and model.blocks[0].attn.q_norm.shape == (8,)
    assert [n for n, _ in GPT(Config(seq=16, layers=1, heads=2, dim=16)).named_parameters()][:2] == ["embed.tok.weight", "embed.pos.weight"]
    with pytest.raises(ValueError, match="no CPU path"):
        model(torch.zeros(1, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="rotary"):
        Config(embed_scale=2.0)
    plain = GPT(Config(seq=16, layers=1, heads=2, dim=16))
    with pytest.raises(ValueError, match="no CPU path"):
        plain(torch.zeros(1, 4, dtype=torch.int64), teacher=(torch.zeros(1, 4, 2, dtype=torch.int64), torch.zeros(1, 4, 2)))


def test_the_rotary_model_keeps_no_inference_tensors():
    """What a first call without gradients leaves behind has to serve a training step; tensors of inference mode cannot be saved for one."""
    from tandem_amd.model import GPT, Config

    attention = GPT(Config(seq=16, layers=1, heads=2, dim=16, rotary=True)).blocks[0].attn
    with torch.inference_mode():
        first = attention._rotation(torch.device("cpu"))
    assert not any(t.is_inference() for t in first)
    assert first[0].tolist() == list(range(16)) and first[1].dtype == torch.float64
    assert attention._rotation(torch.device("cpu")) is first
