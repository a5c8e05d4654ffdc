"""What the model operators do around their launches, on the CPU: the launches are replaced by nothing, the rest is as on the GPU."""

import pytest
import torch
from torch.autograd import forward_ad


class NoLaunches:
    """The library, its kernels left out: every launch is noted with its arguments."""

    def __init__(self, library):
        self.library, self.calls, self.capture = library, [], 0

    def tdm_stream_capture_id(self, stream):
        return self.capture

    def __getattr__(self, name):
        if not name.startswith("tdm_k") or name.endswith("_workspace"):
            return getattr(self.library, name)

        def launch(*args):
            self.calls.append((name, args))
            return 0

        return launch


@pytest.fixture
def launches(monkeypatch):
    from tandem_amd import ops

    stand_in = NoLaunches(ops.lib())
    monkeypatch.setattr(ops, "lib", lambda: stand_in)
    monkeypatch.setattr(ops, "_on_gpu", lambda t, what: None)
    monkeypatch.setattr(ops, "require_device_tensor", lambda t, what: None)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)  # a CPU tensor's get_device()
    monkeypatch.setattr(ops, "_current_stream", lambda device: 0)
    return stand_in.calls


@pytest.fixture
def stand_in(launches):
    from tandem_amd import ops

    return ops.lib()


def operands():
    """The operands of every operator and of its gradient, by name."""
    from tandem_amd import ops

    tokens, positions = torch.tensor([1, 2, 1]), torch.arange(3)
    w, g = torch.randn(5, 8), torch.randn(3, 8)
    q, k, v, qkv = torch.randn(1, 3, 2, 8), torch.randn(1, 3, 1, 8), torch.randn(1, 3, 1, 8), torch.randn(1, 3, 32)
    qw, kw, freq = torch.randn(8), torch.randn(8), ops.rope_frequencies(8, device="cpu")
    x, t, columns, y = torch.randn(3, 9), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64), torch.tensor([1, 2, 3])
    return {
        "embedding": (lambda w: ops.embedding(tokens, w), dict(w=w)),
        "embedding_grad": (lambda g: ops.embedding_grad(g, tokens, 5), dict(g=g)),
        "qk_norm_rope": (lambda q, k, qw, kw, freq: ops.qk_norm_rope(q, k, qw, kw, positions, freq), dict(q=q, k=k, qw=qw, kw=kw, freq=freq)),
        "qk_norm_rope_grad": (lambda dq, dk, q, k, qw, kw, freq: ops.qk_norm_rope_grad(dq, dk, q, k, qw, kw, positions, freq),
                              dict(dq=q.clone(), dk=k.clone(), q=q, k=k, qw=qw, kw=kw, freq=freq)),
        "qkv_norm_rope": (lambda qkv, qw, kw, freq: ops.qkv_norm_rope(qkv, 2, 1, qw, kw, positions, freq), dict(qkv=qkv, qw=qw, kw=kw, freq=freq)),
        "qkv_norm_rope_grad": (lambda dq, dk, dv, qkv, qw, kw, freq: ops.qkv_norm_rope_grad(dq, dk, dv, qkv, 2, 1, qw, kw, positions, freq),
                               dict(dq=q.clone(), dk=k.clone(), dv=v, qkv=qkv, qw=qw, kw=kw, freq=freq)),
        "distill_loss": (lambda x, t: ops.distill_loss(x, columns, t, targets=y, weight=0.5), dict(x=x, t=t)),
        "distill_loss_and_grad": (lambda x, t: ops.distill_loss_and_grad(x, columns, t, targets=y, weight=0.5), dict(x=x, t=t)),
    }


NAMES = ["embedding", "embedding_grad", "qk_norm_rope", "qk_norm_rope_grad", "qkv_norm_rope", "qkv_norm_rope_grad", "distill_loss", "distill_loss_and_grad"]
DIFFERENTIABLE = ["embedding", "qk_norm_rope", "qkv_norm_rope", "distill_loss"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_derivatives_are_refused(launches, name):
    """An operand with a tangent would come out without one: a derivative of zero."""
    call, given = operands()[name]
    with forward_ad.dual_level():
        call(**given)  # no tangents, no refusal
        for which in given:
            done = len(launches)
            with pytest.raises(NotImplementedError, match="forward mode"):
                call(**{**given, which: forward_ad.make_dual(given[which], torch.ones_like(given[which]))})
            assert len(launches) == done, which
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                call(**{**given, which: forward_ad.make_dual(given[which], torch.ones_like(given[which]))})


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_an_upstream_gradient_with_a_tangent_is_refused(launches, name):
    call, given = operands()[name]
    first = next(iter(given))
    out = call(**{**given, first: given[first].clone().requires_grad_()})
    out = out if isinstance(out, torch.Tensor) else out[0]
    leaf = out.grad_fn.next_functions
    assert leaf
    done = len(launches)
    with forward_ad.dual_level():
        up = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward mode"):
            out.backward(up)
    assert len(launches) == done


@pytest.mark.parametrize("name", NAMES)
def test_a_call_that_is_being_recorded_is_refused(launches, name):
    """A trace would hold the result's memory without what is written there."""
    from torch.fx.experimental.proxy_tensor import make_fx

    call, given = operands()[name]
    values = tuple(given.values())
    for record in (lambda: torch.jit.trace(lambda *x: call(*x), values, check_trace=False), lambda: make_fx(lambda *x: call(*x))(*values),
                   lambda: make_fx(lambda *x: call(*x), pre_dispatch=True)(*values)):
        with pytest.raises(NotImplementedError, match="recorded"):
            record()
    assert not launches
    call(**given)
    assert launches


def test_a_backward_pass_that_is_being_recorded_is_refused(launches):
    from torch.fx.experimental.proxy_tensor import make_fx

    call, given = operands()["embedding"]
    out = call(given["w"].requires_grad_())
    with pytest.raises(NotImplementedError, match="recorded"):
        make_fx(lambda g: torch.autograd.grad(out, given["w"], g, retain_graph=True))(torch.ones_like(out))
    assert len(launches) == 1


def test_a_compiled_program_leaves_its_graph_for_a_launch(launches):
    call, given = operands()["embedding"]
    w = given["w"].requires_grad_()
    program = torch.compile(lambda w: call(w) * 0 + 2, backend="eager")
    for n in (1, 2):
        program(w).sum().backward()
        assert [name for name, _ in launches] == ["tdm_k5_embedding", "tdm_k5_embedding_grad"] * n


def test_an_empty_batch_with_hard_targets_is_no_error_in_the_library():
    """No rows, so no targets either: an empty tensor's address is zero. Nothing is launched where no loss is wanted."""
    from tandem_amd import _lib

    L = _lib.lib()
    work = torch.empty(4096, dtype=torch.uint8)
    at = (work.data_ptr() + 15) // 16 * 16
    for weight in (1.0, 0.5, 0.0):
        for reduction in (0, 1, 2):
            how = _lib.DISTILL_HOW.pack(0, 50, -100, 4, 0, 4, 0, 4, reduction, 1.0, weight, 1.0)
            status = L.tdm_k7_distill(how, None, None, None, None, None, None, None, 0, at, L.tdm_k7_distill_workspace(how), None)
            assert status == 0, (weight, reduction, L.tdm_last_error())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [0, 1, 3])
def test_logits_that_come_back_elsewhere_get_a_gradient_at_their_alignment(launches, dtype, lead):
    """Hooks on saved tensors may give the backward pass a copy: the gradient that the forward pass left lies as the logits did then."""
    from tandem_amd import ops

    storage = torch.zeros(4 * 9 + 8, dtype=dtype)
    x = storage[lead:lead + 36].view(4, 9).requires_grad_()
    assert x.data_ptr() % 16 == lead * x.element_size() % 16  # torch's own allocations begin on 64 bytes
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone()):
        loss = ops.distill_loss(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))
    for _ in range(2):
        (grad,) = torch.autograd.grad(loss, x, retain_graph=True)
        name, args = launches[-1]
        logits, written, keep_ones = args[1], args[6], args[8]
        assert name == "tdm_k7_distill" and logits % 16 == 0 and written == grad.data_ptr() and written % 16 == 0
        assert grad.shape == x.shape and (lead == 0 or not keep_ones)


@pytest.mark.parametrize("forward,backward,handed_out", [(0, 0, True), (7, 7, True), (0, 7, False), (7, 0, False), (7, 8, False), (-1, -1, False)])
def test_the_forward_pass_s_gradient_stays_within_its_capture(stand_in, forward, backward, handed_out):
    """A graph that holds the backward pass alone is replayed without the forward pass: a gradient handed out there would be what the last
    replay's user made of it. The forward pass's is handed out within one capture, or where there is none."""
    from tandem_amd import ops

    x = torch.zeros(4, 12, requires_grad=True)
    stand_in.capture = forward
    loss = ops.distill_loss(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))
    left = stand_in.calls[-1][1][6]
    stand_in.capture = backward
    (grad,) = torch.autograd.grad(loss, x)
    _, args = stand_in.calls[-1]
    assert args[8] == handed_out and args[6] == grad.data_ptr() and (args[6] == left) == handed_out


@pytest.mark.parametrize("name", ["qk_norm_rope", "qkv_norm_rope"])
def test_frequencies_that_want_a_gradient_are_refused(launches, name):
    """They get none: a trained table of angles would stay as it is without a word."""
    call, given = operands()[name]
    with pytest.raises(ValueError, match="inv_freq"):
        call(**{**given, "freq": given["freq"].clone().requires_grad_()})
    with torch.no_grad():
        call(**{**given, "freq": given["freq"].clone().requires_grad_()})
    assert len(launches) == 1


def test_the_rotary_model_refuses_sequences_beyond_its_length(launches):
    """Also of a model for one position, whose position would be repeated."""
    from tandem_amd.model import GPT, Config

    for seq in (1, 4):
        model = GPT(Config(seq=seq, layers=1, heads=2, dim=16, rotary=True))
        model(torch.zeros(1, seq, dtype=torch.int64))
        with pytest.raises(ValueError, match=f"{seq + 1} tokens"):
            model(torch.zeros(1, seq + 1, dtype=torch.int64))


def test_hooks_on_the_rotary_model_s_token_embedding_run(launches):
    """The embedding is a module of its own, as in the plain model: what is registered on it is called, and what it is replaced by is used."""
    from tandem_amd.model import GPT, Config

    for rotary in (False, True):
        model = GPT(Config(seq=8, layers=1, heads=2, dim=16, rotary=rotary, embed_scale=3.0 if rotary else 1.0))
        seen = []
        model.embed.tok.register_forward_pre_hook(lambda module, args: seen.append(args[0].shape))
        model.embed.tok.register_forward_hook(lambda module, args, out: seen.append(out.shape))
        model(torch.zeros(2, 5, dtype=torch.int64))
        assert seen == [(2, 5), (2, 5, 16)], rotary
        assert isinstance(model.embed.tok, torch.nn.Embedding) and "embed.tok.weight" in model.state_dict()
        model.embed.tok = torch.nn.Identity()
        model.embed.tok.forward = lambda idx: torch.ones(*idx.shape, 16)
        done = [name for name, _ in launches].count("tdm_k5_embedding")
        model(torch.zeros(2, 5, dtype=torch.int64))
        assert [name for name, _ in launches].count("tdm_k5_embedding") == done
    name, args = next(call for call in launches if call[0] == "tdm_k5_embedding")
    assert args[-2] == 3.0


def without_memory(t):
    """A tensor of t's shape whose storage has been given back, as sharded weights between their uses: its address is zero."""
    t = t.clone()
    t.untyped_storage().resize_(0)
    assert t.data_ptr() == 0
    return t


@pytest.mark.parametrize("name,which", [(name, which) for name in ("qk_norm_rope", "qk_norm_rope_grad", "qkv_norm_rope", "qkv_norm_rope_grad")
                                        for which in ("qw", "kw", "dq", "dk", "dv") if which in ("qw", "kw") or (name.endswith("grad") and (which != "dv" or "qkv" in name))])
def test_an_operand_without_memory_is_no_missing_operand(launches, name, which):
    """For the library an address of zero is "none": weights of one, upstream gradients of zero. (It refuses it itself where an operand is needed.)"""
    call, given = operands()[name]
    operand = without_memory(given[which])
    with pytest.raises(ValueError, match="memory"):
        call(**{**given, which: operand})
    assert not launches


def test_targets_and_upstream_gradients_without_memory_are_refused(launches):
    from tandem_amd import ops

    x, columns, t, y = torch.randn(3, 9, requires_grad=True), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2), torch.tensor([1, 2, 3])
    with pytest.raises(ValueError, match="memory"):
        ops.distill_loss(x, columns, t, targets=without_memory(y))
    loss = ops.distill_loss(x, columns, t, targets=y, reduction="none")
    with pytest.raises(ValueError, match="memory"):
        loss.backward(without_memory(torch.ones(3)))
