"""What the decoder-step operators do where autograd asks for more than they give: they refuse, and never
return a result that a derivative has silently left. No GPU: the tensors are fake CUDA tensors (shapes,
types and autograd state without data) and the library calls are stubbed."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.bfloat16: torch.empty(shape, device="cuda", dtype=dtype)


def _calls(fake, monkeypatch):
    """name -> (the call on (a list of) differentiable inputs, their shapes and dtypes)."""
    from SSA import ssa_cross_entropy, ssa_gated_ffn, ssa_grad_clip, ssa_qk_norm_rope
    t = fake(4, dtype=torch.int64)
    monkeypatch.setattr(ssa_cross_entropy, "_forward", lambda x, w, *a: (
        fake(dtype=torch.float32), x, w, t, fake(5, dtype=torch.float32)))
    monkeypatch.setattr(ssa_gated_ffn, "_forward", lambda x, w: (fake(4, w.shape[0] // 2), x, w))
    monkeypatch.setattr(ssa_qk_norm_rope, "_forward", lambda x, *a: (
        (fake(4, 2, 16), fake(4, 1, 16), fake(4, 1, 16)), (x, a[2], a[3], None, a[0], a[1]), 0))
    monkeypatch.setattr(ssa_grad_clip, "_run", lambda *a, **k: fake(dtype=torch.float32))
    bf, f32 = torch.bfloat16, torch.float32
    cos, sin = fake(4, 16, dtype=f32), fake(4, 16, dtype=f32)
    return {
        "loss": (lambda x, w: ssa_cross_entropy.ssa_linear_cross_entropy(x, w, t),
                 [((4, 64), bf), ((50, 64), bf)]),
        "ffn": (ssa_gated_ffn.ssa_gated_ffn, [((4, 64), bf), ((16, 64), bf)]),
        "rope": (lambda x, a, b: ssa_qk_norm_rope.ssa_qk_norm_rope(x, 2, 1, cos, sin, a, b),
                 [((4, 64), bf), ((16,), bf), ((16,), bf)]),
        "tables": (lambda c, s: ssa_qk_norm_rope.ssa_qk_norm_rope(fake(4, 64), 2, 1, c, s),
                   [((4, 16), f32), ((4, 16), f32)]),
        "norm": (lambda *g: ssa_grad_clip.ssa_grad_norm(g), [((4, 64), bf), ((7,), bf)]),
        "clip": (lambda *g: ssa_grad_clip.ssa_clip_grad_norm(g, 1.0), [((4, 64), bf), ((7,), bf)]),
        "clip into": (lambda *g: ssa_grad_clip.ssa_clip_grad_norm(
            g, 1.0, out=[fake(*t.shape, dtype=f32) for t in g]), [((4, 64), bf), ((7,), bf)]),
    }


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", ["loss", "ffn", "rope", "tables", "norm", "clip", "clip into"])
def test_tangents_are_refused(fake, monkeypatch, name, grad_mode):
    call, inputs = _calls(fake, monkeypatch)[name]
    call(*[fake(*s, dtype=d) for s, d in inputs])  # the same call without a tangent goes through
    for i in range(len(inputs)):
        with fwAD.dual_level(), torch.set_grad_enabled(grad_mode):
            args = [fake(*s, dtype=d) for s, d in inputs]
            call(*args)
            args[i] = fwAD.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                call(*args)


@pytest.mark.parametrize("name", ["loss", "ffn", "rope"])
def test_tangents_of_incoming_gradients_are_refused(fake, monkeypatch, name):
    from SSA import ssa_cross_entropy, ssa_gated_ffn, ssa_qk_norm_rope
    fn, outs = {"loss": (ssa_cross_entropy.SSALinearCrossEntropyFunc, [()]),
                "ffn": (ssa_gated_ffn.SSAGatedFFNFunc, [(4, 8)]),
                "rope": (ssa_qk_norm_rope.SSAQKNormRopeFunc, [(4, 2, 16), (4, 1, 16), (4, 1, 16)])}[name]
    for i in range(len(outs)):
        with fwAD.dual_level():
            grads = [fake(*s) for s in outs]
            grads[i] = fwAD.make_dual(grads[i], torch.ones_like(grads[i]))
            with pytest.raises(NotImplementedError):
                fn.backward(None, *grads)  # before anything of the context is read


def test_the_norm_refuses_gradients_with_a_graph(fake, monkeypatch):
    from SSA import ssa_grad_clip
    monkeypatch.setattr(ssa_grad_clip, "_run", lambda *a, **k: fake(dtype=torch.float32))
    leaf = fake(4, 64).requires_grad_(True)
    made = leaf * 2  # as torch.autograd.grad(..., create_graph=True) returns them
    with pytest.raises(ValueError, match="create_graph"):
        ssa_grad_clip.ssa_grad_norm([fake(3), made])
    ssa_grad_clip.ssa_grad_norm([fake(3), made.detach()])
    with torch.no_grad():
        ssa_grad_clip.ssa_grad_norm([fake(3), made])
    ssa_grad_clip.ssa_grad_norm([leaf])


@pytest.mark.parametrize("which", [0, 1])
def test_rotation_tables_with_a_gradient_are_refused(fake, monkeypatch, which):
    call, inputs = _calls(fake, monkeypatch)["tables"]
    args = [fake(*s, dtype=d) for s, d in inputs]
    args[which].requires_grad_(True)
    with pytest.raises(ValueError, match="without a gradient"):
        call(*args)
    with torch.no_grad():
        call(*args)
