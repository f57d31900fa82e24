"""GPU tests of the operators of include/schemanet_blocks.h at their edges: derivatives that would be lost, values at
the end of a type's range."""
import os
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwd

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "schemanet-pytorch_amd"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from cpp_extension import ops
    return ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------------------ derivatives that would be lost
def test_forward_mode_is_refused(ops):
    """a tangent on an input, or on an upstream gradient, would come out as a derivative of zero"""
    g = gen(1)
    x, w, target = rand(g, 6, 64), torch.ones(64, device=DEV), torch.arange(6, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.gated_residual_norms(d, x, pre=(w, None)), lambda: ops.gated_residual_norms(x, d), lambda: ops.label_log_probs(d, target),
                     lambda: ops.checkpoint8_weight_grad(d, ops.checkpoint8(x)), lambda: ops.linear_checkpoint8(d, rand(gen(2), 16, 64))):
            with pytest.raises(NotImplementedError):
                call()
        leaf = x.clone().requires_grad_()
        for out in (ops.gated_residual_norms(leaf, x, pre=(w, None))[1], ops.gated_residual_norms(leaf, x)[0], ops.label_log_probs(leaf, target).log_probs,
                    ops.label_log_probs(leaf, target).entropy):
            up = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="backward.*no forward-mode"):
                torch.autograd.grad(out, leaf, up)
    ops.gated_residual_norms(x, x), ops.label_log_probs(x, target)


def test_function_transforms_are_refused(ops):
    """torch.func hands over wrapped tensors without memory of their own"""
    x, target = rand(gen(3), 4, 6, 64), torch.arange(24, device=DEV).reshape(4, 6)
    for f in (lambda v: ops.gated_residual_norms(v, v)[0].sum(), lambda v: ops.label_log_probs(v, target).log_probs.sum(),
              lambda v: ops.checkpoint8(v).restore().sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
    for f in (lambda v: ops.gated_residual_norms(v, v)[0], lambda v: ops.checkpoint8(v).restore()):
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x)


# ------------------------------------------------------------------------------------------------ the end of a type's range
@pytest.mark.parametrize("n", [1, 5, 8, 33, 256])
def test_restore_to_float16_stays_finite(ops, n):
    """float16 activations up to the largest: a block with max|x| >= 65280 has step 1024, so an element is off by at most 512, and
    max|x| = 65504 -> 64 steps = 65536, which float16 does not have.  What was infinite or NaN marks its block as before."""
    for top in (65504.0, 65472.0, 65024.0, 64992.0, 65280.0, 65248.0, 32768.0):
        g = gen(int(top) + n)
        x = (torch.rand(7, n, generator=g) * 2 - 1) * top
        x[:, 0], x[3, 0] = top, -top
        x = x.to(F16).to(DEV)
        kept = ops.checkpoint8(x)
        got, held = kept.restore(), kept.restore(F32)
        assert got.dtype == F16 and torch.isfinite(got).all()
        step = 1024.0 if top >= 65280.0 else 512.0 if top >= 32640.0 else 256.0
        assert float((got.double() - x.double()).abs().max()) <= step / 2
        assert torch.equal(got, held.clamp(-65504.0, 65504.0).to(F16))
    wide = torch.tensor([[70000.0, -1e6, 1.0, 0.0], [3e38, -3e38, 0.0, 0.0], [float("inf"), 1.0, 2.0, 3.0], [1.0, float("nan"), 2.0, 3.0]], device=DEV)
    got = ops.checkpoint8(wide).restore(F16)
    assert got[0, :2].tolist() == [65504.0, -65504.0] and got[1].tolist() == [65504.0, -65504.0, 0.0, 0.0] and torch.isnan(got[2:]).all()
