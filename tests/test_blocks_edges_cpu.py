"""CPU (-m "not gpu"): calls of the operators of include/schemanet_blocks.h that have to be turned down before a launch: derivatives that
would be lost, sizes past 32 bits, checkpoints that no longer hold their activation; a GNN that
was pickled before it could be residual; and the workspace functions at any numbers.  No kernel is launched here."""
import os
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture(scope="module")
def ops():
    import cpp_extension
    cpp_extension.build()
    from cpp_extension import ops
    return ops


def dual(*shape):
    return fwd.make_dual(torch.ones(*shape), torch.ones(*shape))


@pytest.mark.parametrize("name", ["x", "branch", "gate", "scale", "post weight", "post bias", "pre weight", "pre bias"])
@pytest.mark.parametrize("grad", [False, True])
def test_norms_refuse_a_forward_mode_tangent(ops, name, grad):
    v = {k: torch.ones(3, 8) for k in ("x", "branch", "gate")}
    v.update({k: torch.ones(8) for k in ("scale", "post weight", "post bias", "pre weight", "pre bias")})
    call = lambda: ops.gated_residual_norms(v["x"], v["branch"], gate=v["gate"], scale=v["scale"], post=(v["post weight"], v["post bias"]),      # noqa: E731
                                            pre=(v["pre weight"], v["pre bias"]))
    with torch.set_grad_enabled(grad), fwd.dual_level():
        v[name] = dual(*v[name].shape)
        with pytest.raises(NotImplementedError, match="gated_residual_norms: no forward-mode"):
            call()
        with fwd._set_fwd_grad_enabled(False):                       # inside a Function's forward: its jvp answers for its inputs
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call()


def test_scores_refuse_a_forward_mode_tangent(ops):
    target = torch.zeros(3, dtype=torch.int64)
    with fwd.dual_level():
        x = dual(3, 8)
        with pytest.raises(NotImplementedError, match="label_log_probs: no forward-mode"):
            ops.label_log_probs(x, target)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="label_log_probs: no forward-mode"):
            ops.label_log_probs(x, target, topk=2)


def test_weight_grad_refuses_a_forward_mode_tangent(ops):
    kept = ops.Checkpoint8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8), (6, 20), torch.float32)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="checkpoint8_weight_grad: no forward-mode"):
        ops.checkpoint8_weight_grad(dual(6, 5), kept)


@pytest.mark.parametrize("n", [(1 << 30) + 1, 1 << 31, (1 << 32) + 32])
def test_features_past_32_bits_are_refused(ops, n):
    """2^32 + 32 features read as 32 would leave most of the checkpoint unwritten.  (Views of one element: no memory.)"""
    with pytest.raises(RuntimeError, match="features"):
        ops.checkpoint8(torch.zeros(1).expand(n))
    with pytest.raises(RuntimeError, match="features"):
        ops.checkpoint8(torch.zeros(1, 1, dtype=torch.bfloat16).expand(2, n))
    npad = (n + 31) // 32 * 32
    kept = ops.Checkpoint8(torch.zeros(0, npad, dtype=torch.int8), torch.zeros(0, npad // 32, dtype=torch.uint8), (0, n), torch.float32)
    with pytest.raises(RuntimeError, match="features"):
        kept.restore()
    with pytest.raises(RuntimeError, match="features"):
        ops.checkpoint8_weight_grad(torch.zeros(0, 4), kept)
    few = ops.Checkpoint8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8), (6, 20), torch.float32)
    with pytest.raises(RuntimeError, match="features"):
        ops.checkpoint8_weight_grad(torch.zeros(1, 1).expand(6, n), few)
    with pytest.raises(RuntimeError, match="features"):
        ops.checkpoint8_weight_grad(torch.zeros(1, 1).expand(6, (1 << 20) + 1), few)


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 1])
def test_vertices_past_32_bits_are_refused(ops, n):
    """2^32 + 1 vertices of one graph read as 1 would take every vertex for a graph with an extent of its own.  (Views: no memory.)"""
    x = torch.zeros(1, 1, 1).expand(1, n, 1)
    with pytest.raises(RuntimeError, match="vertices"):
        ops.gated_residual_norms(x, x, n_valid=torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_residual_norms(x, x)


@pytest.mark.parametrize("change", [lambda k: k.codes.resize_(3, 32), lambda k: k.exps.resize_(0), lambda k: k.codes.t_(), lambda k: k.exps.t_(),
                                    lambda k: k.codes.untyped_storage().resize_(0), lambda k: k.exps.untyped_storage().resize_(5),
                                    lambda k: k.codes.unsqueeze_(0), lambda k: k.codes.as_strided_((6, 32), (1, 1)),
                                    lambda k: setattr(k.codes, "data", torch.zeros(6, 16, dtype=torch.int8))])
def test_a_checkpoint8_changed_in_place_is_refused(ops, change):
    """the kernels read both buffers by the activation's shape: out of range, once they are smaller"""
    kept = ops.Checkpoint8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8), (2, 3, 20), torch.float32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        kept.restore()
    change(kept)
    with pytest.raises(RuntimeError, match="do not hold"):
        kept.restore()
    with pytest.raises(RuntimeError, match="do not hold"):
        ops.checkpoint8_weight_grad(torch.zeros(2, 3, 4), kept)


def test_a_gnn_pickled_before_it_could_be_residual(ops, tmp_path):
    """whole modules saved by earlier versions have neither attribute: they are plain ones"""
    import schema_inference.graph as graph
    gnn = graph.GNN(10, 32, 2)
    del gnn.__dict__["residual"], gnn.__dict__["checkpoint8"]
    torch.save(gnn, tmp_path / "gnn.pt")
    back = torch.load(tmp_path / "gnn.pt", weights_only=False)
    assert back.train_folds() is False and back._mfma_ok() and not back.residual and not back.checkpoint8
    g = torch.Generator().manual_seed(0)
    nodes, edges, ids = torch.rand(2, 5, generator=g), torch.rand(2, 5, 5, generator=g), torch.randint(0, 10, (2, 5), generator=g)
    assert torch.equal(back(nodes, edges, ids), graph.GNN.forward(gnn, nodes, edges, ids))


PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "schemanet-pytorch_amd")
NUMBERS = """
import itertools, sys
sys.path.insert(0, sys.argv[1])
import cpp_extension
lib = cpp_extension.load()
rows = (-2**63, -2**31, -1, 0, 1, 2, 63, 64, 2**24 - 1, 2**24, 2**31 - 1, 2**31, 2**32, 2**40, 2**62, 2**63 - 1)
ints = (-2**31, -1, 0, 1, 31, 32, 33, 128, 256, 4096, 4097, 2**20, 2**20 + 1, 2**30, 2**31 - 1)
"""


def in_a_process(body):
    """(a division by zero ends the process that makes it)"""
    done = subprocess.run([sys.executable, "-c", NUMBERS + body, PACKAGE], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, (done.returncode, done.stdout[-300:], done.stderr[-300:])


def test_workspace_of_the_norms_at_any_numbers(ops):
    in_a_process("""
for r, w in itertools.product(rows, ints):
    size = lib.sn_block_norms_workspace(r, w)
    assert (size > 0) == (0 < r <= 2**48 and 1 <= w <= 4096) and size < 2**28, (r, w, size)
""")


def test_workspace_of_the_scores_at_any_numbers(ops):
    in_a_process("""
for r, n, k in itertools.product(rows, rows, ints):
    size = lib.sn_label_log_probs_workspace(r, n, k)
    assert size == 0 or (0 < r < 1024 and n > 8192 and 0 <= k <= 64 and size <= r * 64 * (4 + 2 * k) * 4), (r, n, k, size)
""")


def test_workspace_of_the_weight_gradient_at_any_numbers(ops):
    in_a_process("""
for r, o, i, t in itertools.product(rows, ints, ints, (-1, 0, 1, 2, 3)):
    size = lib.sn_checkpoint8_weight_grad_workspace(r, o, i, t)
    assert (size > 0) == (0 <= r < 2**31 and 1 <= o <= 2**20 and 1 <= i <= 2**20 and 0 <= t <= 2), (r, o, i, t, size)
    assert size == 0 or size <= 512 * 4 * (o + 1) * (i + 1) + 16, (r, o, i, t, size)
""")


@pytest.mark.parametrize("rows", [1 << 31, 1 << 32])
def test_rows_past_32_bits_are_refused(ops, rows):
    """the workspace of 2^32 rows divided by zero.  (Buffers on the meta device: no memory.)"""
    codes, exps = torch.empty(rows, 32, dtype=torch.int8, device="meta"), torch.empty(rows, 1, dtype=torch.uint8, device="meta")
    kept = ops.Checkpoint8(codes, exps, (rows, 7), torch.float32)
    with pytest.raises(RuntimeError, match="rows"):
        ops.checkpoint8_weight_grad(torch.zeros(1, 1).expand(rows, 5), kept)
