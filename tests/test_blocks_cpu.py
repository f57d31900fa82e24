"""CPU (-m "not gpu"): the second header and its binding, and what the operators of include/schemanet_blocks.h refuse.  No kernel
is launched: every call here is turned down before that."""
import ctypes
import os
import re
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
HEADER = os.path.join(ROOT, "include", "schemanet_blocks.h")


@pytest.fixture(scope="module")
def lib():
    import cpp_extension
    cpp_extension.build()
    return cpp_extension.load()


@pytest.fixture(scope="module")
def ops():
    from cpp_extension import ops
    return ops


def declarations():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_every_declared_symbol_is_bound(lib):
    import cpp_extension._native as N
    declared = set(re.findall(r"\b(sn_[a-z0-9_]+)\s*\(", declarations()))
    assert declared == set(N.BLOCK_SYMBOLS)
    assert all(hasattr(lib, s) for s in declared)
    assert lib.sn_blocks_abi_version() == N.BLOCKS_ABI_VERSION


def test_struct_matches_the_header(lib, tmp_path):
    import cpp_extension._native as N
    body = re.search(r"typedef struct sn_block_norms_args \{(.*?)\} sn_block_norms_args;", declarations(), re.S).group(1)
    names = []
    for statement in body.split(";"):
        fields = statement.strip()
        if fields:
            names += [re.findall(r"\w+", f)[-1] for f in fields.split(",")]
    assert names == [f[0] for f in N.BlockNormsArgs._fields_]
    src = tmp_path / "size.c"
    src.write_text('#include <stdio.h>\n#include "schemanet_blocks.h"\nint main(void) { printf("%zu", sizeof(sn_block_norms_args)); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "size")], check=True)
    size = int(subprocess.run([str(tmp_path / "size")], check=True, capture_output=True, text=True).stdout)
    assert ctypes.sizeof(N.BlockNormsArgs) == size and N.BlockNormsArgs().struct_size == size


def refused(rc, lib, word):
    assert rc < 0 and word in lib.sn_last_error().decode()


def test_c_entry_points_refuse(lib):
    import cpp_extension._native as N
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    refused(lib.sn_checkpoint8(p, 3, 1, 32, 32, p, p, None), lib, "type=3")
    refused(lib.sn_checkpoint8(p, 0, -1, 32, 32, p, p, None), lib, "rows=-1")
    refused(lib.sn_checkpoint8(p, 0, 1, 0, 32, p, p, None), lib, "n=0")
    refused(lib.sn_checkpoint8(None, 0, 1, 32, 32, p, p, None), lib, "NULL")
    assert lib.sn_checkpoint8(None, 0, 0, 32, 32, None, None, None) == 0                # no rows: nothing to do
    refused(lib.sn_checkpoint8_restore(p, None, 1, 32, p, 0, None), lib, "NULL")
    refused(lib.sn_checkpoint8_weight_grad(p, 0, 8, p, p, 0, 8, 8, p, p, 0, p, 4096, None), lib, "rows=0")
    refused(lib.sn_checkpoint8_weight_grad(p, 5, 8, p, p, 1, 8, 8, p, p, 0, p, 4096, None), lib, "type")
    refused(lib.sn_checkpoint8_weight_grad(p, 0, 8, p, p, 1, 8, 8, p, p, 0, p, 0, None), lib, "workspace")
    refused(lib.sn_checkpoint8_weight_grad(p, 0, 8, p, p, 1, 8, 8, None, p, 0, p, 4096, None), lib, "NULL")
    assert lib.sn_checkpoint8_weight_grad_workspace(-1, 8, 8, 0) == 0 and lib.sn_checkpoint8_weight_grad_workspace(100, 8, 8, 0) >= 16

    a = N.BlockNormsArgs()
    a.struct_size -= 8
    refused(lib.sn_block_norms_forward(ctypes.byref(a), None), lib, "struct_size")
    a = N.BlockNormsArgs()
    a.rows, a.width = 1, 4097
    refused(lib.sn_block_norms_forward(ctypes.byref(a), None), lib, "width 4097")
    a.width = 8
    refused(lib.sn_block_norms_forward(ctypes.byref(a), None), lib, "NULL")
    a.has_pre = 1
    refused(lib.sn_block_norms_forward(ctypes.byref(a), None), lib, "without weight")
    a.has_pre, a.x, a.branch, a.y, a.stats, a.dh, a.x_codes = 0, p, p, p, p, p, p
    refused(lib.sn_block_norms_forward(ctypes.byref(a), None), lib, "incomplete")
    a.x_codes = None
    refused(lib.sn_block_norms_backward(ctypes.byref(a), None), lib, "without the norm")
    a.dh, a.dy = None, p
    refused(lib.sn_block_norms_backward(ctypes.byref(a), None), lib, "workspace")
    a.n_valid, a.rows_per_graph = p, 0
    refused(lib.sn_block_norms_forward(ctypes.byref(a), None), lib, "rows_per_graph")
    refused(lib.sn_block_norms_forward(None, None), lib, "NULL")
    assert lib.sn_block_norms_workspace(10, 5000) == 0 and lib.sn_block_norms_workspace(10, 64) > 0

    refused(lib.sn_label_log_probs(p, 0, 1, 10, 10, p, -100, 11, p, p, p, p, p, p, 4096, None), lib, "11 alternatives")
    refused(lib.sn_label_log_probs(p, 0, 1, 100, 100, p, -100, 65, p, p, p, p, p, p, 4096, None), lib, "65 alternatives")
    refused(lib.sn_label_log_probs(p, 0, 1, 10, 10, p, -100, 2, p, p, p, None, p, p, 4096, None), lib, "NULL")
    refused(lib.sn_label_log_probs(p, 0, 1, 100000, 100000, p, -100, 0, p, p, p, None, None, p, 0, None), lib, "workspace")
    assert lib.sn_label_log_probs_workspace(1, 10, 3) == 0 and lib.sn_label_log_probs_workspace(1, 100000, 3) > 0
    refused(lib.sn_label_log_probs(p, 0, 1, 0, 10, p, -100, 0, p, p, p, None, None, p, 4096, None), lib, "n=0")
    refused(lib.sn_label_log_probs_backward(p, 0, 1, 10, 10, p, -100, p, None, None, p, None), lib, "NULL")
    assert lib.sn_label_log_probs(None, 0, 0, 10, 10, None, -100, 0, None, None, None, None, None, None, 0, None) == 0


def test_checkpoint8_refuses(ops):
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        ops.checkpoint8(torch.zeros(3, 4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="at least one feature"):
        ops.checkpoint8(torch.zeros(()))
    with pytest.raises(RuntimeError, match="at least one feature"):
        ops.checkpoint8(torch.zeros(3, 0))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.checkpoint8(torch.zeros(3, 4))
    kept = ops.Checkpoint8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8), (2, 3, 20), torch.float32)
    with pytest.raises(RuntimeError, match="cannot restore"):
        kept.restore(torch.int32)
    with pytest.raises(RuntimeError, match="do not fit"):
        ops.checkpoint8_weight_grad(torch.zeros(6, 5), kept)
    with pytest.raises(RuntimeError, match="do not fit"):
        ops.checkpoint8_weight_grad(torch.zeros(2, 4, 5), kept)
    with pytest.raises(RuntimeError, match="expected a Checkpoint8"):
        ops.checkpoint8_weight_grad(torch.zeros(6, 5), torch.zeros(6, 20))
    with pytest.raises(RuntimeError, match="gradients"):
        ops.checkpoint8_weight_grad(torch.zeros(2, 3, 5, dtype=torch.float64), kept)
    with pytest.raises(RuntimeError, match="cannot write"):
        ops.checkpoint8_weight_grad(torch.zeros(2, 3, 5), kept, out_dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.checkpoint8_weight_grad(torch.zeros(2, 3, 5), kept)


@pytest.mark.parametrize("codes,exps", [
    (torch.zeros(5, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8)),             # fewer rows
    (torch.zeros(7, 32, dtype=torch.int8), torch.zeros(7, 1, dtype=torch.uint8)),             # more
    (torch.zeros(6, 20, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8)),             # not padded
    (torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 0, dtype=torch.uint8)),
    (torch.zeros(6, 32, dtype=torch.int8), torch.zeros(3, 1, dtype=torch.uint8)),
    (torch.zeros(6, 64, dtype=torch.int8)[:, ::2], torch.zeros(6, 1, dtype=torch.uint8)),
    (torch.zeros(6, 32, dtype=torch.uint8), torch.zeros(6, 1, dtype=torch.uint8)),
    (torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1)),
])
def test_checkpoint8_of_another_layout_is_refused(ops, codes, exps):
    with pytest.raises(RuntimeError, match="do not hold"):
        ops.Checkpoint8(codes, exps, (2, 3, 20), torch.float32)


def test_a_checkpoint8_stays_whole(ops):
    kept = ops.Checkpoint8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8), (2, 3, 20), torch.float32)
    for name in ("codes", "exps", "shape"):
        with pytest.raises(AttributeError):
            setattr(kept, name, getattr(kept, name)[:1])
    with pytest.raises(RuntimeError, match="at least one feature"):
        ops.Checkpoint8(kept.codes, kept.exps, (6, 0), torch.float32)


def test_ce_entropy_loss_ignores_rows():
    """ignored rows count for nothing, whatever stands in them"""
    from schema_inference.loss import CEEntropyLoss
    x = torch.randn(6, 9, generator=torch.Generator().manual_seed(2))
    x[0, 3:5] = float("-inf")
    x[1], x[2, 0], x[4] = float("nan"), float("-inf"), float("-inf")
    label = torch.tensor([1, -100, -100, 4, -100, 8])
    used = label != -100
    leaf, alone = x.clone().requires_grad_(), x[used].clone().requires_grad_()
    got, want = CEEntropyLoss()({"pred": leaf}, {"label": label}), CEEntropyLoss()({"pred": alone}, {"label": label[used]})
    tol = 8 * 2.0 ** -24                                            # sums of three terms of size under 8, in another order
    assert all(abs(float((got[k] - want[k]).detach())) <= 8 * tol for k in ("cls", "entropy"))
    g1, = torch.autograd.grad(got["cls"] + got["entropy"], leaf)
    g2, = torch.autograd.grad(want["cls"] + want["entropy"], alone)
    assert not bool(g1[~used].any()) and float((g1[used] - g2).abs().max()) <= tol


def test_linear_checkpoint8_refuses(ops):
    x, w = torch.zeros(4, 32), torch.zeros(16, 32)
    with pytest.raises(RuntimeError, match="weight"):
        ops.linear_checkpoint8(x, torch.zeros(16, 31))
    with pytest.raises(RuntimeError, match="bias"):
        ops.linear_checkpoint8(x, w, torch.zeros(15))
    with pytest.raises(RuntimeError, match="float32"):
        ops.linear_checkpoint8(x.half(), w.half())
    with pytest.raises(RuntimeError, match="multiples of 16"):
        ops.linear_checkpoint8(torch.zeros(4, 30), torch.zeros(16, 30))
    with pytest.raises(RuntimeError, match="empty"):
        ops.linear_checkpoint8(torch.zeros(0, 32), w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_checkpoint8(x, w)


def test_gated_residual_norms_refuses(ops):
    x, v = torch.zeros(2, 3, 8), torch.ones(8)
    call = ops.gated_residual_norms
    for bad, word in ((dict(norm="batch"), "norm must be"), (dict(gate=torch.zeros(2, 3, 7)), "gate"), (dict(gate=x.half()), "gate"),
                      (dict(scale=torch.ones(7)), "parameters"), (dict(post=(v,)), "post"), (dict(pre=(None, v)), "pre"), (dict(pre=(v, v.double())), "parameters"),
                      (dict(eps=-1.0), "eps"), (dict(n_valid=torch.zeros(2)), "n_valid"), (dict(n_valid=torch.zeros(3, dtype=torch.int32)), "n_valid")):
        with pytest.raises(RuntimeError, match=word):
            call(x, x, **bad)
    with pytest.raises(RuntimeError, match="branch"):
        call(x, x[:1])
    with pytest.raises(RuntimeError, match="branch"):
        call(x, x.bfloat16())
    with pytest.raises(RuntimeError, match="branch"):
        call(x, None)
    with pytest.raises(RuntimeError, match="float32, bfloat16"):
        call(x.double(), x.double())
    with pytest.raises(RuntimeError, match="width 4097"):
        call(torch.zeros(1, 4097), torch.zeros(1, 4097))
    with pytest.raises(RuntimeError, match="n_valid"):
        call(x[0], x[0], n_valid=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call(x, x, post=(v, v))


def test_extents_that_are_not_a_tensor_are_refused(ops):
    with pytest.raises(RuntimeError, match="n_valid"):
        ops.gated_residual_norms(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), n_valid=[1, 2])


def test_label_log_probs_refuses(ops):
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    for args, word in (((x, t.int()), "target"), ((x, t[:1]), "target"), ((x.double(), t), "logits"), ((x, t, 6), "alternatives"),
                       ((x, t, -1), "alternatives"), ((torch.zeros(2, 100), t, 65), "alternatives"), ((torch.zeros(2, 0), t), "entries")):
        with pytest.raises(RuntimeError, match=word):
            ops.label_log_probs(*args)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.label_log_probs(x, t)


def test_the_plain_checkpoint_keeps_what_it_says():
    """the definition the GPU tests compare with: errors of at most max / 127.5 in a block, exact multiples kept, bf16 holds every value"""
    from blocks_plain import kept64
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 96, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-20, 20, (50, 96), generator=g).double())
    k = kept64(x)
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    assert bool(((k - x).unflatten(-1, (-1, 32)).abs() <= top / 127.5).all())
    assert torch.equal(k.bfloat16().double(), k)
    e = torch.randint(-127, 128, (50, 96), generator=g).double() / 64
    e[:, ::32] = 127 / 64
    assert torch.equal(kept64(e), e)
