"""GPU tests of `ops.checkpoint8_weight_grad` at the sizes of its large tile (256 x 256: at least four such tiles and 512 rows of work for each
of 256 compute units) and around it: rows, outputs and inputs that end inside a tile, a last split of one row, strided gradients.

Sums of whole numbers: x holds -127 .. 127 with +-127 in every block of 32, so its step is 1 and it is kept exactly; dy holds -3 .. 3.  Every
partial sum is a whole number of at most 33000 * 127 * 3 < 2^24, exact in float32 in whatever order: a row, a column or a block
that is lost, taken twice or taken from its neighbour shows."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "schemanet-pytorch_amd"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

from blocks_plain import HALF, U, check, kept64  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
# (rows, out, in)
LARGE = [(32768, 512, 512),          # whole tiles, the least rows
         (32833, 512, 512),          # 57 splits of 576 rows and one of a single row
         (32833, 500, 490),          # ... with the last tiles moved back
         (32801, 513, 300), (16421, 515, 545), (43723, 257, 289), (14600, 1100, 288)]
NEXT_TO_IT = [(32767, 512, 512), (32833, 255, 512), (32833, 512, 224), (4097, 256, 256), (4160, 129, 161), (64, 128, 97), (63, 128, 128), (65, 300, 260)]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from cpp_extension import ops
    return ops


def whole_numbers(rows, out_f, in_f, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randint(-127, 128, (rows, in_f), generator=g, device=DEV).float()
    x[:, ::32] = torch.where(x[:, ::32] < 0, -127.0, 127.0)
    dy = torch.randint(-3, 4, (rows, out_f), generator=g, device=DEV).float()
    return x, dy.to(dtype), dy.double().t().contiguous() @ x.double(), dy.double().sum(0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,out_f,in_f", LARGE + NEXT_TO_IT)
def test_weight_grad_of_whole_numbers(ops, dtype, rows, out_f, in_f):
    x, dy, dw, db = whole_numbers(rows, out_f, in_f, dtype, rows + out_f + in_f)
    kept = ops.checkpoint8(x)
    got = ops.checkpoint8_weight_grad(dy, kept, out_dtype=F32)
    assert torch.equal(got[0].double(), dw) and torch.equal(got[1].double(), db)
    own = ops.checkpoint8_weight_grad(dy, kept)                     # rounded once, to dy's type
    assert own[0].dtype == dtype and torch.equal(own[0], dw.float().to(dtype)) and torch.equal(own[1], db.float().to(dtype))
    alone, none = ops.checkpoint8_weight_grad(dy, kept, bias=False, out_dtype=F32)
    assert none is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,out_f,in_f", [(32833, 500, 490), (4097, 256, 256)])
def test_weight_grad_of_strided_gradients(ops, dtype, rows, out_f, in_f):
    """rows further apart than their length, from an odd element on"""
    x, dy, dw, db = whole_numbers(rows, out_f, in_f, dtype, 3)
    wide = torch.full((rows, out_f + 5), float("nan"), dtype=dtype, device=DEV)
    wide[:, 3:out_f + 3] = dy
    got = ops.checkpoint8_weight_grad(wide[:, 3:out_f + 3], ops.checkpoint8(x), out_dtype=F32)
    assert torch.equal(got[0].double(), dw) and torch.equal(got[1].double(), db)


def test_weight_grad_of_rows_far_apart(ops):
    """2^22 elements from row to row: past the 32-bit offsets of the tiles"""
    x, dy, dw, db = whole_numbers(200, 140, 150, BF16, 4)
    far = torch.empty(200 << 22, dtype=BF16, device=DEV).as_strided((200, 140), (1 << 22, 1))
    far.copy_(dy)
    got = ops.checkpoint8_weight_grad(far, ops.checkpoint8(x), out_dtype=F32)
    assert torch.equal(got[0].double(), dw) and torch.equal(got[1].double(), db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,out_f,in_f", [(32833, 500, 490), (16421, 515, 545), (4097, 256, 256)])
def test_weight_grad_of_one_row_for_each_output(ops, dtype, rows, out_f, in_f):
    """every output's gradient is zero but for one row, among them the first and last rows of steps and splits: the bf16 pieces of that one
    value times a kept value, each product exact, added up with at most three roundings and rounded to the result"""
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(rows, in_f, generator=g, device=DEV)
    at = torch.randint(0, rows, (out_f,), generator=g, device=DEV)
    edges = [r for b in range(0, rows + 1, 64) for r in (b - 1, b) if 0 <= r < rows]
    at[:len(edges[-(out_f // 2):])] = torch.tensor(edges[-(out_f // 2):], device=DEV)
    value = (torch.randn(out_f, generator=g, device=DEV) * torch.exp2(torch.randint(-8, 8, (out_f,), generator=g, device=DEV).float())).to(dtype)
    dy = torch.zeros(rows, out_f, dtype=dtype, device=DEV)
    dy[at, torch.arange(out_f, device=DEV)] = value
    dw, db = ops.checkpoint8_weight_grad(dy, ops.checkpoint8(x), out_dtype=F32)
    want = value.double()[:, None] * kept64(x.double())[at]
    check(dw, want, (HALF[F32] + 3 * U) * want.abs() + 2.0 ** -140, "dW")
    assert torch.equal(db, value.float())


@pytest.mark.parametrize("dtype", TYPES)
def test_weight_grad_of_a_marked_block(ops, dtype):
    """an infinite activation marks its block of 32 in its row: those 32 inputs come out NaN for every output, no others"""
    x, dy, dw, _ = whole_numbers(32833, 500, 490, dtype, 6)
    x[32832, 480] = float("inf")                                    # the last split's only row, the last block
    got, _ = ops.checkpoint8_weight_grad(dy, ops.checkpoint8(x), out_dtype=F32)
    assert torch.isnan(got[:, 480:]).all() and torch.equal(got[:, :480].double(), dw[:, :480])


@pytest.mark.parametrize("rows,out_f,in_f", [(32833, 512, 496), (32833, 256, 256)])
def test_linear_checkpoint8_over_many_rows(ops, rows, out_f, in_f):
    """the Linear whose weight gradient takes the large tile"""
    x, dy, dw, db = whole_numbers(rows, out_f, in_f, F32, 7)
    w, b = torch.randn(out_f, in_f, device=DEV).requires_grad_(), torch.zeros(out_f, device=DEV).requires_grad_()
    got = torch.autograd.grad(ops.linear_checkpoint8(x, w, b), [w, b], dy)
    assert torch.equal(got[0].double(), dw) and torch.equal(got[1].double(), db)
