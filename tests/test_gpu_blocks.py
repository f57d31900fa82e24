"""GPU tests of the operators of include/schemanet_blocks.h against their definitions in float64 (tests/blocks_plain.py).

Bounds.  U = 2^-24.  A result is rounded once to its type: HALF[type] of its value.  Before that it is float32 arithmetic, where
every operation is off by U of its result, so a formula of k roundings in a row is off by k U of the formula with absolute values
(the *_mag of Norms64).  k for the norms: a row sum is 8 additions in a lane, 6 in a wave and up to 7 over waves (21); the centred
squares the same again; reciprocal, root, division, sigmoid (expf 2, reciprocal 2), the affine steps and the sum: 20 at most; the
backward pass runs through both norms, forward and back, with a row sum in each: 4 x 21 + 40 -> K_ROW = 128.  A column sum adds as many
terms as there are rows in front of it, whatever the order: K_ROW + rows.  Subnormal results: the type's smallest step."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "schemanet-pytorch_amd"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

from blocks_plain import HALF, U, Norms64, check, kept64, scores64  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
K_ROW = 128
TINY = {F32: 2.0 ** -140, BF16: 2.0 ** -133, F16: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from cpp_extension import ops
    return ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(DEV)


def d64(t):
    return None if t is None else t.detach().double()


# ------------------------------------------------------------------------------------------------ 8-bit checkpoints
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (7, 33), (2, 3, 100), (1000, 256), (4099, 17), (3, 4096), (64,)])
def test_checkpoint8_restores_the_nearest_codes(ops, dtype, shape):
    g = gen(sum(shape))
    x = rand(g, *shape, dtype=dtype) * torch.exp(rand(g, *shape, std=2.0)).to(dtype)
    kept = ops.checkpoint8(x)
    assert kept.codes.dtype == torch.int8 and kept.nbytes == kept.codes.shape[0] * ((shape[-1] + 31) // 32) * 33
    want = kept64(d64(x))
    assert torch.equal(kept.restore(F32).double(), want)                       # exact in float32
    assert torch.equal(kept.restore(BF16).double(), want)                      # and in bfloat16
    own = kept.restore()
    assert own.dtype == dtype and own.shape == x.shape and torch.equal(own, want.to(dtype))
    top = torch.nn.functional.pad(d64(x), (0, (-shape[-1]) % 32)).unflatten(-1, (-1, 32)).abs().amax(-1)
    err = torch.nn.functional.pad((want - d64(x)).abs(), (0, (-shape[-1]) % 32)).unflatten(-1, (-1, 32)).amax(-1)
    assert bool((err <= top / 127.5).all())


def test_checkpoint8_values_at_the_edges(ops):
    step = 2.0 ** -3
    rows = [
        [127.0 * step, 0.5 * step, 1.5 * step, 2.5 * step, -0.5 * step, -1.5 * step],     # ties go to even codes
        [127.4 * step, -127.4 * step], [127.5 * step, 1.0 * step],                        # at 127.5 steps the step doubles
        [0.0, -0.0], [2.0 ** -149, 2.0 ** -130], [2.0 ** -126, 2.0 ** -120], [3.4e38, -1e38, 1.0], [3.4028234e38, -3.4028234e38],
        [float("inf"), 1.0], [1.0, float("nan")], [float("-inf"), 0.0],
    ]
    x = torch.zeros(len(rows), 40)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
        x[i, 35] = 3.0                                                                    # another block: untouched by its neighbour
    x = x.to(DEV)
    got = ops.checkpoint8(x).restore()
    want = kept64(d64(x))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.double().nan_to_num(), want.nan_to_num())
    assert torch.isnan(got[8, :32]).all() and float(got[8, 35]) == 3.0
    assert (got[4] == torch.where(torch.arange(40, device=DEV) == 35, 3.0, 0.0)).all()


def test_checkpoint8_strides_and_views(ops):
    g = gen(5)
    big = rand(g, 9, 13, 70)
    for x in (big[:, :, 3:45], big[::2, 1:, :33], big.transpose(0, 1), big[:, :, ::2], big[4, 3], big[:1].expand(6, 13, 70), big[:, :0]):
        got = ops.checkpoint8(x).restore()
        assert got.shape == x.shape and torch.equal(got, ops.checkpoint8(x.contiguous()).restore())
    assert torch.equal(ops.checkpoint8(big[:, :, 3:45]).restore().double(), kept64(d64(big[:, :, 3:45])))


GRAD_SIZES = [(1, 1, 1), (63, 5, 7), (64, 128, 128), (65, 129, 127), (257, 100, 40), (1000, 16, 300), (3001, 260, 132), (700, 1, 513)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,out_f,in_f", GRAD_SIZES)
def test_checkpoint8_weight_grad(ops, dtype, rows, out_f, in_f):
    """products of exact operands: the float32 sums are off by at most one rounding for each of the `rows` terms (and, for
    float32 gradients, 1 more for the part under the third bf16 piece)"""
    g = gen(rows + out_f)
    x = rand(g, rows, in_f)
    dy = rand(g, rows, out_f, dtype=dtype, std=0.02)
    kept = ops.checkpoint8(x)
    dw, db = ops.checkpoint8_weight_grad(dy, kept)
    assert dw.dtype == dtype and db.dtype == dtype and tuple(dw.shape) == (out_f, in_f) and tuple(db.shape) == (out_f,)
    kx, k = kept64(d64(x)), (rows + 4) * U
    want = d64(dy).t() @ kx
    check(dw, want, HALF[dtype] * want.abs() + k * (d64(dy).abs().t() @ kx.abs()) * (1 + HALF[dtype]) + TINY[dtype], "dW")
    wb = d64(dy).sum(0)
    check(db, wb, HALF[dtype] * wb.abs() + k * d64(dy).abs().sum(0) * (1 + HALF[dtype]) + TINY[dtype], "db")
    dw2, none = ops.checkpoint8_weight_grad(dy, kept, bias=False, out_dtype=F32)
    assert none is None and dw2.dtype == F32
    check(dw2, want, HALF[F32] * want.abs() + k * (d64(dy).abs().t() @ kx.abs()) + TINY[F32], "dW in float32")
    again, _ = ops.checkpoint8_weight_grad(dy, kept)
    assert torch.equal(again, dw)


def test_checkpoint8_weight_grad_small_and_large_gradients(ops):
    """float32 gradients over 60 powers of two: three bf16 pieces hold all of their bits"""
    g = gen(11)
    x = rand(g, 200, 48)
    dy = rand(g, 200, 36) * torch.exp2(torch.randint(-40, 20, (1, 36), generator=g).float()).to(DEV)
    kept = ops.checkpoint8(x)
    dw, db = ops.checkpoint8_weight_grad(dy, kept)
    kx = kept64(d64(x))
    want = d64(dy).t() @ kx
    check(dw, want, 205 * U * (d64(dy).abs().t() @ kx.abs()), "dW")
    check(db, d64(dy).sum(0), 205 * U * d64(dy).abs().sum(0), "db")
    x[7, 3] = float("inf")                                     # a block that cannot be kept poisons what it enters, nothing else
    dw, _ = ops.checkpoint8_weight_grad(dy, ops.checkpoint8(x))
    assert torch.isnan(dw[:, :32]).all() and torch.isfinite(dw[:, 32:]).all()


def test_checkpoint8_weight_grad_views(ops):
    g = gen(12)
    wide = rand(g, 6, 50, 90)
    x = rand(g, 6, 50, 64)
    kept = ops.checkpoint8(x)
    for dy in (wide[:, :, 5:41], wide[:, :, :1], wide[..., ::2], wide[:1].expand(6, 50, 90)):
        a, b = ops.checkpoint8_weight_grad(dy, kept)
        c, d = ops.checkpoint8_weight_grad(dy.contiguous(), kept)
        assert torch.equal(a, c) and torch.equal(b, d)
    a, b = ops.checkpoint8_weight_grad(wide[:, :0], ops.checkpoint8(x[:, :0]))
    assert not a.any() and not b.any() and a.shape == (90, 64)


@pytest.mark.parametrize("shape,out_f,bias", [((40, 32), 48, True), ((3, 50, 256), 256, True), ((2, 17, 64), 16, False)])
def test_linear_checkpoint8(ops, shape, out_f, bias):
    """the values and the input gradient of linear_mfma; the weight gradient is that of the kept input"""
    g = gen(out_f)
    x, w = rand(g, *shape).requires_grad_(), rand(g, out_f, shape[-1], std=0.2).requires_grad_()
    b = rand(g, out_f).requires_grad_() if bias else None
    leaves = [t for t in (x, w, b) if t is not None]
    up = rand(g, *shape[:-1], out_f, std=0.1)
    y = ops.linear_checkpoint8(x, w, b)
    y0 = ops.linear_mfma(x, w, b)
    assert torch.equal(y, y0)
    got, ref = torch.autograd.grad(y, leaves, up), torch.autograd.grad(y0, leaves, up)
    assert torch.equal(got[0], ref[0])
    kx, d = kept64(d64(x)).reshape(-1, shape[-1]), d64(up).reshape(-1, out_f)
    k = (d.shape[0] + 4) * U
    check(got[1], d.t() @ kx, k * (d.abs().t() @ kx.abs()), "dW")
    if bias:
        check(got[2], d.sum(0), k * d.abs().sum(0), "db")
    # an input that 8 bits hold exactly: the gradient of the layer itself
    xe = torch.randint(-100, 101, shape, generator=g).float().to(DEV) / 16
    ye = ops.linear_checkpoint8(xe, w, b)
    got = torch.autograd.grad(ye, [w], up)[0]
    check(got, d.t() @ d64(xe).reshape(-1, shape[-1]), k * (d.abs().t() @ d64(xe).abs().reshape(-1, shape[-1])), "dW of an exact input")


# ------------------------------------------------------------------------------------------------ gated residual norms
def norm_inputs(g, shape, dtype, gate=True, scale=True, post=True, pre=True, bias=True, params=None):
    E = shape[-1]
    params = params or dtype
    t = dict(x=rand(g, *shape, dtype=dtype, std=2.0, mean=0.5), branch=rand(g, *shape, dtype=dtype, mean=-0.3))
    t["gate"] = rand(g, *shape, dtype=dtype, std=2.0) if gate else None
    t["scale"] = rand(g, E, dtype=params, std=0.5, mean=1.0) if scale else None
    pair = lambda: (rand(g, E, dtype=params, std=0.3, mean=1.0), rand(g, E, dtype=params, std=0.3) if bias else None)       # noqa: E731
    t["post"], t["pre"] = pair() if post else None, pair() if pre else None
    return t


def check_norms(ops, t, norm, dtype, n_valid=None, dy=True, dh=True, keep8=False, eps=1e-5, seed=0):
    g = gen(seed + 99)
    shape, E = t["x"].shape, t["x"].shape[-1]
    flat = [t["x"], t["branch"], t["gate"], t["scale"], *(t["pre"] or ()), *(t["post"] or ())]
    leaves = [v.detach().requires_grad_() if v is not None else None for v in flat]
    it = iter(leaves)
    x, f, z, sc = (next(it) for _ in range(4))
    pre = (next(it), next(it)) if t["pre"] is not None else None
    post = (next(it), next(it)) if t["post"] is not None else None
    y, h = ops.gated_residual_norms(x, f, gate=z, scale=sc, post=post, pre=pre, norm=norm, eps=eps, n_valid=n_valid, checkpoint8=keep8)
    with torch.no_grad():
        y2, h2 = ops.gated_residual_norms(x, f, gate=z, scale=sc, post=post, pre=pre, norm=norm, eps=eps, n_valid=n_valid)
    assert torch.equal(y, y2) and (h is None) == (pre is None) and (h is None or torch.equal(h, h2))
    index = torch.arange(x.numel() // E, device=DEV)
    if n_valid is not None:
        index = index[(index % shape[1]) < n_valid.long()[index // shape[1]]]
    take = lambda v: None if v is None else d64(v).reshape(-1, E)[index]      # noqa: E731
    up_y = rand(g, *shape, dtype=dtype, std=0.1) if dy else None
    up_h = rand(g, *shape, dtype=dtype, std=0.1) if dh and pre is not None else None
    xs, fs, zs = take(x), take(f), take(z)
    kept = (kept64(xs), kept64(fs), None if zs is None else kept64(zs)) if keep8 else None
    pair = lambda p: None if p is None else (d64(p[0]), d64(p[1]))              # noqa: E731
    want = Norms64(xs, fs, zs, d64(sc), pair(post), pair(pre), norm, eps, take(up_y), take(up_h), kept)

    def rows(got, r, mag, what):
        full = torch.zeros(got.numel() // E, E, dtype=torch.float64, device=DEV)
        bound = full.clone()
        full[index] = r
        bound[index] = HALF[dtype] * r.abs() + K_ROW * U * mag * (1 + HALF[dtype]) + TINY[dtype]
        check(got.reshape(-1, E), full, bound, what)
    rows(y, want.y, want.y_mag, "y")
    if h is not None:
        rows(h, want.h, want.h_mag, "h")
    outs = [(y, up_y)] + ([(h, up_h)] if h is not None else [])
    outs = [(o, u) for o, u in outs if u is not None]
    asked = [v for v in leaves if v is not None]
    grads = dict(zip(map(id, asked), torch.autograd.grad([o for o, _ in outs], asked, [u for _, u in outs], allow_unused=True)))
    rows(grads[id(x)], want.dx, want.dx_mag, "dx")
    rows(grads[id(f)], want.dbranch, want.dbranch_mag, "dbranch")
    if z is not None:
        rows(grads[id(z)], want.dgate, want.dgate_mag, "dgate")

    def column(leaf, r, mag, what):
        if leaf is None:
            return
        got = grads[id(leaf)]
        assert got.dtype == leaf.dtype
        check(got, r, HALF[leaf.dtype] * r.abs() + (K_ROW + index.numel()) * U * mag * (1 + HALF[leaf.dtype]) + TINY[leaf.dtype], what)
    column(sc, want.dscale, want.dscale_mag, "dscale")
    if post is not None:
        column(post[0], want.dpost_w, want.dpost_w_mag, "dpost weight")
        column(post[1], want.dpost_b, want.dpost_b_mag, "dpost bias")
    if pre is not None and up_h is not None:
        column(pre[0], want.dpre_w, want.dpre_w_mag, "dpre weight")
        column(pre[1], want.dpre_b, want.dpre_b_mag, "dpre bias")
    elif pre is not None:
        assert not grads[id(pre[0])].any()


WIDTHS = [1, 5, 32, 63, 64, 100, 256, 257, 500, 512, 513, 1000, 1024, 1111, 2047, 2048, 2056, 4095, 4096]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", WIDTHS)
def test_norms_widths(ops, dtype, width):
    g = gen(width)
    check_norms(ops, norm_inputs(g, (11, width), dtype), "layer", dtype)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("parts", range(16))
def test_norms_every_set_of_parts(ops, norm, parts):
    gate, scale, post, pre = (bool(parts >> b & 1) for b in range(4))
    for dtype, width, rows, keep8 in ((F32, 96, 70, False), (BF16, 700, 9, True), (F32, 300, 33, True), (F16, 48, 5, False)):
        t = norm_inputs(gen(parts), (rows, width), dtype, gate, scale, post, pre, bias=(parts + rows) % 3 != 0)
        check_norms(ops, t, norm, dtype, keep8=keep8)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 300, 5000])
def test_norms_rows(ops, dtype, rows, keep8):
    check_norms(ops, norm_inputs(gen(rows), (rows, 256), dtype), "layer", dtype, keep8=keep8)


@pytest.mark.parametrize("dy,dh", [(True, False), (False, True)])
def test_norms_one_gradient_only(ops, dy, dh):
    check_norms(ops, norm_inputs(gen(1), (40, 130), F32), "layer", F32, dy=dy, dh=dh)
    check_norms(ops, norm_inputs(gen(1), (4, 10, 130), BF16), "rms", BF16, dy=dy, dh=dh, keep8=True,
                n_valid=torch.tensor([10, 0, 3, 1], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("width", [33, 256, 600, 2500])
def test_norms_graphs_with_padding(ops, width, keep8):
    """vertices behind a graph's last one are neither read (NaN there stays there) nor given a gradient"""
    g = gen(width)
    n_valid = torch.tensor([7, 0, 1, 12, 5], dtype=torch.int32, device=DEV)
    t = norm_inputs(g, (5, 12, width), F32)
    pad = torch.arange(12, device=DEV)[None, :] >= n_valid[:, None]
    for k in ("x", "branch", "gate"):
        t[k] = t[k].masked_fill(pad[..., None], float("nan"))
    check_norms(ops, t, "layer", F32, n_valid=n_valid, keep8=keep8)


def test_norms_parameters_of_other_types(ops):
    check_norms(ops, norm_inputs(gen(3), (20, 200), BF16, params=F32), "layer", BF16)
    check_norms(ops, norm_inputs(gen(3), (20, 200), F16, params=F32), "rms", F16, keep8=True)
    t = norm_inputs(gen(3), (20, 200), BF16)
    t["scale"] = t["scale"].float()                                                # mixed: taken in float32
    check_norms(ops, t, "layer", BF16)


def test_norms_strided_inputs(ops):
    g = gen(21)
    big = [rand(g, 6, 10, 300) for _ in range(3)]
    t = norm_inputs(g, (6, 10, 128), F32)
    for cut in (lambda v: v[:, :, 7:135], lambda v: v[:, :, 0:256:2], lambda v: v[:1, :, 9:137].expand(6, 10, 128), lambda v: v[:, 2:3, 1:129].expand(6, 10, 128)):
        s = dict(t, x=cut(big[0]), branch=cut(big[1]), gate=cut(big[2]))
        check_norms(ops, s, "layer", F32)
        check_norms(ops, s, "layer", F32, keep8=True, n_valid=torch.tensor([3, 10, 0, 1, 9, 10], dtype=torch.int32, device=DEV))


def test_norms_extreme_rows(ops):
    """constant rows (no variance), a large common offset, gates at both ends, zero rows"""
    t = norm_inputs(gen(8), (6, 96), F32)
    t["x"][0] = 3.0
    t["branch"][0] = -7.0
    t["branch"][1] += 1000.0
    t["gate"][2] = 200.0
    t["gate"][3] = -200.0
    t["x"][4], t["branch"][4] = 0.0, 0.0
    with torch.no_grad():
        y, h = ops.gated_residual_norms(t["x"], t["branch"], gate=t["gate"], scale=t["scale"], post=t["post"], pre=t["pre"])
    want = Norms64(d64(t["x"]), d64(t["branch"]), d64(t["gate"]), d64(t["scale"]), tuple(map(d64, t["post"])), tuple(map(d64, t["pre"])), "layer", 1e-5)
    check(y, want.y, K_ROW * U * want.y_mag + TINY[F32], "y")
    check(h, want.h, K_ROW * U * want.h_mag + TINY[F32], "h")
    t["gate"][2, 5], t["x"][3, 7] = float("nan"), float("inf")
    with torch.no_grad():
        y, h = ops.gated_residual_norms(t["x"], t["branch"], gate=t["gate"], scale=t["scale"], post=t["post"], pre=t["pre"])
    assert torch.isnan(y[2, 5]) and int(torch.isnan(y).sum()) == 1 and torch.isinf(y[3, 7])
    assert torch.isnan(h[2]).all() and torch.isfinite(h[[0, 1, 4, 5]]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norms_closed_and_open_gates(ops, dtype):
    """gates at the ends of their type, infinities among them: sigmoid 0 or 1 exactly, a gradient of 0 for the gate"""
    t = norm_inputs(gen(17), (4, 300), dtype)
    t["gate"][0], t["gate"][1] = float("inf"), float("-inf")
    t["gate"][2], t["gate"][3] = 88.5, -200.0
    x, z = t["x"].clone().requires_grad_(), t["gate"].clone().requires_grad_()
    y, h = ops.gated_residual_norms(x, t["branch"], gate=z, scale=t["scale"], post=t["post"], pre=t["pre"])
    want = Norms64(d64(t["x"]), d64(t["branch"]), d64(t["gate"]), d64(t["scale"]), tuple(map(d64, t["post"])), tuple(map(d64, t["pre"])), "layer", 1e-5)
    check(y, want.y, HALF[dtype] * want.y.abs() + K_ROW * U * want.y_mag * 2 + TINY[dtype], "y")
    check(h, want.h, HALF[dtype] * want.h.abs() + K_ROW * U * want.h_mag * 2 + TINY[dtype], "h")
    assert torch.equal(y[1], t["x"][1])
    dz, dx = torch.autograd.grad((y.float().sum() + h.float().sum()), [z, x])
    assert not dz[:2].any() and torch.isfinite(dx).all() and torch.isfinite(dz).all()


@pytest.mark.parametrize("n_valid", [[0, 0, 0], [-1, 7, 100], [3, 0, 4]])
def test_norms_extents_outside_the_graph(ops, n_valid):
    """no vertex at all, and extents beyond the padded length (= every vertex) or below zero (= none)"""
    t = norm_inputs(gen(18), (3, 5, 70), F32)
    nv = torch.tensor(n_valid, dtype=torch.int32, device=DEV)
    check_norms(ops, t, "layer", F32, n_valid=nv.clamp(0, 5))
    y, h = ops.gated_residual_norms(t["x"], t["branch"], gate=t["gate"], pre=t["pre"], n_valid=nv)
    y2, h2 = ops.gated_residual_norms(t["x"], t["branch"], gate=t["gate"], pre=t["pre"], n_valid=nv.clamp(0, 5))
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("keep8", [False, True])
def test_norms_gradient_against_differences(ops, keep8):
    """the derivative along a direction from central differences of the float64 definition; with 8-bit checkpoints the inputs are such
    that 8 bits hold them.  Differences err by h^2 (h = 1e-4: third derivatives of order 10 -> 1e-7 of the slope's scale), the
    gradients by the K_ROW roundings of each of the terms added up."""
    g = gen(31)
    E, R = 64, 12
    q = lambda: (torch.randint(-60, 61, (R, E), generator=g).float() / 32).to(DEV)         # noqa: E731
    t = norm_inputs(g, (R, E), F32)
    t.update(x=q(), branch=q(), gate=q())
    names = ["x", "branch", "gate", "scale"]
    leaf = {k: t[k].clone().requires_grad_() for k in names}
    post = tuple(v.clone().requires_grad_() for v in t["post"])
    pre = tuple(v.clone().requires_grad_() for v in t["pre"])
    y, h = ops.gated_residual_norms(leaf["x"], leaf["branch"], gate=leaf["gate"], scale=leaf["scale"], post=post, pre=pre, checkpoint8=keep8)
    uy, uh = rand(g, R, E, std=0.1), rand(g, R, E, std=0.1)
    leaves = [leaf[k] for k in names] + list(post) + list(pre)
    grads = torch.autograd.grad([y, h], leaves, [uy, uh])
    base = [d64(v) for v in leaves]

    def value(vs):
        r = Norms64(vs[0], vs[1], vs[2], vs[3], (vs[4], vs[5]), (vs[6], vs[7]), "layer", 1e-5)
        return float((r.y * d64(uy)).sum() + (r.h * d64(uh)).sum())
    for i, gi in enumerate(grads):
        v = rand(g, *base[i].shape).double()
        eps = 1e-4
        plus = value([b + eps * v if j == i else b for j, b in enumerate(base)])
        minus = value([b - eps * v if j == i else b for j, b in enumerate(base)])
        slope, got = (plus - minus) / (2 * eps), float((gi.double() * v).sum())
        scale = float((gi.double() * v).abs().sum())
        assert abs(got - slope) <= (K_ROW + R) * U * scale * 4 + 1e-6 * scale, (i, got, slope)


# ------------------------------------------------------------------------------------------------ log probabilities
def score_bounds(x, target, lp_all, ent):
    """a lane adds up at most n / 64 + 8 terms one by one, joins add 8 more; exp is off by 2 U and U |d| (d = x - max, weighted by
    exp(-|d|)): s and t are off by A U with A = n / 64 + 64, relative to sums of absolute values"""
    a = x.shape[-1] / 64 + 64
    d = (x - x.amax(-1, keepdim=True)).clamp(min=-1e30).abs()
    p = torch.exp(lp_all)
    spread = torch.where(p > 0, p * d, torch.zeros_like(p)).sum(-1)
    logs = torch.log(torch.exp(x - x.amax(-1, keepdim=True)).sum(-1)).abs()
    return a, d, p, spread, logs


def check_scores(ops, x, target, topk=0, grads=True, ignore=-100, seed=0):
    leaf = x.detach().requires_grad_(grads)
    got = ops.label_log_probs(leaf, target, topk=topk, ignore_index=ignore)
    n = x.shape[-1]
    x2, t2 = d64(x).reshape(-1, n), target.reshape(-1)
    lp, ent, lp_all = scores64(x2, t2, ignore)
    a, d, p, spread, logs = score_bounds(x2, t2, lp_all, ent)
    base = a * U * (1 + logs + spread)
    d_t = d.gather(-1, t2.clamp(0, n - 1)[:, None])[:, 0]
    check(got.log_probs.reshape(-1), lp, base + 4 * U * d_t.clamp(max=1e30), "log_probs")
    check(got.entropy.reshape(-1), ent, base * 2, "entropy")
    if topk:
        order = torch.sort(x2, dim=-1, descending=True, stable=True).indices[:, :topk]
        assert torch.equal(got.top_ids.reshape(-1, topk), order)
        want = lp_all.gather(-1, order)
        check(got.top_log_probs.reshape(-1, topk), want, base[:, None] + 4 * U * d.gather(-1, order).clamp(max=1e30), "top_log_probs")
        assert not got.top_ids.requires_grad and not got.top_log_probs.requires_grad
    else:
        assert got.top_ids is None and got.top_log_probs is None
    if not grads:
        return
    g = gen(seed)
    u1, u2 = rand(g, *target.shape), rand(g, *target.shape)
    grad, = torch.autograd.grad((got.log_probs, got.entropy), leaf, (u1, u2))
    assert grad.dtype == x.dtype
    used = (t2 != ignore).double()
    g1, g2 = d64(u1).reshape(-1) * used, d64(u2).reshape(-1)
    finite = torch.where(p > 0, lp_all, torch.zeros_like(p))
    want = -p * (g1[:, None] + g2[:, None] * (finite + ent[:, None]))
    want.scatter_add_(-1, t2.clamp(0, n - 1)[:, None], g1[:, None])
    mag = p * (g1.abs()[:, None] + g2.abs()[:, None] * (finite.abs() + ent[:, None] + logs[:, None] + spread[:, None] + 1))
    dead = torch.isinf(lp_all).all(-1, keepdim=True)
    want = torch.where(dead, torch.zeros_like(want), want)
    bound = HALF[x.dtype] * want.abs() + (a + 16 + (d.clamp(max=200) if x.dtype != F32 else 4)) * U * (mag + want.abs()) + TINY[x.dtype] * 4
    check(grad.reshape(-1, n), want, bound, "gradient")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (5, 7), (4, 100), (9, 512), (3, 1000), (2, 2048), (3, 2049), (2, 5001), (5, 32769), (1, 131072), (700, 4100), (3, 8192), (3, 8193), (2048, 2100), (2100, 5001),
                                     (2047, 16385)])
def test_scores_sizes(ops, dtype, rows, n):
    g = gen(rows * 7 + n)
    x = rand(g, rows, n, dtype=dtype, std=3.0)
    target = torch.randint(0, n, (rows,), generator=g).to(DEV)
    check_scores(ops, x, target, topk=min(n, 5))
    check_scores(ops, x, target)


@pytest.mark.parametrize("topk", [1, 2, 13, 32, 63, 64])
@pytest.mark.parametrize("n", [64, 700, 9000, 70001])
def test_scores_alternatives(ops, topk, n):
    g = gen(topk + n)
    target = torch.randint(0, n, (6,), generator=g).to(DEV)
    x = rand(g, 6, n, std=2.0)
    check_scores(ops, x, target, topk, grads=False)
    check_scores(ops, x.bfloat16(), target, topk, grads=False)                      # many equal values
    check_scores(ops, (x > 1).float(), target, topk, grads=False)                   # two values
    check_scores(ops, torch.zeros_like(x), target, topk, grads=False)               # one value: ids 0 .. k - 1
    check_scores(ops, torch.arange(n, dtype=F32, device=DEV).expand(6, n) / n, target, topk, grads=False)      # ascending: the list changes all the time
    check_scores(ops, -torch.arange(n, dtype=F32, device=DEV).expand(6, n) / n, target, topk, grads=False)


@pytest.mark.parametrize("n", [10, 1500, 6000, 50000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_masks(ops, dtype, n):
    """-inf entries, rows with one entry left, rows with none, the type's lowest value, ignored and masked targets"""
    g = gen(n)
    x = rand(g, 8, n, dtype=dtype, std=2.0)
    x[0, n // 2:] = float("-inf")
    x[1] = float("-inf")
    x[1, n - 1] = -5.0
    x[2] = float("-inf")                                                            # nothing left
    x[3] = torch.finfo(dtype).min                                                   # all equal: a uniform distribution
    x[4, 1:] = torch.finfo(dtype).min
    x[5] = x[5] * 0 + torch.finfo(dtype).max / 4
    target = torch.randint(0, n // 2, (8,), generator=g).to(DEV)
    target[0] = n - 1                                                               # a masked target: -inf
    target[1] = n - 1
    target[6] = -100
    check_scores(ops, x, target, topk=7)
    got = ops.label_log_probs(x, target, topk=3)
    assert float(got.log_probs[0]) == float("-inf") and float(got.entropy[2]) == 0.0 and float(got.log_probs[2]) == float("-inf")
    assert got.top_ids[2].tolist() == [0, 1, 2] and got.top_ids[1].tolist() == [n - 1, 0, 1] and float(got.log_probs[6]) == 0.0


@pytest.mark.parametrize("topk", [1, 7, 64])
@pytest.mark.parametrize("n", [300, 2000, 7000, 16000, 60000])
def test_scores_few_entries_left(ops, n, topk):
    """constrained answers: a few entries far apart, more and fewer of them than alternatives"""
    g = gen(n + topk)
    rows = 12
    x = torch.full((rows, n), float("-inf"))
    for r in range(rows):
        left = torch.randperm(n, generator=g)[:[1, 2, 3, 5, 6, 7, 8, 9, 40, 63, 64, 100][r]]
        x[r, left] = torch.randn(len(left), generator=g)
    target = x.argmax(-1)
    check_scores(ops, x.to(DEV), target.to(DEV), topk=topk)


def test_scores_most_parts_with_most_alternatives(ops):
    """rows so long that 64 workgroups share one"""
    g = gen(3)
    x = rand(g, 2, 300000, std=2.0)
    check_scores(ops, x, x.argmin(-1), topk=64)
    check_scores(ops, (x > 3).float(), x.argmin(-1), topk=64)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [9, 3000, 20000])
def test_scores_rows_without_a_part_in_the_loss(ops, dtype, n):
    """ignored rows, NaN or infinite as padding may be, get zeros; the others what they get alone"""
    g = gen(n)
    x = rand(g, 6, n, dtype=dtype, std=2.0)
    x[1] = float("nan")
    x[3] = float("inf")
    x[4] = float("-inf")
    target = torch.randint(0, n, (6,), generator=g).to(DEV)
    target[[1, 3, 4]] = -100
    used = target != -100
    leaf, alone = x.clone().requires_grad_(), x[used].clone().requires_grad_()
    got, part = ops.label_log_probs(leaf, target), ops.label_log_probs(alone, target[used])
    grad, = torch.autograd.grad(got.log_probs.sum() + got.entropy.masked_fill(~used, 0.0).sum(), leaf)
    want, = torch.autograd.grad(part.log_probs.sum() + part.entropy.sum(), alone)
    assert not bool(grad[~used].any()) and torch.equal(grad[used], want)
    assert torch.equal(got.log_probs[used], part.log_probs) and not bool(got.log_probs[~used].any())


@pytest.mark.parametrize("n", [40, 5000, 40000])
def test_scores_not_a_number(ops, n):
    g = gen(n)
    x = rand(g, 5, n, std=2.0)
    x[1, 3] = float("nan")
    x[2] = float("nan")
    x[3, n - 2] = float("inf")
    target = torch.tensor([0, 1, 2, 3, n], device=DEV)                              # the last one lies outside
    leaf = x.clone().requires_grad_()
    got = ops.label_log_probs(leaf, target, topk=4)
    lp, ent = got.log_probs.tolist(), got.entropy.tolist()
    assert all(v != v for v in lp[1:]) and lp[0] == lp[0] and all(v != v for v in ent[1:4]) and ent[4] == ent[4]
    assert got.top_ids[2].tolist() == [-1] * 4 and int(got.top_ids[3, 0]) == n - 2
    clean = x[1].clone()
    clean[3] = float("-inf")
    assert got.top_ids[1].tolist() == torch.topk(clean, 4).indices.tolist() and torch.isnan(got.top_log_probs[1]).all()
    grad, = torch.autograd.grad(got.log_probs.sum(), leaf)
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[2]).all() and torch.isnan(grad[4]).all()


def test_scores_shapes_strides_and_one_gradient(ops):
    g = gen(77)
    big = rand(g, 4, 6, 3000)
    target = torch.randint(0, 200, (4, 6), generator=g).to(DEV)
    for x in (big[:, :, 5:305], big[:, :, :2600:2], big.transpose(0, 1)[:4, :4], big[:1, :, 1:500].expand(4, 6, 499), big[:, :, 1:2500]):
        check_scores(ops, x, target[:x.shape[0], :x.shape[1]], topk=3)
    x = big[:, :, 1:301].detach().requires_grad_()
    got = ops.label_log_probs(x, target)
    a, = torch.autograd.grad(got.log_probs.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(got.entropy.sum(), x, retain_graph=True)
    both, = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), x)
    torch.testing.assert_close(a + b, both, rtol=0, atol=8 * U)                     # three results of size <= 1, each off by a few U
    empty = ops.label_log_probs(big[:, :0, :10], target[:, :0], topk=2)
    assert empty.log_probs.shape == (4, 0) and empty.top_ids.shape == (4, 0, 2)
    single = ops.label_log_probs(big[0, 0], target[0, 0], topk=1)
    assert single.log_probs.shape == () and int(single.top_ids[0]) == int(big[0, 0].argmax())


def test_scores_gradient_against_differences(ops):
    """central differences of the float64 definition along a direction: error h^2 = 1e-8 of the slope's scale"""
    g = gen(41)
    x = rand(g, 7, 300, std=2.0).requires_grad_()
    target = torch.randint(0, 300, (7,), generator=g).to(DEV)
    u1, u2, v = rand(g, 7), rand(g, 7), rand(g, 7, 300).double()
    got = ops.label_log_probs(x, target)
    grad, = torch.autograd.grad((got.log_probs, got.entropy), x, (u1, u2))

    def value(t):
        lp, ent, _ = scores64(t, target)
        return float((lp * d64(u1)).sum() + (ent * d64(u2)).sum())
    slope = (value(d64(x) + 1e-4 * v) - value(d64(x) - 1e-4 * v)) / 2e-4
    scale = float((grad.double() * v).abs().sum())
    assert abs(float((grad.double() * v).sum()) - slope) <= scale * (80 * U + 1e-6)


# ------------------------------------------------------------------------------------------------ as a program uses them
def training_step(ops, t):
    """a residual block and its loss: Linear with a kept input, the block's end with kept inputs, scores"""
    f = ops.linear_checkpoint8(t["x"], t["w"], t["b"])
    y, h = ops.gated_residual_norms(t["x"], f, gate=t["gate"], scale=t["scale"], post=(t["pw"], t["pb"]), pre=(t["qw"], t["qb"]), n_valid=t["n_valid"],
                                    checkpoint8=True)
    logits = ops.linear_checkpoint8(h, t["head"])
    got = ops.label_log_probs(logits, t["target"])
    used = (t["target"] != -100).float()
    loss = -(got.log_probs.sum() + 0.1 * (got.entropy * used).sum()) / used.sum() + 1e-3 * y.square().mean()
    leaves = [t[k] for k in ("x", "w", "b", "gate", "scale", "pw", "pb", "qw", "qb", "head")]
    return (loss,) + torch.autograd.grad(loss, leaves)


def step_inputs(seed, G=3, n=40, E=64, K=48):
    g = gen(seed)
    t = dict(x=rand(g, G, n, E), w=rand(g, E, E, std=0.2), b=rand(g, E, std=0.1), gate=rand(g, G, n, E), scale=rand(g, E, std=0.1, mean=0.5),
             pw=rand(g, E, mean=1.0, std=0.1), pb=rand(g, E, std=0.1), qw=rand(g, E, mean=1.0, std=0.1), qb=rand(g, E, std=0.1), head=rand(g, K, E, std=0.3))
    for v in t.values():
        v.requires_grad_()
    t["n_valid"] = torch.tensor([n, 7, 23][:G], dtype=torch.int32, device=DEV)
    target = torch.randint(0, K, (G, n), generator=g).to(DEV)
    t["target"] = torch.where(torch.arange(n, device=DEV)[None] < t["n_valid"][:, None], target, -100)
    return t


def test_a_training_step_of_all_of_them(ops):
    """block, kept activations and loss together, against autograd in float64 at inputs the 8 bits hold exactly.  x and gate are
    exact multiples; the branch and the head's input are computed, so those are kept with an error of at most step / 2 <= max / 127.5:
    the gradients agree to a few hundredths of their norm, and exactly in what does not see a rounded value."""
    t = step_inputs(1)
    exact = lambda v: (v.detach() * 16).round().clamp(-100, 100).div(16).requires_grad_()       # noqa: E731
    t["x"], t["gate"] = exact(t["x"]), exact(t["gate"])
    got = training_step(ops, t)
    ref = {k: (v.detach().double().requires_grad_(v.requires_grad) if v.is_floating_point() else v) for k, v in t.items()}
    live = (torch.arange(40, device=DEV)[None] < t["n_valid"][:, None])[..., None]
    f = torch.nn.functional.linear(ref["x"], ref["w"], ref["b"])
    ln = lambda v, w, b: torch.nn.functional.layer_norm(v, (64,), w, b, 1e-5)                    # noqa: E731
    y = (ref["x"] + ref["scale"] * torch.sigmoid(ref["gate"]) * ln(f, ref["pw"], ref["pb"])) * live
    h = ln(y, ref["qw"], ref["qb"]) * live
    lp = torch.log_softmax(h @ ref["head"].t(), -1)
    used = (t["target"] != -100).double()
    picked = lp.gather(-1, t["target"].clamp(min=0)[..., None])[..., 0] * used
    ent = -(lp.exp() * lp).sum(-1) * used
    loss = -(picked.sum() + 0.1 * ent.sum()) / used.sum() + 1e-3 * y.square().mean()
    want = torch.autograd.grad(loss, [ref[k] for k in ("x", "w", "b", "gate", "scale", "pw", "pb", "qw", "qb", "head")])
    assert abs(float(got[0].detach()) - float(loss.detach())) <= 1e-5 * abs(float(loss.detach()))
    for a, b in zip(got[1:], want):
        assert float((a.double() - b).norm() / b.norm()) < 0.05


def test_captured_step_replays_like_an_eager_one(ops):
    a, b = step_inputs(2), step_inputs(3)
    eager = [[v.detach().clone() for v in training_step(ops, t)] for t in (a, b)]
    assert all(torch.equal(x, y) for x, y in zip(eager[0], [v.detach() for v in training_step(ops, a)]))     # the same bits every time
    static = {k: v.detach().clone().requires_grad_(v.requires_grad) for k, v in a.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            training_step(ops, static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = training_step(ops, static)
    for turn in range(4):
        src = (a, b)[turn % 2]
        with torch.no_grad():
            for k, v in static.items():
                v.copy_(src[k])
        graph.replay()
        torch.cuda.synchronize()
        scratch = torch.full((1 << 20,), float(turn), device=DEV).sum()             # eager work between the replays
        for x, y in zip(out, eager[turn % 2]):
            assert torch.equal(x.detach(), y), turn
        del scratch


def test_captured_operators_one_by_one(ops):
    g = gen(4)
    x, dy = rand(g, 500, 96), rand(g, 500, 80)
    logits = rand(g, 6, 20000, dtype=BF16, std=2.0)
    target = torch.randint(0, 20000, (6,), generator=g).to(DEV)

    def run():
        kept = ops.checkpoint8(x)
        return [*ops.checkpoint8_weight_grad(dy, kept), kept.restore(), *ops.label_log_probs(logits, target, topk=9)]
    want = run()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(4):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_other_streams(ops):
    """called on a side stream, the results are those of the current one; two streams at once do not disturb each other"""
    t = step_inputs(5)
    want = [v.detach().clone() for v in training_step(ops, t)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(training_step(ops, t))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for out in outs:
        assert all(torch.equal(a.detach(), b) for a, b in zip(out, want))


def test_autocast_computes_in_float32(ops):
    g = gen(6)
    t = norm_inputs(g, (10, 64), F32)
    logits, target = rand(g, 5, 50), torch.randint(0, 50, (5,), generator=g).to(DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, h = ops.gated_residual_norms(t["x"], t["branch"].bfloat16(), post=t["post"], pre=t["pre"])
        got = ops.label_log_probs(logits.bfloat16(), target)
        z = ops.linear_checkpoint8(t["x"].bfloat16(), t["branch"][:, :64].contiguous()[:, :64].repeat(2, 1)[:16])
    y2, h2 = ops.gated_residual_norms(t["x"], t["branch"].bfloat16().float(), post=t["post"], pre=t["pre"])
    assert y.dtype == F32 and torch.equal(y, y2) and torch.equal(h, h2) and z.dtype == F32
    assert torch.equal(got.log_probs, ops.label_log_probs(logits.bfloat16().float(), target).log_probs)


def test_only_what_is_asked_for(ops):
    """gradients of some inputs only, an unused result, no second derivatives"""
    t = norm_inputs(gen(9), (20, 100), F32)
    x = t["x"].clone().requires_grad_()
    y, h = ops.gated_residual_norms(x, t["branch"], gate=t["gate"], post=t["post"], pre=t["pre"])
    full = torch.autograd.grad((y * y).sum(), x)[0]
    w = t["post"][0].clone().requires_grad_()
    y2, _ = ops.gated_residual_norms(x, t["branch"], gate=t["gate"], post=(w, t["post"][1]), pre=t["pre"])
    gw, = torch.autograd.grad((y2 * y2).sum(), w)
    assert gw.shape == w.shape and torch.equal(full, 2 * y.detach())               # dL/dy = 2 y passes straight to x
    leaf = rand(gen(1), 3, 20).requires_grad_()
    got = ops.label_log_probs(leaf, torch.zeros(3, dtype=torch.int64, device=DEV))
    first, = torch.autograd.grad(got.log_probs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)
    y, h = ops.gated_residual_norms(torch.empty(0, 8, device=DEV).requires_grad_(), torch.empty(0, 8, device=DEV), pre=(torch.ones(8, device=DEV), None))
    assert y.shape == (0, 8) and h.shape == (0, 8)
    y.sum().backward()


def both(ops, t, keep8=False):
    """-> leaves and the results of both differentiable operators"""
    leaves = [v.clone().requires_grad_() for v in (t["x"], t["branch"], t["gate"], t["scale"], *t["post"], *t["pre"])]
    x, branch, gate, scale, pw, pb, w, b = leaves
    y, h = ops.gated_residual_norms(x, branch, gate=gate, scale=scale, post=(pw, pb), pre=(w, b), checkpoint8=keep8)
    got = ops.label_log_probs(h, torch.arange(h.shape[0], device=DEV) % h.shape[1])
    return leaves, [y, got.log_probs, got.entropy]


def grads_of(leaves, out, **how):
    return torch.autograd.grad(out, leaves, [torch.ones_like(o) * (i + 1) for i, o in enumerate(out)], **how)


@pytest.mark.parametrize("keep8", [False, True])
def test_backward_twice_and_through_hooks(ops, keep8):
    """a kept graph gives the same gradients again, a freed one raises; what is saved goes through the hooks for saved tensors"""
    t = norm_inputs(gen(31), (40, 200), F32)
    leaves, out = both(ops, t, keep8)
    first = grads_of(leaves, out, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, grads_of(leaves, out)))
    with pytest.raises(RuntimeError, match="second time"):
        grads_of(leaves, out)
    with torch.autograd.graph.save_on_cpu():
        leaves, out = both(ops, t, keep8)
    assert all(torch.equal(a, b) for a, b in zip(first, grads_of(leaves, out)))
    leaves, out = both(ops, t, keep8)
    for o, leaf in ((out, leaves),):
        torch.autograd.backward(o, [torch.ones_like(v) * (i + 1) for i, v in enumerate(o)])
        assert all(torch.equal(a, v.grad) for a, v in zip(first, leaf))
    seen = []
    leaves, out = both(ops, t, keep8)
    leaves[0].register_hook(lambda g: seen.append(g.clone()))
    grads_of(leaves, out)
    assert torch.equal(seen[0], first[0])


def test_inputs_changed_before_the_backward_pass(ops):
    """an input that the backward pass refers to must not change in between; with checkpoints it may"""
    t = norm_inputs(gen(32), (20, 64), F32)
    for keep8 in (False, True):
        x = t["x"].clone()
        branch = t["branch"].clone().requires_grad_()
        y, h = ops.gated_residual_norms(x, branch, post=t["post"], pre=t["pre"], checkpoint8=keep8)
        before, = torch.autograd.grad(h.sum() + (y * y).sum(), branch, retain_graph=True)
        again = h.sum() + (y * y).sum()
        x.zero_()
        if keep8:
            assert torch.equal(before, torch.autograd.grad(again, branch)[0])
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(again, branch)


def test_without_gradients(ops):
    t = norm_inputs(gen(33), (20, 64), F32)
    x = t["x"].clone().requires_grad_()
    want = ops.gated_residual_norms(x, t["branch"], post=t["post"], pre=t["pre"])
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            y, h = ops.gated_residual_norms(x, t["branch"], post=t["post"], pre=t["pre"])
            got = ops.label_log_probs(h, torch.zeros(20, dtype=torch.int64, device=DEV), topk=2)
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])
        assert not any(v.requires_grad for v in (y, h, *got))
    plain = ops.gated_residual_norms(t["x"], t["branch"], post=t["post"])
    assert plain[1] is None and not plain[0].requires_grad


def test_capture_beside_an_eager_graph_is_refused(ops):
    """the forward call says so: the backward pass could not be captured.  (It is not called here.)  With the eager graph gone it can"""
    t = norm_inputs(gen(35), (20, 64), F32)
    w = rand(gen(36), 64, 64).requires_grad_()
    x, logits = t["x"].clone().requires_grad_(), rand(gen(37), 20, 50).requires_grad_()
    target = torch.arange(20, device=DEV)
    calls = {"gated_residual_norms": lambda: ops.gated_residual_norms(x, t["branch"], post=t["post"])[0],
             "label_log_probs": lambda: ops.label_log_probs(logits, target).log_probs,
             "linear_checkpoint8": lambda: ops.linear_checkpoint8(t["branch"], w)}
    for name, call in calls.items():
        leaf = {"gated_residual_norms": x, "label_log_probs": logits, "linear_checkpoint8": w}[name]
        alive = call()
        want = torch.autograd.grad(alive.sum(), leaf, retain_graph=True)[0]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match=name + ".*captured"):
                call()
        del alive, graph
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call().sum(), leaf)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call().sum(), leaf)[0]
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_second_derivatives_are_refused(ops):
    t = norm_inputs(gen(34), (20, 64), F32)
    leaves, out = both(ops, t)
    first = grads_of(leaves, out)
    leaves, out = both(ops, t)
    graph = grads_of(leaves, out, create_graph=True)
    assert all(torch.equal(a, b.detach()) for a, b in zip(first, graph))
    for g in graph:
        with pytest.raises(RuntimeError, match="no second derivatives"):
            torch.autograd.grad(g.sum(), leaves, allow_unused=True, retain_graph=True)
    leaves, out = both(ops, t)
    up = [torch.ones_like(o).requires_grad_() for o in out]
    g, = torch.autograd.grad(out, leaves[:1], up, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(g.sum(), up)


def test_long_rows_pass_32_bit_offsets(ops):
    """an activation of more than 2^32 bytes: the last rows are where they should be"""
    rows, n = (1 << 21) + 3, 1056
    x = torch.zeros(rows, n, dtype=BF16, device=DEV)
    tail = rand(gen(2), 5, n, dtype=BF16)
    x[-5:] = tail
    kept = ops.checkpoint8(x)
    assert torch.equal(kept.restore()[-5:].double(), kept64(d64(tail))) and not bool(kept.codes[:-5].any())
    dy = torch.zeros(rows, 16, dtype=BF16, device=DEV)
    dy[-5:] = rand(gen(3), 5, 16, dtype=BF16)
    dw, _ = ops.checkpoint8_weight_grad(dy, kept, out_dtype=F32)
    want = d64(dy[-5:]).t() @ kept64(d64(tail))
    check(dw, want, 16 * U * (d64(dy[-5:]).abs().t() @ kept64(d64(tail)).abs()), "dW")
    del kept
    with torch.no_grad():
        y, h = ops.gated_residual_norms(x, x, pre=(torch.ones(n, dtype=BF16, device=DEV), None))
    small = ops.gated_residual_norms(tail, tail, pre=(torch.ones(n, dtype=BF16, device=DEV), None))
    assert torch.equal(y[-5:], small[0]) and torch.equal(h[-5:], small[1])
    got = ops.label_log_probs(x, torch.zeros(rows, dtype=torch.int64, device=DEV), topk=2)
    assert torch.equal(got.log_probs[-5:], ops.label_log_probs(tail, torch.zeros(5, dtype=torch.int64, device=DEV)).log_probs)
    assert torch.equal(got.top_ids[-5:], ops.label_log_probs(tail, torch.zeros(5, dtype=torch.int64, device=DEV), topk=2).top_ids)
