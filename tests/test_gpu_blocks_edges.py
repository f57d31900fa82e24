"""GPU tests of the operators of include/schemanet_blocks.h at their edges: derivatives that would be lost, values at
the end of a type's range, gates far open, what a block with 8-bit checkpoints holds in memory, errors from below,
and tensors of other kinds."""
import os
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwd

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "schemanet-pytorch_amd"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

from blocks_plain import HALF, U, Norms64, check, kept64  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
K_ROW = 128                                       # roundings in a row of the norms' backward pass, as counted in test_gpu_blocks.py
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


# ------------------------------------------------------------------------------------------------ gates far open and far closed
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [3, 200, 300, 1100])
def test_gradient_of_open_and_closed_gates(ops, dtype, width, keep8):
    """dgate = dy scale branch s (1 - s) without norms: each factor has its own relative error, 1 - s of an open gate among them.  The
    roundings: the exponent's product |z| U twice, exp 2, sum, reciprocal 2, e s, four products: (16 + 2 |z|) U of the value."""
    g = gen(width)
    z = (torch.rand(9, width, generator=g) * 60 - 30).to(dtype)
    z[0], z[1], z[2], z[3] = 17.5, 30.0, -30.0, 0.0
    z = z.to(DEV).requires_grad_()
    x, f, dy, scale = rand(g, 9, width, dtype=dtype), rand(g, 9, width, dtype=dtype, std=20.0), rand(g, 9, width, dtype=dtype, std=50.0), rand(g, width, dtype=dtype)
    y, _ = ops.gated_residual_norms(x, f, gate=z, scale=scale, checkpoint8=keep8)
    got, = torch.autograd.grad(y, z, dy)
    zz, ff = (kept64(d64(z)), kept64(d64(f))) if keep8 else (d64(z), d64(f))
    want = d64(dy) * d64(scale) * ff * torch.sigmoid(zz) * torch.sigmoid(-zz)
    check(got, want, HALF[dtype] * want.abs() + (16 + 2 * zz.abs()) * U * want.abs() * (1 + HALF[dtype]) + TINY[dtype], "dgate")


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dtype,width", [(F32, 256), (F32, 700), (BF16, 128), (BF16, 2000)])
def test_gradient_of_open_gates_between_norms(ops, dtype, width, norm, keep8):
    """the same between both norms: K_ROW roundings of the formula with absolute values, s (1 - s) in it"""
    g = gen(width)
    shape = (33, width)
    z = (torch.rand(*shape, generator=g) * 22 + 8).to(dtype).to(DEV).requires_grad_()
    x, f, dy, dh = (rand(g, *shape, dtype=dtype, std=s) for s in (2.0, 1.0, 30.0, 30.0))
    scale, w1, b1, w2, b2 = (rand(g, width, dtype=dtype, std=0.3, mean=m) for m in (1.0, 1.0, 0.0, 1.0, 0.0))
    y, h = ops.gated_residual_norms(x, f, gate=z, scale=scale, post=(w1, b1), pre=(w2, b2), norm=norm, checkpoint8=keep8)
    got, = torch.autograd.grad([y, h], z, [dy, dh])
    kept = tuple(kept64(d64(t)) for t in (x, f, z)) if keep8 else None
    r = Norms64(d64(x), d64(f), d64(z), d64(scale), (d64(w1), d64(b1)), (d64(w2), d64(b2)), norm, 1e-5, d64(dy), d64(dh), kept)
    zz = kept[2] if keep8 else d64(z)
    closed = torch.sigmoid(-zz)
    want = r.dgate / (1 - torch.sigmoid(zz)) * closed               # (the definition's own 1 - s cancels in 64 bits too, by 1e-3 at 30)
    check(got, want, HALF[dtype] * want.abs() + (K_ROW + 2 * zz.abs()) * U * r.dgate_mag * closed * (1 + HALF[dtype]) + TINY[dtype], "dgate")


# ------------------------------------------------------------------------------------------------ what a block holds
def residual_gnn(activation, layers, checkpoint8, E=256):
    import schema_inference.graph as graph
    torch.manual_seed(7)
    gnn = graph.GNN(50, E, layers, activation=activation, residual=True, checkpoint8=checkpoint8).to(DEV)
    with torch.no_grad():
        for layer in gnn.layers:
            layer.scale.add_(0.5)
    return gnn


def graphs(G=4, n=192, edge_grad=False):
    g = gen(5)
    return dict(nodes=torch.rand(G, n, generator=g).to(DEV), edges=(torch.rand(G, n, n, generator=g) / n).to(DEV).requires_grad_(edge_grad),
                ingredients=torch.randint(0, 50, (G, n), generator=g).to(DEV), n_valid=torch.tensor([192, 3, 100, 191], dtype=torch.int32, device=DEV),
                divisor=torch.tensor([n], dtype=torch.int32, device=DEV))


def held(gnn, data):
    before = torch.cuda.memory_allocated(DEV)
    out = gnn(**data)
    return torch.cuda.memory_allocated(DEV) - before, out


@pytest.mark.parametrize("edge_grad", [False, True])
@pytest.mark.parametrize("activation,checkpoint8,whole,bytes8", [("relu", True, 0, 6), ("swish", True, 1, 5), ("none", True, 0, 5), ("relu", False, 5, 0), ("swish", False, 6, 0)])
def test_what_a_block_holds(ops, activation, checkpoint8, whole, bytes8, edge_grad):
    """bytes of one more block, by the allocator.  whole: float32 tensors; bytes8: those of one byte an element, all with their 1 / 32 of
    exponents but for ReLU's signs.  Without checkpoints h and the Linear's input are among the whole ones and a gradient for the edges
    adds none; with them it adds h and takes its checkpoint away.  Beside them 16 bytes of statistics a row and, for each allocation,
    rounding up to 512 bytes."""
    data = graphs(edge_grad=edge_grad)
    some, more = residual_gnn(activation, 2, checkpoint8), residual_gnn(activation, 3, checkpoint8)
    for gnn in (some, more):
        gnn(**data)                                                   # (what is built once and kept)
    a, out = held(some, data)
    del out
    b, out = held(more, data)
    elements = 4 * 192 * 256
    if checkpoint8 and edge_grad:
        whole, bytes8 = whole + 1, bytes8 - 1
    signs = 1 if checkpoint8 and activation == "relu" else 0
    want = elements * (4 * whole + signs + (bytes8 - signs) * 33 / 32) + 16 * 4 * 192
    assert want <= b - a <= want + 16 * 512, (b - a) / elements
    torch.autograd.grad(out.sum(), list(more.parameters()))


@pytest.mark.parametrize("activation", ["relu", "swish", "none"])
@pytest.mark.parametrize("edge_grad", [False, True])
def test_a_block_that_holds_less_computes_the_same(ops, activation, edge_grad):
    """the forward pass is that of the block without checkpoints; gradients, those of the edges among them, differ by what 8 bits round:
    each kept element by at most 1 / 127.5 of its block's maximum, uniformly distributed, so by under a tenth of a gradient's norm"""
    data = graphs(edge_grad=edge_grad)
    plain, kept = residual_gnn(activation, 3, False), residual_gnn(activation, 3, True)
    kept.load_state_dict(plain.state_dict())
    up = rand(gen(9), 4, 256)
    results = []
    for gnn in (plain, kept):
        out = gnn(**data)
        leaves = list(gnn.parameters()) + ([data["edges"]] if edge_grad else [])
        results.append((out.detach(), torch.autograd.grad(out, leaves, up)))
    assert torch.equal(results[0][0], results[1][0])
    for a, b in zip(results[1][1], results[0][1]):
        assert float((a.double() - b.double()).norm()) <= 0.1 * float(b.double().norm())


def test_relu_of_signs_is_relu(ops):
    from schema_inference.graph.gnn import _ReluOfSigns
    x = rand(gen(11), 1000)
    x[:6] = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 1e-45], device=DEV)
    up = rand(gen(12), 1000)
    got, want = [], []
    for f, into in ((_ReluOfSigns.apply, got), (torch.relu, want)):
        leaf = x.clone().requires_grad_()
        y = f(leaf)
        into += [y.detach(), torch.autograd.grad(y, leaf, up)[0]]
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(a.isnan(), b.isnan())


def test_the_adjacency_product_keeps_its_operand_for_the_edges_only(ops):
    x = rand(gen(13), 3, 40, 64).requires_grad_()
    for edge_grad in (False, True):
        edges = rand(gen(14), 3, 40, 40).requires_grad_(edge_grad)
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t, lambda t: t):
            y = ops.edges_adj_matmul(edges, x)
        assert len(seen) == int(edge_grad)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        adj = (d64(edges) + d64(edges).transpose(1, 2)) / 2 + torch.eye(40, dtype=torch.float64, device=DEV)
        want = adj.sum(1, keepdim=True).transpose(1, 2).expand(3, 40, 64)
        # split-fp16 products are off by 2^-22 of an operand's largest magnitude for each of the 40 terms
        assert float((dx.double() - want).abs().max()) <= 2.0 ** -22 * 40 * 2 * float(adj.abs().max())


# ------------------------------------------------------------------------------------------------ errors from below
def test_out_of_memory_is_torch_s(ops):
    """4 TiB and more, which no card has: the allocator says so at once.  (Views of a few elements.)"""
    x = torch.zeros(1, 1, device=DEV).expand(1 << 20, 1 << 20)
    with pytest.raises(torch.OutOfMemoryError):
        ops.checkpoint8(x)
    with pytest.raises(torch.OutOfMemoryError):
        ops.label_log_probs(x, torch.zeros(1 << 20, dtype=torch.int64, device=DEV))
    narrow = torch.zeros(1, 1, device=DEV).expand(1 << 30, 4096)
    with pytest.raises(torch.OutOfMemoryError):
        ops.gated_residual_norms(narrow, narrow)
    x = rand(gen(1), 4, 64)
    assert torch.equal(ops.gated_residual_norms(x, x)[0], x + x)


def test_hooks_for_saved_tensors_raise_their_own(ops):
    x, target = rand(gen(2), 4, 64).requires_grad_(), torch.arange(4, device=DEV)

    class Full(Exception):
        pass

    def raises(t):
        raise Full("no room for " + str(tuple(t.shape)))
    for call in (lambda: ops.gated_residual_norms(x, x), lambda: ops.gated_residual_norms(x, x, checkpoint8=True), lambda: ops.label_log_probs(x, target)):
        with pytest.raises(Full, match="no room"):
            with torch.autograd.graph.saved_tensors_hooks(raises, lambda t: t):
                call()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, raises):
            out = call()[0]
        with pytest.raises(Full, match="no room"):
            out.sum().backward()
    with pytest.raises(RuntimeError, match="width 4097"):
        ops.gated_residual_norms(torch.zeros(1, 4097, device=DEV), torch.zeros(1, 4097, device=DEV))
    with pytest.raises(TypeError):
        ops.gated_residual_norms(x, x, eps="small")


@pytest.mark.parametrize("change", [lambda t: t.float() if t.dtype != F32 else t.double(), lambda t: t.cpu(), lambda t: t[..., :1].clone(), lambda t: t.flatten()[:-1].clone(),
                                    lambda t: t[None].clone()])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_saved_tensors_that_come_back_as_others_are_refused(ops, dtype, change):
    """hooks that compress or move what is saved and hand back something else: the kernels would read it by the forward call's sizes.  Each
    saved tensor in turn; the other order of elements is fine"""
    g = gen(4)
    x, f, z = (rand(g, 2, 6, 64, dtype=dtype).requires_grad_() for _ in range(3))
    w = [rand(g, 64, dtype=dtype).requires_grad_() for _ in range(5)]
    nv, target = torch.tensor([6, 3], dtype=torch.int32, device=DEV), torch.zeros(2, 6, dtype=torch.int64, device=DEV)
    norms = lambda keep8: ops.gated_residual_norms(x, f, gate=z, scale=w[0], post=(w[1], w[2]), pre=(w[3], w[4]), n_valid=nv, checkpoint8=keep8)[1]      # noqa: E731
    for call, saved in ((lambda: norms(False), 10), (lambda: norms(True), 13), (lambda: ops.label_log_probs(x, target).log_probs, 3)):
        for at in range(saved):
            count = iter(range(100))
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(count), t), lambda p: change(p[1]) if p[0] == at else p[1]):
                out = call()
            assert next(count) == saved
            with pytest.raises(RuntimeError, match="came back as|do not hold|different devices|CUDA tensors"):
                out.float().sum().backward()
    for call in (lambda: norms(False), lambda: ops.label_log_probs(x, target).log_probs):
        want = torch.autograd.grad(call().float().sum(), x)[0]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t.transpose(0, -1).contiguous().transpose(0, -1)):
            out = call()
        assert torch.equal(torch.autograd.grad(out.float().sum(), x)[0], want)


# ------------------------------------------------------------------------------------------------ tensors of other kinds
def message_without(tensor, call):
    """what `call` raises while the tensor's storage is freed ("": nothing).  The memory is back before anybody can look at the tensor: a
    failing test prints its arguments, and printing a freed tensor reads address 0."""
    storage, message = tensor.untyped_storage(), ""
    size = storage.nbytes()
    storage.resize_(0)
    try:
        call()
    except RuntimeError as error:
        message = str(error)
    finally:
        storage.resize_(size)
    return message


def test_tensors_without_memory_are_refused(ops):
    """storages freed to save memory (and not yet filled again): a gate, scale or bias among them must not pass for one that was not given"""
    g = gen(6)
    x, f, z = (rand(g, 4, 64) for _ in range(3))
    w = [rand(g, 64) for _ in range(5)]
    norms = lambda: ops.gated_residual_norms(x, f, gate=z, scale=w[0], post=(w[1], w[2]), pre=(w[3], w[4]))      # noqa: E731
    assert all("has no memory" in m for m in [message_without(t, norms) for t in (x, f, z, *w)])
    target, scale, nv = torch.zeros(4, dtype=torch.int64, device=DEV), w[0].clone().requires_grad_(), torch.ones(2, dtype=torch.int32, device=DEV)
    y, _ = ops.gated_residual_norms(x, f, scale=scale)
    kept = ops.checkpoint8(x)
    messages = [message_without(scale, lambda: y.sum().backward()),
                message_without(nv, lambda: ops.gated_residual_norms(f.reshape(2, 2, 64), f.reshape(2, 2, 64), n_valid=nv)),
                message_without(target, lambda: ops.label_log_probs(f, target)), message_without(x, lambda: ops.label_log_probs(x, target)),
                message_without(x, lambda: ops.checkpoint8(x)), message_without(x, lambda: ops.checkpoint8_weight_grad(x, kept))]
    assert all("has no memory" in m for m in messages)


@pytest.mark.parametrize("width", [1, 64])
def test_negated_views(ops, width):
    """views that stand for the negative of what lies in memory (imag of a conjugate; with one feature they look contiguous): inputs,
    parameters and upstream gradients"""
    g = gen(8)
    view = lambda *shape: torch._neg_view(rand(g, *shape))      # noqa: E731
    pair = torch.view_as_complex(rand(g, 6, 1, 2)).conj().imag
    assert pair.is_neg() and view(3).is_neg() and view(3).is_contiguous()
    x, f, z = (view(6, width) for _ in range(3)) if width > 1 else (pair, view(6, 1), pair)
    w = [view(width) for _ in range(5)]
    norms = lambda x, f, z, w: ops.gated_residual_norms(x, f, gate=z, scale=w[0], post=(w[1], w[2]), pre=(w[3], w[4]))      # noqa: E731
    real = lambda t: t.resolve_neg().clone()      # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(norms(x, f, z, w), norms(real(x), real(f), real(z), [real(t) for t in w])))
    kept, plain = ops.checkpoint8(x), ops.checkpoint8(real(x))
    assert torch.equal(kept.codes, plain.codes) and torch.equal(kept.restore(), plain.restore())
    assert all(torch.equal(a, b) for a, b in zip(ops.checkpoint8_weight_grad(f, kept), ops.checkpoint8_weight_grad(real(f), kept)))
    target = torch.zeros(6, dtype=torch.int64, device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(ops.label_log_probs(x, target, topk=1), ops.label_log_probs(real(x), target, topk=1)))
    leaf, up, up1 = rand(g, 6, width).requires_grad_(), view(6, width), view(6)
    for out, u in ((ops.gated_residual_norms(leaf, f)[0], up), (ops.label_log_probs(leaf, target).log_probs, up1), (ops.label_log_probs(leaf, target).entropy, up1)):
        a, = torch.autograd.grad(out, leaf, u, retain_graph=True)
        assert torch.equal(a, torch.autograd.grad(out, leaf, real(u))[0])
    scale = rand(g, width).requires_grad_()
    y, _ = norms(x, f, z, [torch._neg_view(scale)] + w[1:])
    a, = torch.autograd.grad(y, scale, up, retain_graph=True)
    y2, _ = norms(real(x), real(f), real(z), [-scale] + [real(t) for t in w[1:]])
    assert torch.equal(a, torch.autograd.grad(y2, scale, real(up))[0])


# ------------------------------------------------------------------------------------------------ several backward passes over one graph
@pytest.mark.parametrize("residual,checkpoint8", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("layers", [2, 3])
def test_several_backward_passes_of_a_gnn(ops, residual, checkpoint8, layers):
    """a kept graph differentiated again, wholly or for the last layer's parameters only, as programs do that weigh several losses: each pass
    gives the gradients of a fresh graph, bit for bit.  (The layers sum their products' edge gradients in one buffer.)"""
    import schema_inference.graph as graph
    torch.manual_seed(4)
    kw = dict(residual=True, checkpoint8=checkpoint8) if residual else {}
    gnn = graph.GNN(50, 64, layers, **kw).to(DEV)
    data = graphs(n=192, edge_grad=True)
    data["feat_mask"] = torch.arange(192, device=DEV)[None] >= data["n_valid"][:, None]
    leaves = [data["edges"]] + list(gnn.parameters())
    last = [p for p in gnn.layers[-1].parameters()]
    up = rand(gen(1), 4, 64)
    fresh = lambda inputs: [t.clone() for t in torch.autograd.grad(gnn(**data), inputs, up)]      # noqa: E731
    whole, part = fresh(leaves), fresh(last)
    out = gnn(**data)
    for inputs, want in ((leaves, whole), (leaves, whole), (last, part), (leaves, whole), (last, part), (last, part), (leaves[:1], whole[:1]), (leaves, whole)):
        got = torch.autograd.grad(out, inputs, up, retain_graph=True, allow_unused=True)
        assert all(a is not None and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["gather", "edges"])
def test_products_of_one_operand_in_parts(ops, kind):
    """three products in sequence on one edge tensor that autograd reaches in parts: the first two only, the third from a detached input (a
    backward pass in stages), both at once; the edges' gradient is each time that of products that share nothing"""
    g = gen(21)
    G, n, E = 3, 50, 64
    edges, x = torch.rand(G, n, n, generator=g).to(DEV).requires_grad_(), rand(g, G, n, E).requires_grad_()
    table, ids = rand(g, 30, E).requires_grad_(), torch.randint(0, 30, (G, n), generator=g).to(DEV)
    up = rand(g, G, n, E)

    def run(summed):
        planes = ops.gcn_adjacency_planes(edges.detach())
        first = (lambda: ops.gather_adj_matmul(edges, table, ids, adj_planes=planes, sum_edge_grads=summed)) if kind == "gather" else (
            lambda: ops.edges_adj_matmul(edges, x, planes, summed))
        h1 = first()
        h2 = ops.edges_adj_matmul(edges, h1.tanh(), planes, summed)
        cut = h2.detach().requires_grad_()
        h3 = ops.edges_adj_matmul(edges, cut.tanh(), planes, summed)
        whole = ops.edges_adj_matmul(edges, h2.tanh(), planes, summed)
        out = [torch.autograd.grad(h2, edges, up, retain_graph=True)[0]]
        a, stage = torch.autograd.grad(h3, [edges, cut], up, retain_graph=True)
        out += [a, torch.autograd.grad(h2, edges, stage, retain_graph=True)[0]]
        out += [torch.autograd.grad([h3, h2], edges, [up, up], retain_graph=True)[0], torch.autograd.grad(whole, edges, up, retain_graph=True)[0]]
        torch.autograd.grad(whole, h2, up, retain_graph=True)          # (a pass that does not want the edges)
        out += [torch.autograd.grad(whole, edges, up)[0]]
        assert planes.grad_sum is None and planes.pending == 0
        return out
    for a, b in zip(run(True), run(False)):
        # sums of two or three products, symmetrised before or after they are added: a few roundings of the largest
        assert float((a - b).abs().max()) <= 8 * U * float(b.abs().max())


def test_operands_do_not_outlive_their_step(ops):
    """no cycle keeps an adjacency operand, its edges or the graph alive"""
    import gc
    import weakref
    gc.collect()
    gc.disable()
    try:
        edges, x = rand(gen(1), 2, 40, 40).requires_grad_(), rand(gen(2), 2, 40, 64).requires_grad_()
        planes = ops.gcn_adjacency_planes(edges.detach())
        y = ops.edges_adj_matmul(edges, ops.edges_adj_matmul(edges, x, planes, True), planes, True)
        y.sum().backward()
        assert planes.edge_token[1]() is not None
        del y
        assert planes.edge_token[1]() is None                          # (the graph is gone, the operand keeps nothing of it)
        seen = [weakref.ref(t) for t in (planes.hi, edges)]
        del planes, edges
        assert [r() for r in seen] == [None, None]
    finally:
        gc.enable()


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("keep8", [False, True])
def test_under_recomputation(ops, reentrant, keep8):
    """torch's activation checkpointing runs the forward pass again inside the backward pass: the same gradients"""
    from torch.utils.checkpoint import checkpoint
    g = gen(31)
    x, f = rand(g, 3, 10, 64).requires_grad_(), rand(g, 3, 10, 64).requires_grad_()
    edges, w = torch.rand(3, 10, 10, generator=g).to(DEV).requires_grad_(), rand(g, 64).requires_grad_()
    target = torch.arange(30, device=DEV).reshape(3, 10)

    def block(x, f, edges, w):
        planes = ops.gcn_adjacency_planes(edges.detach())
        y, h = ops.gated_residual_norms(x, ops.edges_adj_matmul(edges, f, planes, True), scale=w, pre=(w, None), checkpoint8=keep8)
        return ops.label_log_probs(ops.edges_adj_matmul(edges, h, planes, True), target).log_probs + y.sum(-1)
    results = []
    for run in (block, lambda *a: checkpoint(block, *a, use_reentrant=reentrant)):
        for leaf in (x, f, edges, w):
            leaf.grad = None
        out = run(x, f, edges, w)
        out.sum().backward()
        results.append([out.detach()] + [leaf.grad.clone() for leaf in (x, f, edges, w)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_an_operand_used_for_several_steps(ops):
    """the adjacency operand of edges that stay the same: eager steps one after the other, on another stream, and captured, each with the
    gradients of an operand of its own"""
    g = gen(41)
    edges, x, up = torch.rand(2, 40, 40, generator=g).to(DEV).requires_grad_(), rand(g, 2, 40, 64).requires_grad_(), rand(g, 2, 40, 64)

    def step(planes):
        y = ops.edges_adj_matmul(edges, ops.edges_adj_matmul(edges, x, planes, True).tanh(), planes, True)
        return torch.autograd.grad(y, [edges, x], up)
    want = [t.clone() for t in step(ops.gcn_adjacency_planes(edges.detach()))]
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))      # noqa: E731
    planes = ops.gcn_adjacency_planes(edges.detach())
    assert same(step(planes)) and same(step(planes))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(planes)
    torch.cuda.current_stream().wait_stream(side)
    assert same(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(planes)
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out)
    assert same(step(planes))
