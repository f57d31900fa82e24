"""GPU tests of what calls the operators of include/schemanet_blocks.h: the residual GNN (with and without 8-bit checkpoints), the
loss `ce_entropy_loss` and `SchemaNetPredictor.answers`, against float64 torch.

Bounds.  The products of the GNN run on split-fp16 operands with float32 sums: off by 2^-22 of an operand's largest magnitude; a block
holds three of them and two norms, so results agree with float64 to 2^-22 x (roundings added up over widths of 64 .. 128 and 3
blocks: under 2^9) = 2^-13 of the result's norm.  An 8-bit checkpoint is off by at most 1 / 127.5 of its block's maximum,
uniformly distributed: gradients by under a tenth of their norm."""
import os
import sys

import pytest
import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "schemanet-pytorch_amd"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

import datagen  # noqa: E402
from test_gpu_parity import T, mods  # noqa: E402,F401  (mods: fixture)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
REL = 2.0 ** -13


def make(G, n, words, E, layers, seed, **kw):
    import schema_inference.graph as graph
    torch.manual_seed(seed)
    gnn = graph.GNN(words, E, layers, activation="swish", residual=True, **kw).to(DEV)
    with torch.no_grad():
        for p in gnn.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn_like(p))
        for layer in gnn.layers:
            layer.scale.add_(0.5)
        gnn.fc.weight.mul_(0.1)
    g = torch.Generator().manual_seed(seed)
    nodes = torch.rand(G, n, generator=g).to(DEV)
    edges = (torch.rand(G, n, n, generator=g) / n).to(DEV)
    ids = torch.randint(0, words, (G, n), generator=g).to(DEV)
    n_valid = torch.randint(1, n + 1, (G,), generator=g).to(torch.int32)
    n_valid[0] = n
    return gnn, nodes, edges, ids, n_valid.to(DEV)


def gnn64(gnn, nodes, edges, ids, n_valid, divisor):
    """the residual GNN in float64 torch -> features and the parameters that gradients can be asked for"""
    ps = {k: v.detach().double().requires_grad_() for k, v in gnn.named_parameters()}
    E = gnn.embed_dim
    ln = lambda t, k: F.layer_norm(t, (E,), ps[k + ".weight"], ps[k + ".bias"], 1e-5)        # noqa: E731
    live = torch.ones(*ids.shape, 1, dtype=torch.float64, device=DEV)
    if n_valid is not None:
        live = (torch.arange(ids.shape[1], device=DEV)[None] < n_valid[:, None]).double()[..., None]
    emb = ps["embedding.weight"]
    x = F.embedding(ids, emb, padding_idx=gnn.embedding.padding_idx) * live
    adj = (edges + edges.transpose(1, 2)) / 2 + torch.eye(ids.shape[1], dtype=torch.float64, device=DEV)
    h = ln(x, "layers.0.norm") * live
    L = len(gnn.layers)
    for i in range(L):
        p = "layers.%d." % i
        f = F.silu(F.linear(adj.matmul(h), ps[p + "g_conv.linear.weight"], ps[p + "g_conv.linear.bias"]))
        gate = torch.sigmoid(F.linear(h, ps[p + "gate.weight"], ps[p + "gate.bias"]))
        x = (x + ps[p + "scale"] * gate * ln(f, p + "post")) * live
        h = ln(x, "layers.%d.norm" % (i + 1) if i + 1 < L else "out_norm") * live
    pooled = (h * nodes[..., None]).sum(1) / divisor
    return F.linear(pooled, ps["fc.weight"], ps["fc.bias"]), ps


def close(a, b, rel, what):
    err = float((a.double() - b).norm() / (b.norm() + 1e-30))
    assert err <= rel, (what, err)


@pytest.mark.parametrize("G,n,E,layers,masked", [(3, 20, 64, 1, True), (5, 33, 96, 3, True), (2, 50, 128, 2, False), (2, 9, 40, 2, True)])
def test_residual_gnn(G, n, E, layers, masked):
    gnn, nodes, edges, ids, n_valid = make(G, n, 30, E, layers, G + n)
    n_valid = n_valid if masked else None
    divisor = torch.tensor([n], dtype=torch.int32, device=DEV)
    edges = edges.requires_grad_()
    if masked:                                         # padding has no edges and no weight, as the graph builder leaves it
        live = torch.arange(n, device=DEV)[None] < n_valid[:, None]
        edges = (edges.detach() * live[:, :, None] * live[:, None, :]).requires_grad_()
        nodes = nodes * live
    nodes = nodes.requires_grad_()
    got = gnn(nodes, edges, ids, n_valid=n_valid, divisor=divisor)
    with torch.no_grad():
        close(gnn(nodes, edges, ids, n_valid=n_valid, divisor=divisor), got.detach().double(), REL, "inference and training forms")
    e64, w64 = edges.detach().double().requires_grad_(), nodes.detach().double().requires_grad_()
    want, ps = gnn64(gnn, w64, e64, ids, n_valid, float(n))
    close(got.detach(), want.detach(), REL, "features")
    up = torch.randn(got.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    named = dict(gnn.named_parameters())
    grads = torch.autograd.grad(got, [nodes, edges] + list(named.values()), up)
    wants = torch.autograd.grad(want, [w64, e64] + [ps[k] for k in named], up.double())
    for k, a, b in zip(["nodes", "edges"] + list(named), grads, wants):
        close(a, b, 8 * REL, k)


def test_checkpoints_keep_less_and_give_near_gradients():
    """the same forward pass; what autograd holds shrinks; the gradients see values that 8 bits hold"""
    args = (4, 96, 50, 256, 3, 7)
    plain, nodes, edges, ids, n_valid = make(*args)
    kept, *_ = make(*args, checkpoint8=True)
    kept.load_state_dict(plain.state_dict())
    divisor = torch.tensor([96], dtype=torch.int32, device=DEV)
    up = torch.randn(4, 256, generator=torch.Generator().manual_seed(1)).to(DEV)
    results, held = [], []
    for gnn in (plain, kept):
        seen = {}

        def pack(t):
            seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            return t
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            out = gnn(nodes, edges, ids, n_valid=n_valid, divisor=divisor)
        results.append((out.detach(), torch.autograd.grad(out, list(gnn.parameters()), up)))
        held.append(sum(seen.values()))
    assert torch.equal(results[0][0], results[1][0])
    own = 4 * sum(p.numel() for p in plain.parameters()) + 4 * edges.numel()
    assert held[1] - own < 0.62 * (held[0] - own), held
    for (name, _), a, b in zip(plain.named_parameters(), results[1][1], results[0][1]):
        close(a, b.double(), 0.1, name)


def test_default_gnn_has_the_reference_parameters():
    import schema_inference.graph as graph
    keys = list(graph.GNN(10, 32, 2).state_dict())
    assert keys == ["embedding.weight"] + [f"layers.{i}.{k}" for i in range(2) for k in ("g_conv.linear.weight", "g_conv.linear.bias", "norm.weight", "norm.bias")] \
        + ["fc.weight", "fc.bias"]
    with pytest.raises(ValueError):
        graph.GNN(10, 32, 2, checkpoint8=True)


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_a_residual_matcher_trains(checkpoint8):
    """Matcher with a residual GNN: instance and class graphs, similarity, `ce_entropy_loss`; gradients reach every parameter.  With
    sizes this small an eager and a captured iteration give the same bits."""
    import schema_inference.graph as graph
    from schema_inference.loss import get_loss_fn
    torch.manual_seed(3)
    words, K, bs, n = 40, 12, 6, 30
    m = graph.Matcher("inner_product", words, dict(embed_dim=64, num_layers=3, activation="swish", residual=True, checkpoint8=checkpoint8)).to(DEV)
    g = torch.Generator().manual_seed(5)
    nv = torch.tensor([30, 4, 11, 1, 22, 17], dtype=torch.int32, device=DEV)
    live = torch.arange(n, device=DEV)[None] < nv[:, None]
    inst = dict(ids=torch.where(live, torch.randint(0, words, (bs, n), generator=g).to(DEV), words), vertices=torch.rand(bs, n, generator=g).to(DEV) * live,
                edges=(torch.rand(bs, n, n, generator=g).to(DEV) / n) * live[:, :, None] * live[:, None, :], n=nv, n_max=torch.tensor([30], dtype=torch.int32, device=DEV))
    atlas = dict(class_vertices=torch.rand(K, 25, generator=g).to(DEV).requires_grad_(), class_edges=(torch.rand(K, 25, 25, generator=g) / 25).to(DEV).requires_grad_(),
                 class_ingredients=torch.randint(0, words, (K, 25), generator=g).to(DEV))
    label = torch.tensor([0, 3, 11, -100, 5, 5], device=DEV)
    loss_fn = get_loss_fn(dict(name="ce_entropy_loss"))

    def step():
        pred = m.forward_padded(inst, atlas)
        parts = loss_fn({"pred": pred}, {"label": label})
        loss = parts["cls"] - 0.1 * parts["entropy"]
        return (pred, loss) + torch.autograd.grad(loss, [atlas["class_vertices"], atlas["class_edges"]] + list(m.parameters()))
    first = [t.detach().clone() for t in step()]
    assert all(torch.isfinite(t).all() for t in first) and all(bool(t.any()) for t in first[2:])
    logits = first[0].double()
    lp = torch.log_softmax(logits, -1)
    used = label != -100
    want = -lp[used, label[used]].mean() - 0.1 * (-(lp.exp() * lp).sum(-1)[used].mean())
    assert abs(float(first[1]) - float(want)) <= 64 * 2.0 ** -24 * (1 + abs(float(want)) + float(lp.abs().max()))
    assert all(torch.equal(a, b.detach()) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    m_graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(m_graph):
        out = step()
    for _ in range(3):
        m_graph.replay()
        torch.cuda.synchronize()
        torch.zeros(1 << 16, device=DEV).add_(1).sum()
        assert all(torch.equal(a, b.detach()) for a, b in zip(first, out))


def test_ce_entropy_loss_matches_torch():
    from schema_inference.loss import CEEntropyLoss, get_loss_fn
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(64, 100, generator=g) * 3)
    label = torch.randint(0, 100, (64,), generator=g)
    label[::9] = -100
    fn = get_loss_fn(dict(name="ce_entropy_loss"))
    assert isinstance(fn, CEEntropyLoss)
    cpu = fn({"pred": x}, {"label": label})
    leaf = x.to(DEV).requires_grad_()
    gpu = fn({"pred": {"pred": leaf}}, {"label": label.to(DEV)})
    want = F.cross_entropy(x.double(), label)
    tol = 128 * 2.0 ** -24 * (1 + float(x.abs().max()))        # sums of 100 terms and of 57 rows, values up to the largest logit
    for out in (cpu, gpu):
        assert abs(float(out["cls"].detach()) - float(want)) <= tol
        assert abs(float(out["entropy"].detach()) - float(cpu["entropy"])) <= tol
    grad, = torch.autograd.grad(gpu["cls"] - 0.2 * gpu["entropy"], leaf)
    ref = x.double().requires_grad_()
    lp = torch.log_softmax(ref, -1)
    used = label != -100
    value = F.cross_entropy(ref, label) + 0.2 * (lp.exp() * lp).sum(-1)[used].mean()
    want, = torch.autograd.grad(value, ref)
    assert float((grad.cpu().double() - want).abs().max()) <= tol * float(want.abs().max())


def test_predictor_answers(mods):
    from test_gpu_api import _predictor
    B, L, D, M, K = 6, 196, 192, 64, 11
    batches = [(T(datagen.bellish((L + 1, B, D), 1, 1.0)), T(datagen.bellish((B * 3, L + 1, L + 1), 2, 1.5)))]
    predictor, _ = _predictor(mods, batches, M, D, K, 64)
    x = torch.zeros(B, 3, 4, 4, device=DEV)
    with torch.no_grad():
        pred = predictor(x)["pred"]
        out = predictor.answers(x, topk=3)
        assert out.log_probs is None and torch.equal(out.top_ids, torch.sort(pred, dim=-1, descending=True, stable=True).indices[:, :3])
        lp = torch.log_softmax(pred.double(), -1)
        tol = 128 * 2.0 ** -24 * (1 + float(lp.abs().max()))           # sums of 11 terms, values up to the largest log probability
        assert float((out.top_log_probs.double() - lp.gather(-1, out.top_ids)).abs().max()) <= tol
        label = out.top_ids[:, 1].contiguous()
        named = predictor.answers(x, topk=50, label=label)
        assert named.top_ids.shape == (B, K) and float((named.log_probs.double() - lp.gather(-1, label[:, None])[:, 0]).abs().max()) <= tol
