"""Tensor-level wrappers of include/schemanet_blocks.h, re-exported by `cpp_extension.ops`: the operators of deep residual graph
networks (`gated_residual_norms`), of activations kept in 8 bits for the backward pass (`checkpoint8`, `checkpoint8_weight_grad`,
`linear_checkpoint8`) and of large sets of answers (`label_log_probs`).

They take CUDA tensors in float32, bfloat16 or float16 with rows of any stride, compute in float32 and round each result
once; outputs are new contiguous tensors; nothing synchronises, all of them can be captured into a graph.  Under `torch.autocast`
their floating-point inputs are cast to float32, like those of the other HIP-backed ops of this package.  Arguments that do not
fit raise RuntimeError before anything is launched."""
import math
import struct
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_NORM_WIDTH = 4096
MAX_ALTERNATIVES = 64


def _need(ok, message, *args):
    if not ok:
        raise RuntimeError(message.format(*args))


def _one_device(*ts):
    dev = None
    for t in ts:
        if t is not None:
            d = t.device
            if dev is None:
                dev = d
                _need(d.type == "cuda", "expected CUDA tensors (the HIP path has no CPU fallback)")
            elif d != dev:
                _need(d.type == "cuda", "expected CUDA tensors (the HIP path has no CPU fallback)")
                _need(False, "tensors on different devices: {} vs {}", d, dev)
    return dev


def _p(t):
    return 0 if t is None else t.data_ptr()


_raw_stream = torch._C._cuda_getCurrentRawStream


def _launch(fn, what, dev, *args):
    """fn(*args, current stream of dev) with dev as the current device.  The host's part of a small call is most of it (about 25 us a
    forward call, and the autograd thread runs Python at a third of that speed): the device is only switched where it is another
    one, and the stream is asked for as a number."""
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev.index))
    if rc != 0:
        N.check(rc, what)


def _library():
    return N._lib if N._lib is not None else N.require_gpu()


def _once(backward):
    """a backward pass without second derivatives: the wrapper that says so on their use is only taken under create_graph"""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(run)


def _rows(t, width):
    """[..., width] as (tensor that holds the rows, stride of a row): a view where the rows lie evenly apart, a copy otherwise"""
    if t.is_contiguous():
        return t, width
    if t.stride(-1) != 1 and width > 1:
        t = t.contiguous()
    if t.dim() == 2:
        return t, t.stride(0)
    if t.dim() == 1:
        return t, width
    if not t.is_contiguous():
        try:
            v = t.view(-1, width)
            return v, v.stride(0)
        except RuntimeError:
            t = t.contiguous()
    return t, width


def _autocast(*ts):
    if not torch.is_autocast_enabled("cuda"):
        return ts
    return tuple(t.float() if t is not None and t.is_floating_point() and t.is_cuda else t for t in ts)


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ------------------------------------------------------------------------------------------- activations kept in 8 bits
class Checkpoint8:
    """An activation [..., n] kept in 8 bits: `codes` int8 [rows, npad] and `exps` uint8 [rows, npad / 32], npad = n rounded up to a
    multiple of 32.  A block of 32 features shares one power of two s, the smallest with max|x| < 127.5 s, and an element is kept
    as round(x / s) (half to even): off by at most s / 2 <= max|x| / 127.5, up to max|x| / 254 where the maximum is just under
    127.5 s.  A block that held an infinity or a NaN comes back as NaN; magnitudes under 2^-126 as zero."""

    __slots__ = ("_codes", "_exps", "_shape", "dtype")

    def __init__(self, codes, exps, shape, dtype):
        # (checked here, once: the kernels read both by the shape, and none of the three can be replaced later)
        shape = tuple(shape)
        _need(len(shape) >= 1 and shape[-1] >= 1, "checkpoint8: expected at least one feature, got shape {}", shape)
        rows, npad = math.prod(shape[:-1]), (shape[-1] + 31) // 32 * 32
        _need(codes.dtype == torch.int8 and exps.dtype == torch.uint8 and codes.shape == (rows, npad) and exps.shape == (rows, npad // 32)
              and codes.is_contiguous() and exps.is_contiguous() and codes.device == exps.device,
              "checkpoint8: codes {} and exponents {} do not hold an activation {}", tuple(codes.shape), tuple(exps.shape), shape)
        self._codes, self._exps, self._shape, self.dtype = codes, exps, shape, dtype

    @classmethod
    def _of(cls, codes, exps, shape, dtype):
        """without the checks: buffers that this module has made"""
        self = cls.__new__(cls)
        self._codes, self._exps, self._shape, self.dtype = codes, exps, tuple(shape), dtype
        return self

    @property
    def codes(self):
        return self._codes

    @property
    def exps(self):
        return self._exps

    @property
    def shape(self):
        return self._shape

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def restore(self, dtype=None):
        """the kept values, [..., n] in `dtype` (default: the type of the activation; bfloat16 and float32 hold them exactly)"""
        dtype = dtype or self.dtype
        _need(dtype in _TYPES, "checkpoint8: cannot restore to {}", dtype)
        out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        if out.numel():
            _launch(_library().sn_checkpoint8_restore, "sn_checkpoint8_restore", out.device, _p(self.codes), _p(self.exps), self.codes.shape[0],
                    self.shape[-1], _p(out), _TYPES[dtype])
        return out


def _empty_checkpoint(shape, dtype, dev):
    n = shape[-1]
    rows, npad = math.prod(shape[:-1]), (n + 31) // 32 * 32
    return Checkpoint8._of(torch.empty((rows, npad), dtype=torch.int8, device=dev), torch.empty((rows, npad // 32), dtype=torch.uint8, device=dev), shape, dtype)


def checkpoint8(x):
    """x [..., n] float32 / bfloat16 / float16 (CUDA) -> Checkpoint8, 1 + 1/32 bytes an element.  No autograd: what a backward pass
    keeps."""
    _need(torch.is_tensor(x) and x.dtype in _TYPES, "checkpoint8: expected a float32, bfloat16 or float16 tensor")
    _need(x.dim() >= 1 and x.shape[-1] >= 1, "checkpoint8: expected at least one feature, got shape {}", tuple(x.shape))
    dev = _one_device(x)
    x = x.detach()
    kept = _empty_checkpoint(x.shape, x.dtype, dev)
    if x.numel():
        v, stride = _rows(x, x.shape[-1])
        _launch(_library().sn_checkpoint8, "sn_checkpoint8", dev, _p(v), _TYPES[x.dtype], kept.codes.shape[0], x.shape[-1], stride, _p(kept.codes),
                _p(kept.exps))
    return kept


def checkpoint8_weight_grad(dy, kept, bias=True, out_dtype=None):
    """The gradients of y = x W^T + b with respect to W and b from the kept activation: dy [..., out] of float32, bfloat16 or float16,
    kept = checkpoint8(x) of x [..., in] with the same leading sizes -> (dW [out, in], db [out] or None).

    dW = sum_r dy[r]^T kept[r] on the bf16 matrix cores with float32 sums.  The kept values are exact in bf16 and dy enters as
    bf16 pieces that add up to it (float32: three, float16: two), so the products carry no rounding of their own.  A gradient that is
    infinite or NaN (float32: or beyond bfloat16's largest, 3.39e38) makes its feature's row of dW infinite or NaN.
    out_dtype: the type of both results (default dy's)."""
    _need(isinstance(kept, Checkpoint8), "checkpoint8_weight_grad: expected a Checkpoint8, got {}", type(kept).__name__)
    _need(torch.is_tensor(dy) and dy.dtype in _TYPES, "checkpoint8_weight_grad: expected float32, bfloat16 or float16 gradients")
    out_dtype = out_dtype or dy.dtype
    _need(out_dtype in _TYPES, "checkpoint8_weight_grad: cannot write {}", out_dtype)
    _need(dy.dim() >= 2 and dy.shape[-1] >= 1 and tuple(dy.shape[:-1]) == kept.shape[:-1],
          "checkpoint8_weight_grad: gradients {} do not fit the activation {}", tuple(dy.shape), kept.shape)
    dev = _one_device(dy, kept.codes)
    dy = dy.detach()
    out_f, in_f, rows = dy.shape[-1], kept.shape[-1], kept.codes.shape[0]
    if rows == 0:
        return (torch.zeros((out_f, in_f), dtype=out_dtype, device=dev), torch.zeros(out_f, dtype=out_dtype, device=dev) if bias else None)
    lib = _library()
    dw = torch.empty((out_f, in_f), dtype=out_dtype, device=dev)
    db = torch.empty(out_f, dtype=out_dtype, device=dev) if bias else None
    v, stride = _rows(dy, out_f)
    size = lib.sn_checkpoint8_weight_grad_workspace(rows, out_f, in_f, _TYPES[dy.dtype])
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    _launch(lib.sn_checkpoint8_weight_grad, "sn_checkpoint8_weight_grad", dev, _p(v), _TYPES[dy.dtype], stride, _p(kept.codes), _p(kept.exps), rows, out_f,
            in_f, _p(dw), _p(db), _TYPES[out_dtype], _p(ws), size)
    return dw, db


class _LinearCheckpoint8(torch.autograd.Function):
    """`ops.linear_mfma` that keeps its input in 8 bits: forward and dX are its products, dW and db come from the kept input"""

    @staticmethod
    def forward(ctx, x, weight, bias):
        from . import ops
        x3 = ops._f32c(x.detach())
        x3 = x3[None] if x3.dim() == 2 else x3
        wp = ops.split_planes(weight.detach())
        y = ops.gcn_gemm(ops.split_planes(x3), wp, x3.shape[0], bias=bias, want_c=True)["c"]
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            kept = checkpoint8(x)
            ctx.save_for_backward(weight, kept.codes, kept.exps)
        else:
            ctx.save_for_backward(weight)
        ctx.shape, ctx.scale, ctx.has_bias = tuple(x.shape), wp.scale, bias is not None
        return y[0] if x.dim() == 2 else y

    @_once
    def backward(ctx, dy):
        from . import ops
        weight = ctx.saved_tensors[0]
        dx = dw = db = None
        dy3 = ops._f32c(dy)
        dy3 = dy3[None] if dy3.dim() == 2 else dy3
        if ctx.needs_input_grad[0]:
            dx = ops.gcn_gemm(ops.split_planes(dy3), ops.split_planes(weight.detach(), scale=ctx.scale, transpose=True), dy3.shape[0], want_c=True)["c"]
            dx = dx[0] if len(ctx.shape) == 2 else dx
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            kept = Checkpoint8._of(ctx.saved_tensors[1], ctx.saved_tensors[2], ctx.shape, torch.float32)
            dw, db = checkpoint8_weight_grad(dy3[0] if len(ctx.shape) == 2 else dy3, kept, bias=ctx.has_bias)
            dw = dw if ctx.needs_input_grad[1] else None
        return dx, dw, db


def linear_checkpoint8(x, weight, bias=None):
    """x W^T + b on x [G, n, in] or [rows, in] float32 (CUDA; in and out multiples of 16) with the values and the input gradient of
    `linear_mfma`; the backward pass takes the weight's gradient from x kept in 8 bits (`checkpoint8`) instead of x."""
    _need(all(torch.is_tensor(t) for t in (x, weight)) and x.dim() in (2, 3) and weight.dim() == 2 and x.shape[-1] == weight.shape[1],
          "linear_checkpoint8: expected x [G, n, in] or [rows, in] and weight [out, in]")
    _need(bias is None or tuple(bias.shape) == (weight.shape[0],), "linear_checkpoint8: expected bias [out]")
    x, weight, bias = _autocast(x, weight, bias)
    _need(all(t is None or t.dtype == torch.float32 for t in (x, weight, bias)), "linear_checkpoint8: expected float32 tensors")
    _need(weight.shape[0] % 16 == 0 and weight.shape[1] % 16 == 0, "linear_checkpoint8: in and out must be multiples of 16, got {} and {}",
          weight.shape[1], weight.shape[0])
    _need(x.numel() > 0, "linear_checkpoint8: an empty batch")
    _one_device(x, weight, bias)
    return _LinearCheckpoint8.apply(x, weight, bias)


# ------------------------------------------------------------- the end of a residual block and the norm before the next one
# sn_block_norms_args as one packed value (N.BlockNormsArgs names its members): setting 45 members one by one is a sixth of a small call
_NORM_ARGS = struct.Struct("@IiiiqiiPfiiPPPqqqPPPPPPPPPPPPPPPPqqPPPPPPPPPN")


def _norms_forward(x, branch, gate, params, rms, eps, n_valid, train, keep8):
    """-> y, h, row statistics (train), checkpoints of x, branch and gate (train and keep8)"""
    scale, post_w, post_b, pre_w, pre_b = params
    dev, width = x.device, x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if pre_w is not None else None
    stats, kept = None, ()
    rows = x.numel() // width
    if rows == 0:
        return y, h, stats, kept
    vx, sx = _rows(x, width)
    vb, sb = _rows(branch, width)
    vg, sg = _rows(gate, width) if gate is not None else (None, 0)
    codes = (0,) * 6
    if train:
        stats = torch.empty((rows, 4), dtype=torch.float32, device=dev)
        if keep8:
            kept = tuple(None if t is None else _empty_checkpoint((rows, width), x.dtype, dev) for t in (x, branch, gate))
            codes = [0 if k is None else t.data_ptr() for k in kept for t in ((k.codes, k.exps) if k is not None else (None, None))]
    args = _NORM_ARGS.pack(_NORM_ARGS.size, _TYPES[x.dtype], _param_type(params), rms, rows, width, 0 if n_valid is None else x.shape[1], _p(n_valid), eps,
                           post_w is not None, pre_w is not None, _p(vx), _p(vb), _p(vg), sx, sb, sg, _p(scale), _p(post_w), _p(post_b), _p(pre_w), _p(pre_b),
                           _p(y), _p(h), _p(stats), *codes, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _launch(_library().sn_block_norms_forward, "sn_block_norms_forward", dev, args)
    return y, h, stats, kept


def _param_type(params):
    for t in params:
        if t is not None:
            return _TYPES[t.dtype]
    return 0


class _GatedResidualNorms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, scale, post_w, post_b, pre_w, pre_b, rms, eps, n_valid, keep8):
        params = (scale, post_w, post_b, pre_w, pre_b)
        y, h, stats, kept = _norms_forward(x, branch, gate, params, rms, eps, n_valid, True, keep8)
        if kept:
            held = [t for k in kept for t in ((k.codes, k.exps) if k is not None else (None, None))]
        else:
            held = [x, branch, gate]
        ctx.save_for_backward(*params, n_valid, stats, *held)
        ctx.opts = (x.shape, x.dtype, rms, eps, bool(kept))
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @_once
    def backward(ctx, dy, dh=None):
        scale, post_w, post_b, pre_w, pre_b, n_valid, stats, *held = ctx.saved_tensors
        shape, dtype, rms, eps, kept = ctx.opts
        width, dev = shape[-1], (dy if dy is not None else dh).device
        want = ctx.needs_input_grad
        params = (scale, post_w, post_b, pre_w, pre_b)
        if stats is None:                                                   # no rows
            whole = [torch.zeros(shape, dtype=dtype, device=dev) if want[i] else None for i in range(3)]
            return (*whole, *(torch.zeros_like(p) if p is not None and want[3 + i] else None for i, p in enumerate(params)), None, None, None, None)
        rows = stats.shape[0]
        codes = vx = vb = vg = None
        sx = sb = sg = 0
        if kept:
            codes = [_p(t) for t in held]
            gated = held[4] is not None
        else:
            vx, sx = _rows(held[0], width)
            vb, sb = _rows(held[1], width)
            gated = held[2] is not None
            if gated:
                vg, sg = _rows(held[2], width)
        vy, sy = _rows(dy, width) if dy is not None else (None, 0)
        vh, sh = _rows(dh, width) if dh is not None else (None, 0)
        dx = torch.empty(shape, dtype=dtype, device=dev) if want[0] else None
        dbranch = torch.empty(shape, dtype=dtype, device=dev) if want[1] else None
        dgate = torch.empty(shape, dtype=dtype, device=dev) if gated and want[2] else None
        columns = [p is not None and want[3 + i] for i, p in enumerate(params)]
        grads = [None] * 5
        if any(columns):
            lines = torch.empty((5, width), dtype=next(p.dtype for p in params if p is not None), device=dev).unbind(0)
            grads = [lines[i] if c else None for i, c in enumerate(columns)]
        into = [_p(g) for g in grads]
        if dh is None:                                                      # the norm before the next block took no part
            for i in (3, 4):
                into[i] = 0
                if grads[i] is not None:
                    grads[i].zero_()
        lib = _library()
        size = lib.sn_block_norms_workspace(rows, width)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        args = _NORM_ARGS.pack(_NORM_ARGS.size, _TYPES[dtype], _param_type(params), rms, rows, width, 0 if n_valid is None else shape[1], _p(n_valid), eps,
                               post_w is not None, pre_w is not None, _p(vx), _p(vb), _p(vg), sx, sb, sg, _p(scale), _p(post_w), _p(post_b), _p(pre_w), _p(pre_b),
                               0, 0, _p(stats), *(codes or (0,) * 6), _p(vy), _p(vh), sy, sh, _p(dx), _p(dbranch), _p(dgate), *into, _p(ws), size)
        _launch(lib.sn_block_norms_backward, "sn_block_norms_backward", dev, args)
        return (dx, dbranch, dgate, *grads, None, None, None, None)


def gated_residual_norms(x, branch, gate=None, scale=None, post=None, pre=None, norm="layer", eps=1e-5, n_valid=None, checkpoint8=False):
    """The end of a residual block and the norm before the next one, as one pass over the rows:

        y = x + scale * sigmoid(gate) * N_post(branch),    h = N_pre(y)          -> (y, h); h is None without `pre`

    x, branch, gate: [..., width] of one type (float32, bfloat16 or float16), width <= 4096; gate None = no gate.
    scale: [width] (a learned residual scale for each feature) or None = 1.
    post, pre: (weight [width], bias [width] or None) or None = no such norm.  norm "layer": LayerNorm, "rms": division by the root of
    the mean square.  All parameters have one type, their own or x's (mixed ones are taken in float32).
    n_valid: int32 [G] with x [G, n, width]: the vertices of graph g from n_valid[g] on are padding - not read, zeros in y and h, no
    gradient.
    checkpoint8: the backward pass keeps x, branch and gate in 8 bits (`checkpoint8`) instead of referring to them; it evaluates the
    gradient's formulas at the kept values, with the row statistics of the forward pass.

    Differentiable in x, branch, gate and all parameters."""
    # (plain tests: a message is only put together where one fails)
    if norm != "layer" and norm != "rms":
        _need(False, "gated_residual_norms: norm must be 'layer' or 'rms', got {!r}", norm)
    if not torch.is_tensor(x) or x.dtype not in _TYPES or x.dim() < 1:
        _need(False, "gated_residual_norms: expected a float32, bfloat16 or float16 tensor")
    autocast = torch.is_autocast_enabled("cuda")
    if autocast:
        x, branch, gate, scale = _autocast(x, branch, gate, scale)
    dtype, shape = x.dtype, x.shape
    width = shape[-1]
    if not 1 <= width <= MAX_NORM_WIDTH:
        _need(False, "gated_residual_norms: width {} outside 1 .. {}", width, MAX_NORM_WIDTH)
    if not torch.is_tensor(branch) or branch.dtype != dtype or branch.shape != shape:
        _need(False, "gated_residual_norms: branch must have x's shape {} and type", tuple(shape))
    if gate is not None and (not torch.is_tensor(gate) or gate.dtype != dtype or gate.shape != shape):
        _need(False, "gated_residual_norms: gate must have x's shape {} and type", tuple(shape))
    params = [scale, None, None, None, None]
    for at, pair in ((1, post), (3, pre)):
        if pair is not None:
            if len(pair) != 2 or not torch.is_tensor(pair[0]):
                _need(False, "gated_residual_norms: {} must be (weight, bias or None)", "post" if at == 1 else "pre")
            params[at], params[at + 1] = _autocast(*pair) if autocast else pair
    types = None
    for i, t in enumerate(params):
        if t is not None:
            if not torch.is_tensor(t) or t.dtype not in _TYPES or t.dim() != 1 or t.shape[0] != width:
                _need(False, "gated_residual_norms: parameters must be [{}]", width)
            types = t.dtype if types is None or types == t.dtype else torch.float64       # (float64: mixed)
            if not t.is_contiguous():
                params[i] = t.contiguous()
    if eps < 0:
        _need(False, "gated_residual_norms: eps {}", eps)
    if n_valid is not None and not (torch.is_tensor(n_valid) and x.dim() == 3 and n_valid.dtype == torch.int32 and n_valid.shape == shape[:1] and n_valid.is_contiguous()):
        _need(False, "gated_residual_norms: n_valid must be int32 [G] with x [G, n, width]")
    _one_device(x, branch, gate, n_valid, *params)
    if types == torch.float64:
        params = [None if t is None else t.float() for t in params]
    if _wants_grad(x, branch, gate, *params):
        out = _GatedResidualNorms.apply(x, branch, gate, *params, norm == "rms", float(eps), n_valid, bool(checkpoint8))
        return out if pre is not None else (out, None)
    return _norms_forward(x, branch, gate, params, norm == "rms", float(eps), n_valid, False, False)[:2]


# -------------------------------------------------------------------------------- log probabilities of given tokens
LabelLogProbs = namedtuple("LabelLogProbs", ["log_probs", "entropy", "top_log_probs", "top_ids"])


def _scores_forward(logits, target, ignore_index, topk, train):
    lib = _library()
    dev, n = logits.device, logits.shape[-1]
    lead = target.shape
    rows = target.numel()
    f32 = dict(dtype=torch.float32, device=dev)
    lp, ent = torch.empty(lead, **f32), torch.empty(lead, **f32)
    stats = torch.empty((rows, 3), **f32) if train else None             # what the backward pass reads
    top_lp = torch.empty((*lead, topk), **f32) if topk else None
    top_ids = torch.empty((*lead, topk), dtype=torch.int64, device=dev) if topk else None
    if rows:
        v, stride = _rows(logits, n)
        size = lib.sn_label_log_probs_workspace(rows, n, topk)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _launch(lib.sn_label_log_probs, "sn_label_log_probs", dev, _p(v), _TYPES[logits.dtype], rows, n, stride, _p(target), ignore_index, topk, _p(lp), _p(ent),
                _p(stats), _p(top_lp), _p(top_ids), _p(ws), size)
    return lp, ent, stats, top_lp, top_ids


class _LabelLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index, topk):
        logits = logits.detach()
        lp, ent, stats, top_lp, top_ids = _scores_forward(logits, target, ignore_index, topk, True)
        ctx.save_for_backward(logits, target, stats)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if not topk:
            return lp, ent
        ctx.mark_non_differentiable(top_lp, top_ids)
        return lp, ent, top_lp, top_ids

    @_once
    def backward(ctx, g_lp, g_ent, *unused):
        logits, target, stats = ctx.saved_tensors
        if g_lp is None and g_ent is None:
            return None, None, None, None
        lib = _library()
        dev, n, rows = logits.device, logits.shape[-1], target.numel()
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        if rows:
            g_lp = None if g_lp is None else g_lp.float().contiguous()
            g_ent = None if g_ent is None else g_ent.float().contiguous()
            v, stride = _rows(logits, n)
            _launch(lib.sn_label_log_probs_backward, "sn_label_log_probs_backward", dev, _p(v), _TYPES[logits.dtype], rows, n, stride, _p(target),
                    ctx.ignore_index, _p(stats), _p(g_lp), _p(g_ent), _p(grad))
        return grad, None, None, None


def label_log_probs(logits, target, topk=0, ignore_index=-100):
    """Log probabilities of given tokens (classes, words) under softmax(logits), the entropy of the distribution and its top alternatives.

    logits [..., n] float32 / bfloat16 / float16, target int64 [...] -> LabelLogProbs of
        log_probs [...] float32: log p[target]; 0 where target == ignore_index, NaN for any other target outside 0 .. n - 1
        entropy [...] float32: -sum p log p (entries at -inf count as 0)
        top_log_probs, top_ids [..., topk]: the topk largest, the lowest index first among equals (None for topk = 0; at most 64)
    log_probs and entropy are differentiable in the logits, the alternatives are not.  A row of -inf only has no distribution: log_probs
    and top_log_probs -inf, entropy 0, no gradient.  A NaN or +inf logit makes its row's results NaN; a row whose upstream gradients are
    zeros (an ignored target) gets zeros, whatever its logits.  Under 2^24 rows of under 2^30 entries."""
    if not torch.is_tensor(logits) or logits.dtype not in _TYPES or logits.dim() < 1:
        _need(False, "label_log_probs: expected float32, bfloat16 or float16 logits")
    if not torch.is_tensor(target) or target.dtype != torch.int64 or target.shape != logits.shape[:-1]:
        _need(False, "label_log_probs: expected an int64 target of shape {}", tuple(logits.shape[:-1]))
    n, topk = logits.shape[-1], int(topk)
    if not (1 <= n < 1 << 30 and target.numel() < 1 << 24):
        _need(False, "label_log_probs: {} rows of {} entries", target.numel(), n)
    if not 0 <= topk <= min(n, MAX_ALTERNATIVES):
        _need(False, "label_log_probs: {} alternatives of {} entries (at most {})", topk, n, MAX_ALTERNATIVES)
    _one_device(logits, target)
    logits, = _autocast(logits)
    target = target.contiguous()
    if _wants_grad(logits):
        out = _LabelLogProbs.apply(logits, target, int(ignore_index), topk)
        return LabelLogProbs(*out) if topk else LabelLogProbs(*out, None, None)
    lp, ent, _, top_lp, top_ids = _scores_forward(logits, target, int(ignore_index), topk, False)
    return LabelLogProbs(lp, ent, top_lp, top_ids)
