"""Tensor-level wrappers of include/schemanet_blocks.h, re-exported by `cpp_extension.ops`: the operators of deep residual graph
networks (`gated_residual_norms`), of activations kept in 8 bits for the backward pass (`checkpoint8`, `checkpoint8_weight_grad`,
`linear_checkpoint8`) and of large sets of answers (`label_log_probs`).

They take CUDA tensors in float32, bfloat16 or float16 with rows of any stride, compute in float32 and round each result
once; outputs are new contiguous tensors; nothing synchronises, all of them can be captured into a graph.  Under `torch.autocast`
`gated_residual_norms`, `linear_checkpoint8` and `label_log_probs` cast their floating-point inputs to float32, like the other HIP-backed
ops of this package; `checkpoint8` and `checkpoint8_weight_grad` keep the types that they are given.  Arguments that do not
fit raise RuntimeError before anything is launched; tensors with a forward-mode tangent, which would be lost, raise
NotImplementedError.

Checks, buffers, launches and autograd nodes are C++ (csrc/sn_torch.cpp): a small call is bound by its host part."""
import math
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N


def _need(ok, message, *args):
    if not ok:
        raise RuntimeError(message.format(*args))


def _once(backward):
    """a backward pass without second derivatives: the wrapper that says so on their use is only taken under create_graph"""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(run)


def _autocast(*ts):
    if not torch.is_autocast_enabled("cuda"):
        return ts
    return tuple(t.float() if torch.is_tensor(t) and t.is_floating_point() and t.is_cuda else t for t in ts)


# ------------------------------------------------------------------------------------------- activations kept in 8 bits
class Checkpoint8:
    """An activation [..., n] kept in 8 bits: `codes` int8 [rows, npad] and `exps` uint8 [rows, npad / 32], npad = n rounded up to a
    multiple of 32.  A block of 32 features shares one power of two s, the smallest with max|x| < 127.5 s, and an element is kept
    as round(x / s) (half to even): off by at most s / 2 <= max|x| / 127.5, up to max|x| / 254 where the maximum is just under
    127.5 s.  A block that held an infinity or a NaN comes back as NaN; magnitudes under 2^-126 as zero."""

    __slots__ = ("_codes", "_exps", "_shape", "dtype")

    def __init__(self, codes, exps, shape, dtype):
        # (none of the three can be replaced later; what happens to the tensors in place is checked at each use)
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
        """the kept values, [..., n] in `dtype` (default: the type of the activation).  bfloat16 and float32 hold them exactly; float16 rounds
        them and takes those beyond its largest to +-65504: 8 bits keep 65024 .. 65504 as 65536, and no finite activation comes back infinite"""
        return N.blocks().restore(self._codes, self._exps, self._shape, dtype or self.dtype)


def checkpoint8(x):
    """x [..., n] float32 / bfloat16 / float16 (CUDA) -> Checkpoint8, 1 + 1/32 bytes an element, up to 2^30 features.  No autograd:
    what a backward pass keeps."""
    codes, exps = N.blocks().checkpoint8(x)
    return Checkpoint8._of(codes, exps, x.shape, x.dtype)


def checkpoint8_weight_grad(dy, kept, bias=True, out_dtype=None):
    """The gradients of y = x W^T + b with respect to W and b from the kept activation: dy [..., out] of float32, bfloat16 or float16,
    kept = checkpoint8(x) of x [..., in] with the same leading sizes -> (dW [out, in], db [out] or None); in and out up to 2^20,
    under 2^31 rows.

    dW = sum_r dy[r]^T kept[r] on the bf16 matrix cores with float32 sums.  The kept values are exact in bf16 and dy enters as
    bf16 pieces that add up to it (float32: three, float16: two), so the products carry no rounding of their own.  A gradient that is
    infinite or NaN (float32: or beyond bfloat16's largest, 3.39e38) makes its feature's row of dW infinite or NaN.  No autograd: the
    results carry no history of dy, and a dy with a forward-mode tangent is refused.
    out_dtype: the type of both results (default dy's)."""
    _need(isinstance(kept, Checkpoint8), "checkpoint8_weight_grad: expected a Checkpoint8, got {}", type(kept).__name__)
    return N.blocks().weight_grad(dy, kept._codes, kept._exps, kept._shape, bias, out_dtype)


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
    for t in (x, weight, bias):
        _need(t is None or t.is_cuda, "expected CUDA tensors (the HIP path has no CPU fallback)")
        _need(t is None or t.device == x.device, "tensors on different devices: {} vs {}", x.device, None if t is None else t.device)
    N.blocks().before_capture(x, weight, bias)
    return _LinearCheckpoint8.apply(x, weight, bias)


# ------------------------------------------------------------- the end of a residual block and the norm before the next one
def _norm_pair(pair, name):
    if pair is None:
        return None, None
    if len(pair) != 2 or not torch.is_tensor(pair[0]):
        _need(False, "gated_residual_norms: {} must be (weight, bias or None)", name)
    return pair


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
    if norm != "layer" and norm != "rms":
        _need(False, "gated_residual_norms: norm must be 'layer' or 'rms', got {!r}", norm)
    post_w, post_b = _norm_pair(post, "post")
    pre_w, pre_b = _norm_pair(pre, "pre")
    if torch.is_autocast_enabled("cuda"):
        x, branch, gate, scale, post_w, post_b, pre_w, pre_b = _autocast(x, branch, gate, scale, post_w, post_b, pre_w, pre_b)
    return N.blocks().gated_residual_norms(x, branch, gate, scale, post_w, post_b, pre_w, pre_b, norm == "rms", eps, n_valid, checkpoint8)


# -------------------------------------------------------------------------------- log probabilities of given tokens
LabelLogProbs = namedtuple("LabelLogProbs", ["log_probs", "entropy", "top_log_probs", "top_ids"])


def label_log_probs(logits, target, topk=0, ignore_index=-100):
    """Log probabilities of given tokens (classes, words) under softmax(logits), the entropy of the distribution and its top alternatives.

    logits [..., n] float32 / bfloat16 / float16, target int64 [...] -> LabelLogProbs of
        log_probs [...] float32: log p[target]; 0 where target == ignore_index, NaN for any other target outside 0 .. n - 1
        entropy [...] float32: -sum p log p (entries at -inf count as 0)
        top_log_probs, top_ids [..., topk]: the topk largest, the lowest index first among equals (None for topk = 0; at most 64)
    log_probs and entropy are differentiable in the logits, the alternatives are not.  A row of -inf only has no distribution: log_probs
    and top_log_probs -inf, entropy 0, no gradient.  A NaN or +inf logit makes its row's results NaN; a row whose upstream gradients are
    zeros (an ignored target) gets zeros, whatever its logits.  Under 2^24 rows of under 2^30 entries."""
    if torch.is_autocast_enabled("cuda"):
        logits, = _autocast(logits)
    return LabelLogProbs(*N.blocks().label_log_probs(logits, target, int(topk), int(ignore_index)))
