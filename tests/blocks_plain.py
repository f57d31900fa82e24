"""Definitions in float64 of the operators of include/schemanet_blocks.h, and the magnitudes their error bounds are made of."""
import torch

U = 2.0 ** -24                                    # half a step of float32, relative
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def kept64(x):
    """the values of an 8-bit checkpoint of x [..., n] (float64): blocks of 32, the smallest power of two step with max < 127.5 step"""
    out = torch.zeros_like(x)
    for a in range(0, x.shape[-1], 32):
        v = x[..., a:a + 32]
        top = v.abs().amax(-1, keepdim=True)
        bad = ~torch.isfinite(top)
        k = torch.floor(torch.log2(torch.where((top > 0) & ~bad, top, torch.ones_like(top)))) - 8
        step = torch.exp2(k)
        for _ in range(4):
            step = torch.where(top >= 127.5 * step, step * 2, step)
        step = step.clamp(min=2.0 ** -125, max=2.0 ** 121)
        q = torch.round(v / step).clamp(-127, 127) * step
        out[..., a:a + 32] = torch.where(bad, torch.full_like(q, float("nan")), q)
    return out


class Norms64:
    """y, h and every gradient on [rows, width] float64 tensors; `kept`: the backward pass's view of x, f, z (default: themselves).
    For each result r, r_mag is the formula with absolute values: what a rounding error anywhere in it is relative to."""

    def __init__(self, x, f, z, scale, post, pre, norm, eps, dy=None, dh=None, kept=None):
        E = x.shape[-1]
        one, zero = torch.ones(E, dtype=x.dtype, device=x.device), torch.zeros(E, dtype=x.dtype, device=x.device)
        sc = one if scale is None else scale
        w1, b1 = (one, zero) if post is None else (post[0], zero if post[1] is None else post[1])
        w2, b2 = (one, zero) if pre is None else (pre[0], zero if pre[1] is None else pre[1])
        mean = (lambda v: v.mean(-1, keepdim=True))          # noqa: E731

        def stats(v):
            mu = mean(v) if norm == "layer" else torch.zeros_like(v[..., :1])
            return mu, 1 / torch.sqrt(mean((v - mu) ** 2) + eps)

        def forward(x, f, z, s1=None, s2=None):
            s = torch.ones_like(x) if z is None else torch.sigmoid(z)
            if post is not None:
                s1 = stats(f) if s1 is None else s1
                n1 = (f - s1[0]) * s1[1]
                # the mean's rounding error shows as a shift of every unit value by a share of the row's root mean square
                n1_mag = n1.abs() + torch.sqrt(mean(f * f)) * s1[1]
            else:
                s1, n1, n1_mag = (torch.zeros_like(x[..., :1]), torch.ones_like(x[..., :1])), f, f.abs()
            p, p_mag = n1 * w1 + b1, n1_mag * w1.abs() + b1.abs()
            y, y_mag = x + sc * s * p, x.abs() + sc.abs() * s * p_mag
            s2 = stats(y) if s2 is None and pre is not None else s2
            if pre is not None:
                n2 = (y - s2[0]) * s2[1]
                n2_mag = (y_mag + torch.sqrt(mean(y_mag ** 2))) * s2[1] + n2.abs() * (1 + mean(n2.abs() * y_mag) * s2[1])
            else:
                n2 = n2_mag = None
            return s, s1, n1, n1_mag, p, p_mag, y, y_mag, s2, n2, n2_mag
        s, s1, n1, n1_mag, p, p_mag, self.y, self.y_mag, s2, n2, n2_mag = forward(x, f, z)
        self.h = self.h_mag = None
        if pre is not None:
            self.h, self.h_mag = n2 * w2 + b2, n2_mag * w2.abs() + b2.abs()
        if dy is None and dh is None:
            return
        if kept is not None:
            s, _, n1, n1_mag, p, p_mag, _, _, _, n2, n2_mag = forward(*kept, s1, s2)
        u = torch.zeros_like(x) if dy is None else dy
        u_mag = u.abs()
        centre = mean if norm == "layer" else (lambda v: torch.zeros_like(v[..., :1]))      # noqa: E731
        if dh is not None:
            d, d_mag = dh * w2, (dh * w2).abs()
            u = u + s2[1] * (d - centre(d) - n2 * mean(d * n2))
            u_mag = u_mag + s2[1] * (d_mag + mean(d_mag) + 2 * n2_mag * mean(d_mag * n2_mag))
            self.dpre_w, self.dpre_w_mag = (dh * n2).sum(0), (dh.abs() * n2_mag).sum(0)
            self.dpre_b, self.dpre_b_mag = dh.sum(0), dh.abs().sum(0)
        self.dx, self.dx_mag = u, u_mag
        self.dscale, self.dscale_mag = (u * s * p).sum(0), (u_mag * s * p_mag).sum(0)
        self.dgate, self.dgate_mag = u * sc * p * s * (1 - s), u_mag * sc.abs() * p_mag * s
        dp, dp_mag = u * sc * s, u_mag * sc.abs() * s
        self.dpost_w, self.dpost_w_mag = (dp * n1).sum(0), (dp_mag * n1_mag).sum(0)
        self.dpost_b, self.dpost_b_mag = dp.sum(0), dp_mag.sum(0)
        self.dbranch, self.dbranch_mag = dp, dp_mag
        if post is not None:
            d, d_mag = dp * w1, dp_mag * w1.abs()
            self.dbranch = s1[1] * (d - centre(d) - n1 * mean(d * n1))
            self.dbranch_mag = s1[1] * (d_mag + mean(d_mag) + 2 * n1_mag * mean(d_mag * n1_mag))


def scores64(logits, target, ignore=-100):
    """-> log p of the targets, entropy, all log p (rows without a finite entry: -inf, 0)"""
    x = logits.double()
    dead = (x == float("-inf")).all(-1, keepdim=True)
    d = x - torch.where(dead, torch.zeros_like(x[..., :1]), x.amax(-1, keepdim=True))       # (first: at 1e38 a logarithm would be lost in x)
    lp = torch.where(dead, torch.full_like(x, float("-inf")), d - torch.log(torch.exp(d).sum(-1, keepdim=True)))
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    used = target != ignore
    wrong = used & ((target < 0) | (target >= x.shape[-1]))
    at = target.clamp(0, x.shape[-1] - 1)
    got = lp.gather(-1, at[..., None])[..., 0]
    got = torch.where(used, got, torch.zeros_like(got))
    return torch.where(wrong, torch.full_like(got, float("nan")), got), ent, lp


def check(got, want, bound, what):
    """|got - want| <= bound elementwise, NaN exactly where NaN is wanted"""
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    same = (got == want) | torch.isnan(want)
    off = torch.where(same, torch.zeros_like(got), (got - want).abs() - bound)
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"{what}: {float(got.reshape(-1)[worst])} for {float(want.reshape(-1)[worst])}, allowed {float((bound + torch.zeros_like(got)).reshape(-1)[worst])}"
