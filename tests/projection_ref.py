"""64-bit restatements of the projection operators with element-wise error bounds.

A bound counts what the kernels may lose: half a step of the output's type, half a step of each
value that is rounded to the inputs' type on the way to the tensor cores (plus half the smallest
subnormal of f16), and the f32 sums: K products accumulated in f32, whose steps may truncate,
are off by at most K * 2^-23 of the sum of their absolute values.  The activations' f32
evaluation is counted with 2^-19 of their value's scale (a few units of __expf and division)."""
import math

import torch

SUM = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest subnormal (f16 2^-25; bf16's is negligible)."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134


def act_ref(g, kind):
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if kind == "gelu":
        phi = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k, c = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(k * (g + c * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * c * g * g)


def gated_ref(x, wg, wu, kind, dh=None):
    """[(value, bound)] of h, or of h, dx, dwg, dwu."""
    dt = x.dtype
    e, z = half_step(dt), tiny(dt)
    T, H = x.shape
    I = wg.shape[0]
    X, G, U = x.double(), wg.double(), wu.double()
    g, u = X @ G.t(), X @ U.t()
    eg, eu = H * SUM * (X.abs() @ G.abs().t()), H * SUM * (X.abs() @ U.abs().t())
    a, da = act_ref(g, kind)
    ea = 1.2 * eg + 2.0 ** -19 * (g.abs() + a.abs())   # |act'| < 1.2
    eda = 1.2 * eg + 2.0 ** -19 * (1 + g.abs())         # |act''| < 1.2
    h = a * u
    out = [(h, e * h.abs() + (1 + e) * (ea * u.abs() + a.abs() * eu + ea * eu) + z)]
    if dh is None:
        return out
    D = dh.double()
    dg, du = D * u * da, D * a
    edg = D.abs() * (u.abs() * eda + da.abs() * eu + eu * eda)
    edu = D.abs() * ea
    edg, edu = edg + e * (dg.abs() + edg) + z, edu + e * (du.abs() + edu) + z
    dx = dg @ G + du @ U
    ax = (dg.abs() + edg) @ G.abs() + (du.abs() + edu) @ U.abs()
    out.append((dx, e * dx.abs() + (1 + e) * (edg @ G.abs() + edu @ U.abs() + 2 * I * SUM * ax) + z))
    for d, ed in ((dg, edg), (du, edu)):
        dw = d.t() @ X
        out.append((dw, e * dw.abs() + (1 + e) * (ed.t() @ X.abs() + T * SUM * ((d.abs() + ed).t() @ X.abs())) + z))
    return out


def lora_ref(x, w, a, b, idx, scale=None):
    """(value, bound) of y."""
    dt = x.dtype
    e, z = half_step(dt), tiny(dt)
    K, r = x.shape[1], a.shape[1]
    X, W = x.double(), w.double()
    y = X @ W.t()
    err = (K + r) * SUM * (X.abs() @ W.abs().t())
    for k in range(a.shape[0]):
        rows = (idx == k).nonzero().flatten()
        if rows.numel() == 0:
            continue
        s = 1.0 if scale is None else float(scale[k])
        A, B, xr = a[k].double(), b[k].double(), X[rows]
        v = s * (xr @ A.t())
        ev = abs(s) * K * SUM * (xr.abs() @ A.abs().t()) + 2.0 ** -23 * v.abs()
        ev = ev + e * (v.abs() + ev) + z
        y[rows] += v @ B.t()
        err[rows] += ev @ B.abs().t() + (K + r) * SUM * ((v.abs() + ev) @ B.abs().t())
    return y, e * y.abs() + (1 + e) * err + z


def check(got, ref, what=""):
    val, bound = ref
    assert got.shape == val.shape, (what, got.shape, val.shape)
    over = (got.double() - val).abs() / bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 1.0 and not torch.isnan(over).any(), (what, worst, (over > 1).sum().item(), over.numel())
