"""A layer's norms and products in 64 bits (numpy), how far a kernel's results may be from them, and the buffers that their tests share."""
import math

import numpy as np
import torch

from mimir_framework_b200 import abi, runtime as rt
from serving_ref import TORCH, half_step

ACTS = {"none": -1, "gelu": abi.ELT_GELU, "silu": abi.ELT_SILU, "relu": abi.ELT_RELU, "tanh": abi.ELT_TANH, "sigmoid": abi.ELT_SIGMOID}


def d(t):
    return t.double().cpu().numpy()


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def padded(t, wide, fill=float("nan"), lead=0):
    """t's rows `wide` elements apart (after `lead` of them); everything between holds rubbish."""
    rows, n = t.shape
    raw = torch.full((lead + rows * wide + 64,), fill, device=t.device).to(t.dtype)
    view = raw[lead : lead + rows * wide].view(rows, wide)[:, :n]
    view.copy_(t)
    return view


# ---- norms --------------------------------------------------------------------------------------------------------------------------
def norm_rows(x, residual, gamma, norm, eps):
    """s and v."""
    s = x if residual is None else x + residual
    v = s
    if norm:
        v = s / np.sqrt((s * s).mean(1, keepdims=True) + eps)
        v = v if gamma is None else v * gamma
    return s, v


def e4m3_half_step(q):
    """Half of the distance of neighbouring codes at |q|."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(q), 2.0**-6))) - 4)


# A sum of squares is a product and three fmas, joined in at most 8 + 1 + 5 + 4 additions of positive numbers; with the squares' own relative error (twice
# s's 2^-24), 1 / n's and the fma with eps 26 units of 2^-24, halved by the root; the root (1.5), s (1) and two products (2): 17.5 units.
NORM_UNITS = 17.5 * 2.0**-24


# ---- products -------------------------------------------------------------------------------------------------------------------------
class Operand:
    """Rows of a product's operand with rubbish between them; 8-bit ones have a scale a row."""

    def __init__(self, rows, n, type_, seed, scale=1.0, extra=0):
        unit = 16 if type_ == abi.T_E4M3 else 8
        wide = -(-n // unit) * unit + extra * unit
        self.scale = None
        if type_ == abi.T_E4M3:
            self.x = padded(normal(rows, n, seed=seed, scale=100.0).clamp_(-448, 448).to(TORCH[type_]), wide)
            self.scale = (0.5 + torch.rand(rows, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")) * (scale / 100.0)
        else:
            self.x = padded(normal(rows, n, seed=seed, scale=scale, dtype=TORCH[type_]), wide)
        self.stride = wide

    @property
    def value(self):
        v = d(self.x)
        return v if self.scale is None else v * d(self.scale)[:, None]

    def at(self):
        return self.x.data_ptr()

    def scale_at(self):
        return None if self.scale is None else self.scale.data_ptr()


def act(z, name):
    if name == "gelu":
        return z * 0.5 * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    if name in ("silu", "sigmoid"):
        with np.errstate(over="ignore"):
            return (z if name == "silu" else 1) / (1 + np.exp(-z))
    return np.maximum(z, 0) if name == "relu" else np.tanh(z) if name == "tanh" else z


def sums_lose(n_in, type_, out_type):
    """What a product's sum may be off by, in parts of the sum of its terms' magnitudes: an instruction adds 16 (E4M3: 32) products to the running
    sum by truncation, up to 2^-22 of the magnitudes (2^-23 of the sum, and as much among its terms); results of F32 begin anew every 256 and add
    up rounded.  Parts of n_in meet in up to 16 rounded additions."""
    step = 32 if type_ == abi.T_E4M3 else 16
    if out_type == abi.T_F32:
        return math.ceil(256 / step) * 2.0**-22 + (math.ceil(n_in / 256) + 16) * 2.0**-24
    return math.ceil(n_in / step) * 2.0**-22 + 16 * 2.0**-24


def product(x, w, bias, type_, out_type):
    """z and how far it may be off: the sums, two scales and the bias a rounding each."""
    xv, wv = x.value, w.value
    z, size = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    b = 0.0 if bias is None else d(bias)
    off = size * (sums_lose(xv.shape[1], type_, out_type) + 2 * 2.0**-24) + (size + np.abs(b)) * 2.0**-24
    return z + b, off


def act_off(z, off, name):
    """Slopes are at most 1.13; an activation's own arithmetic is off by 2^-20 and, for its exponent, 2^-22 of its argument's size, of its value."""
    a = np.abs(act(z, name))
    if name in ("none", "relu"):
        return off
    return 1.13 * off + a * (2.0**-20 + 2.0**-22 * (np.abs(z) + 0.1 * np.abs(z) ** 3)) + 1e-35


def rounded(y, off, out_type):
    return off + (np.abs(y) + off) * half_step(out_type) * 1.001 + (2.0**-25 if out_type == abi.T_F16 else 1e-40)


def linear_args(x, w, out, type_, out_type, rows, n_in, n_out, **more):
    a = dict(x=x.at(), w=w.at(), out=out.data_ptr(), rows=rows, n_in=n_in, n_out=n_out, type=type_, out_type=out_type, x_stride=x.stride, w_stride=w.stride,
             out_stride=out.stride(0), x_scale=x.scale_at(), w_scale=w.scale_at())
    return rt.linear(**(a | more))


def check_product(backend, rows, n_in, n_out, type_, out_type, name="none", bias=True, residual=False, gated=False, seed=0, out_wide=None, lead=0, in_place=False,
                  stream=0):
    """One call against its definition; nothing around the result is touched."""
    x, w = Operand(rows, n_in, type_, seed, 1.0, extra=1), Operand(n_out, n_in, type_, seed + 1, 1 / math.sqrt(n_in))
    b = normal(n_out, seed=seed + 2) if bias else None
    t = TORCH[out_type]
    out_wide = out_wide or n_out + 3
    raw = torch.full((lead + (rows + 1) * out_wide,), -7.0, dtype=t, device="cuda")
    out = raw[lead:].view(rows + 1, out_wide)
    res = normal(rows, n_out, seed=seed + 3, dtype=t) if residual else None
    more = dict(bias=None if b is None else b.data_ptr(), activation=ACTS[name])
    if residual:
        if in_place:
            out[:rows, :n_out] = res
            more |= dict(residual=out.data_ptr(), residual_stride=out.stride(0))
        else:
            more |= dict(residual=res.data_ptr(), residual_stride=n_out)
    z, off = product(x, w, b, type_, out_type)
    y, off = act(z, name), act_off(z, off, name)
    if gated:
        u = Operand(n_out, n_in, type_, seed + 4, 1 / math.sqrt(n_in), extra=2)
        ub = normal(n_out, seed=seed + 5) if bias else None
        more |= dict(up=u.at(), up_stride=u.stride, up_scale=u.scale_at(), up_bias=None if ub is None else ub.data_ptr())
        z2, off2 = product(x, u, ub, type_, out_type)
        off = off * (np.abs(z2) + off2) + np.abs(y) * off2 + np.abs(y * z2) * 2.0**-24
        y = y * z2
    elif residual:
        y = y + d(res)
        off = off + np.abs(y) * 2.0**-24
    a = linear_args(x, w, out, type_, out_type, rows, n_in, n_out, **more)
    (backend.dev_gated_linear if gated else backend.dev_linear)(a, stream)
    torch.cuda.synchronize()
    backend.check_device()
    got = d(out)
    err, bound = np.abs(got[:rows, :n_out] - y), rounded(y, off, out_type)
    assert np.all(err <= bound), f"{(err / bound).max()} of the bound at {np.unravel_index(np.argmax(err / bound), err.shape)}"
    assert (got[:rows, n_out:] == -7).all() and (got[rows] == -7).all() and (raw[:lead] == -7).all()
    return out[:rows, :n_out]
