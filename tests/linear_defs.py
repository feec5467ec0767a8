"""The linear-layer and gradient-list routines from their definitions in 64 bits, and error bounds
derived from the number of roundings. Shared by the GPU tests of those routines.

Bounds. u = eps/2 of the element type is the most one rounding to it moves a value, relative to the
value (plus half the smallest subnormal). A sum of n products in FP32 moves by at most
(n + 8) * 2^-23 times the sum of the magnitudes: every addition loses at most one unit in the last
place (the tensor core truncates) and there are at most n of them beside a few scalings. The
activations have slopes of at most 1.13, and are computed in FP32 with an error below 2^-18 of
max(|value|, |slope argument| stays below 30): 16 units in the last place of FP32 cover __expf's
2 + 1.17 |x| up to |x| = 12 and the values beyond that are below 1e-4; 2^-18 is 64 of them.
"""
import math

import torch

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
SLOPE = 1.13
F_ERR = 2.0 ** -18


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the smallest subnormal of the type (BF16 and FP32: nothing that matters here)."""
    return 2.0 ** -25 if dt == torch.float16 else 1e-38


def act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if name == "silu":
        g = torch.sigmoid(z)
        return g * (1.0 + z * (1.0 - g))
    return torch.ones_like(z)


class Mat:
    """A column-major rows x cols matrix in a buffer of its own: `ld` >= rows entries a column, the first
    column `offset` elements behind an aligned address, everything around the matrix NaN."""

    def __init__(self, rows, cols, dt, pad=0, offset=0, device="cuda"):
        self.rows, self.cols, self.dt = rows, cols, dt
        self.ld = max(1, rows) + pad
        self.buf = torch.full((offset + self.ld * max(cols, 1) + 8,), float("nan"), dtype=dt, device=device)
        self.t = torch.as_strided(self.buf, (rows, cols), (1, self.ld), offset)     # entry (i, j)
        self.addr = self.buf[offset:]

    def set(self, values):
        self.t.copy_(values)
        return self

    @property
    def m(self):
        return self.t.double()

    def outside_untouched(self):
        """Whether everything around the matrix is still NaN."""
        mask = torch.ones_like(self.buf, dtype=torch.bool)
        torch.as_strided(mask, (self.rows, self.cols), (1, self.ld), self.buf.numel() - self.addr.numel()).fill_(False)
        return bool(torch.isnan(self.buf[mask]).all())


def op(m, flag):
    return m.T if flag in "TtCc" else m


def rand(gen, rows, cols, scale=1.0):
    return torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.float32) * scale


def forward_want(A, B, ta, tb, alpha, bias, name, beta, C, dt):
    """(D, pre, tolerance of D, tolerance of pre) in 64 bits."""
    a, b = op(A, ta), op(B, tb)
    K = a.shape[1]
    z = alpha * (a @ b)
    mag = abs(alpha) * (a.abs() @ b.abs())
    if bias is not None:
        z = z + bias.double()[:, None]
        mag = mag + bias.double().abs()[:, None]
    zerr = (K + 8) * 2.0 ** -23 * mag
    v = act(z, name)
    d, u = v, half_step(dt)
    extra = F_ERR * v.abs() + SLOPE * zerr
    if beta:
        d = d + beta * C
        extra = extra + 2.0 ** -22 * (v.abs() + (beta * C).abs())
    return (d, z, u * (d.abs() + extra) + extra + tiny(dt) + 1e-30,
            u * (z.abs() + zerr) + zerr + tiny(dt) + 1e-30)


def grad_want(A, B, ta, tb, alpha, name, pre, dD, dt):
    """{name: (value, tolerance)} for dA, dB, dbias."""
    a, b = op(A, ta), op(B, tb)
    u = half_step(dt)
    dz = dD * slope(pre, name) if name != "none" else dD
    # what dZ is off: the slope's evaluation, then its rounding
    slope_err = F_ERR * SLOPE * dD.abs() if name not in ("none", "relu") else torch.zeros_like(dD)
    round_err = u * dz.abs() + tiny(dt) if name not in ("none", "relu") else torch.zeros_like(dD)
    dz_err = slope_err * (1 + u) + round_err
    out = {}
    for key, x, y, xe, ye, flag in (("dA", dz, b.T, dz_err, None, ta), ("dB", a.T, dz, None, dz_err, tb)):
        n = x.shape[1]
        v = alpha * (x @ y)
        mag = abs(alpha) * (x.abs() @ y.abs())
        prop = abs(alpha) * ((xe @ y.abs()) if xe is not None else (x.abs() @ ye))
        err = (n + 8) * 2.0 ** -23 * (mag + prop) + prop
        tol = u * (v.abs() + err) + err + tiny(dt) + 1e-30
        out[key] = (v.T, tol.T) if flag in "TtCc" else (v, tol)
    s = dz.sum(dim=1)
    err = (dz.shape[1] + 8) * 2.0 ** -23 * dz.abs().sum(dim=1) + slope_err.sum(dim=1)
    out["dbias"] = (s, u * (s.abs() + err) + err + tiny(dt) + 1e-30)
    return out


def check(got, want, tol, what):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} entries off, first at {i}: "
                             f"got {float(got[i])}, want {float(want[i])} +- {float(tol[i])}")
