"""64-bit references of the packed-training operators (torch on the CPU), and how far an
f32 result may be from them.

Bounds are first-order sums of the roundings on the way, u = 2^-24 an f32 rounding:
 - a product of two f32 values is held to W = 2^-21 of it: the kernels may carry an operand
   in two 11-bit parts (an error of at most 2^-22 each, and 2^-22 for the dropped product
   of the small parts: 3 * 2^-22 < W);
 - a sum of K terms adds at most K u of the sum of their magnitudes;
 - exp(x) with x off by e is off by 2 e relatively, for the small e here (e^e - 1 < 2 e).
"""
import ctypes

import numpy as np
import torch

U = 2.0 ** -24
W = 2.0 ** -21


def f64(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.float64)


class Buf:
    """An f32 [T, H, D] view of a device buffer with a layout of choice, every float of the
    buffer outside the view (and the view itself, for an output) set to `around`."""

    def __init__(self, vh, a, kind="plain", around=-777.0, dev=None):
        T, H, D = a.shape
        off, st, sh = {"plain": (0, H * D, D), "cols": (8, H * D + 24, D), "odd": (3, H * (D + 1) + 2, D + 1),
                       "heads_first": (4, D, T * D + 8)}[kind]
        n = off + max(0, (T - 1)) * st + max(0, (H - 1)) * sh + D + 16
        self.idx = off + np.arange(T)[:, None, None] * st + np.arange(H)[None, :, None] * sh + np.arange(D)
        self.host = np.full(n, around, np.float32)
        if dev is None:
            self.host[self.idx] = a
        self.vh, self.shape = vh, a.shape
        self.dev = vh.DeviceBuffer.from_array(self.host)
        self.ptr = self.dev.ptr + 4 * off
        self.lay = vh.layout([T, H, D], [st, sh, 1])
        self.l = ctypes.byref(self.lay)

    def get(self):
        """The view's values; everything around it must be as it was."""
        now = self.dev.to_array(self.host.shape)
        left = np.ones(now.shape, bool)
        left[self.idx.reshape(-1)] = False
        np.testing.assert_array_equal(now[left], self.host[left], err_msg="written outside the view")
        return now[self.idx]


def like(vh, shape, kind="plain"):
    return Buf(vh, np.empty(shape, np.float32), kind, dev=True)


# ---------------------------------------------------------------- attention --

def attention(q, k, v, do, lens, scale, causal, first=0):
    """out, lse, dq, dk, dv in 64 bits over [T, H, D] arrays, sequences of `lens` from token
    `first` on, and the bound of each. Rows in no sequence are NaN."""
    q, k, v, do = (f64(x) for x in (q, k, v, do))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    val = {n: torch.full_like(x, float("nan")) for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    val["lse"] = torch.full((Hq, T), float("nan"), dtype=torch.float64)
    tol = {n: x.clone() for n, x in val.items()}
    t0 = first
    for L in lens:
        s = slice(t0, t0 + L)
        t0 += L
        if L == 0:
            continue
        for n in ("dk", "dv"):
            val[n][s] = 0
            tol[n][s] = 0
        mask = torch.ones(L, L, dtype=torch.bool).tril() if causal else torch.ones(L, L, dtype=torch.bool)
        for h in range(Hq):
            Q, K, V, G_ = q[s, h], k[s, h // G], v[s, h // G], do[s, h]
            z = torch.where(mask, scale * (Q @ K.T), -torch.inf)
            mag = torch.where(mask, scale * (Q.abs() @ K.abs().T), 0.0)
            lse = torch.logsumexp(z, 1)
            P = torch.exp(z - lse[:, None])
            O = P @ V
            e = (mag * (W + (D + 4) * U)).amax(1)  # a row's largest score error
            d = 2 * e + (4 * lse.abs() + 8 + L) * U  # P, relatively
            eo = (P @ V.abs()) * (2 * d[:, None] + W + (L + 4) * U)
            val["o"][s, h], tol["o"][s, h] = O, eo
            val["lse"][h, s], tol["lse"][h, s] = lse, e + 2 * U * lse.abs() + (L + 8) * U
            delta = (G_ * O).sum(1)
            edel = (G_.abs() * O.abs()).sum(1) * (D + 1) * U + (G_.abs() * eo).sum(1)
            dP = G_ @ V.T
            edP = (G_.abs() @ V.abs().T) * (W + (D + 1) * U)
            dS = P * (dP - delta[:, None])
            edS = P * (d[:, None] * (dP.abs() + delta.abs()[:, None]) + edP + edel[:, None]) + dS.abs() * 4 * U
            # dS in two parts under a scale of its row's or column's largest: 2^-30 of that.
            flo = dS.abs().amax(1, keepdim=True) + dS.abs().amax(0, keepdim=True)
            edS = edS + torch.where(mask, 2.0 ** -30 * flo, 0.0)
            val["dq"][s, h] = scale * (dS @ K)
            tol["dq"][s, h] = scale * (edS @ K.abs() + (dS.abs() @ K.abs()) * (W + (L + 4) * U))
            val["dk"][s, h // G] += scale * (dS.T @ Q)
            tol["dk"][s, h // G] += scale * (edS.T @ Q.abs() + (dS.abs().T @ Q.abs()) * (W + (G * L + 4) * U))
            val["dv"][s, h // G] += P.T @ G_
            tol["dv"][s, h // G] += (P * d[:, None]).T @ G_.abs() + (P.T @ G_.abs()) * (W + (G * L + 4) * U) \
                + 2.0 ** -30 * G_.abs().amax(0)
    return {n: x.numpy() for n, x in val.items()}, {n: x.numpy() for n, x in tol.items()}


def starts_of(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int32)


class Attention:
    """One call of the forward, or of forward and backward, with buffers of its own."""

    def __init__(self, vh, q, k, v, do, starts, scale, causal, kinds=("plain",) * 4, okind="plain", around=-777.0):
        self.vh, self.scale, self.causal = vh, scale, causal
        self.q, self.k, self.v, self.do = (Buf(vh, x, c, around) for x, c in zip((q, k, v, do), kinds))
        self.starts = vh.DeviceBuffer.from_array(np.asarray(starts, np.int32))
        self.n = len(starts) - 1
        self.o, self.dq = like(vh, q.shape, okind), like(vh, q.shape, okind)
        self.dk, self.dv = like(vh, k.shape, okind), like(vh, k.shape, okind)
        self.lse_shape = (q.shape[1], q.shape[0])
        self.lse = vh.DeviceBuffer.from_array(np.full(self.lse_shape, -777.0, np.float32))
        self.sizes = (q.shape[0], self.n, q.shape[1], k.shape[1], q.shape[2])

    def args(self):
        return (self.q.ptr, self.q.l, self.k.ptr, self.k.l, self.v.ptr, self.v.l, self.starts.ptr, self.n, self.scale,
                int(self.causal))

    def forward(self, scratch=None, stream=None):
        p, nb = (scratch.ptr, scratch.nbytes) if scratch else (None, 0)
        self.vh.check(self.vh.lib.vh_packed_attention_fwd(*self.args(), self.o.ptr, self.o.l, self.lse.ptr, p, nb, stream))

    def backward(self, scratch=None, stream=None):
        p, nb = (scratch.ptr, scratch.nbytes) if scratch else (None, 0)
        self.vh.check(self.vh.lib.vh_packed_attention_bwd(
            *self.args(), self.o.ptr, self.o.l, self.lse.ptr, self.do.ptr, self.do.l, self.dq.ptr, self.dq.l, self.dk.ptr,
            self.dk.l, self.dv.ptr, self.dv.l, p, nb, stream))

    def results(self):
        self.vh.sync()
        return {"o": self.o.get(), "lse": self.lse.to_array(self.lse_shape), "dq": self.dq.get(), "dk": self.dk.get(),
                "dv": self.dv.get()}

    def run(self):
        self.forward()
        self.backward()
        return self.results()


def check(got, val, tol, names=None):
    """Every element of a sequence within its bound; every row in none as it was."""
    for n in names or val:
        g, x, t = got[n].astype(np.float64), val[n], tol[n]
        none = np.isnan(t)
        np.testing.assert_array_equal(g[none], -777.0, err_msg=f"{n}: a row in no sequence was written")
        bad = ~(np.abs(g - x) <= t + 1e-37) & ~none
        if bad.any():
            i = np.unravel_index(np.argmax(np.where(bad, np.abs(g - x) / (t + 1e-37), 0)), bad.shape)
            raise AssertionError(f"{n}{i}: {g[i]} against {x[i]}, bound {t[i]}; {bad.sum()} of {bad.size} beyond theirs")


# ----------------------------------------------------------------- rotation --

def rope(x, w, dy, pos, eps, base, R, interleaved):
    """y, dx, dw in 64 bits over [T, H, D], and the bound of each."""
    x, w, dy, pos = f64(x), f64(w), f64(dy), f64(pos)
    T, H, D = x.shape
    i = torch.arange(R // 2, dtype=torch.float64)
    ang = (pos[:, None] * base ** (-2 * i / R))[:, None] if R else torch.zeros(T, 1, 0, dtype=torch.float64)
    cos, sin = ang.cos(), ang.sin()
    ia, ib = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))

    def turn(z, sgn):
        z, y = z, z.clone()
        y[..., ia] = z[..., ia] * cos - sgn * z[..., ib] * sin
        y[..., ib] = sgn * z[..., ia] * sin + z[..., ib] * cos
        return y

    def reach(z):  # the magnitudes that make an element of the turned row
        y = z.abs().clone()
        y[..., ia] = y[..., ib] = z[..., ia].abs() + z[..., ib].abs()
        return y

    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    g = turn(dy, -1)
    h = g * w
    m = (h * n).mean(-1, keepdim=True)
    hm = reach(dy) * w.abs()
    mm = (hm * n.abs()).mean(-1, keepdim=True)
    dx = r * (h - n * m)
    # r: half of (D + 2) u from its sum, 3 roundings; sine, cosine 4 u with their angle.
    k = (D / 2 + 16) * U
    val = {"y": turn(n * w, 1), "dx": dx, "dw": (g * n).sum((0, 1))}
    tol = {"y": reach(n * w) * k, "dx": r * (hm + n.abs() * mm) * (2 * k + (D + 16) * U),
           "dw": (reach(dy) * n.abs()).sum((0, 1)) * (k + (T * H + 16) * U)}
    return {a: b.numpy() for a, b in val.items()}, {a: b.numpy() for a, b in tol.items()}


# ----------------------------------------------------- linear cross-entropy --

def linear_xent(x, w, t, ignore, go):
    """loss, stats, dx, dw in 64 bits, and the bound of each."""
    x, w = f64(x), f64(w)
    R, D = x.shape
    V = w.shape[0]
    keep = torch.as_tensor(~(np.asarray(t) == np.float32(ignore)))
    tt = torch.where(keep, f64(t), 0.0).long()
    n = int(keep.sum())
    z = x @ w.T
    e = ((x.abs() @ w.abs().T) * (W + (D + 4) * U)).amax(1)  # a row's largest logit error
    top = z.amax(1)
    s = torch.exp(z - top[:, None]).sum(1)
    term = torch.where(keep, top + s.log() - z[torch.arange(R), tt], 0.0)
    eterm = torch.where(keep, 2 * e + 8 * U * (top.abs() + s.log() + z.abs().amax(1) + 1) + V * U, 0.0)
    c = go / n if n else 0.0
    p = torch.exp(z - top[:, None]) / s[:, None]
    d = p.clone()
    d[torch.arange(R), tt] -= 1
    d = d * keep[:, None] * c
    ep = p * (4 * e[:, None] + (V + 16) * U) + 2 * U
    ed = (ep * keep[:, None] + d.abs() / (abs(c) or 1.0) * 4 * U) * abs(c)
    val = {"loss": term.sum().reshape(1) / max(n, 1), "stats": torch.stack([top, s], 1), "dx": d @ w, "dw": d.T @ x}
    tol = {"loss": (eterm.sum() + term.abs().sum() * (R + 4) * U).reshape(1) / max(n, 1),
           "stats": torch.stack([e, s * (2 * 2 * e + (V + 8) * U)], 1),
           "dx": ed @ w.abs() + (d.abs() @ w.abs()) * (W + (V + 4) * U),
           "dw": ed.T @ x.abs() + (d.abs().T @ x.abs()) * (W + (R + 4) * U)}
    return {a: b.numpy() for a, b in val.items()}, {a: b.numpy() for a, b in tol.items()}
