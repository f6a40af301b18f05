"""vh_linear_cross_entropy_* against the 64-bit reference and its bounds (packed_ref.py), and
a run of the three packed-training operators as a model makes it."""
import math

import numpy as np
import pytest
import torch

import packed_ref as R
from test_packed_attention_gpu import Graph
from test_packed_rope_gpu import Call
from test_streams_gpu import Streams

pytestmark = pytest.mark.gpu
BIG = (1100, 700, 17003)  # the gradient's products by f16 parts too


class Xent:
    def __init__(self, vh, Rr, D, V, ignored=0.0, ignore=-100.0, go=1.0, pad=0, offset=0, scale=0.3, seed=0, t=None):
        r = np.random.default_rng(70 + seed)
        self.vh, self.sizes, self.ignore, self.go, self.pad, self.offset = vh, (Rr, D, V), ignore, go, pad, offset
        self.x = r.standard_normal((Rr, D)).astype(np.float32)
        self.w = (scale * r.standard_normal((V, D))).astype(np.float32)
        self.t = r.integers(0, V, Rr).astype(np.float32) if t is None else np.asarray(t, np.float32)
        if t is None and ignored:
            self.t[r.random(Rr) < ignored] = ignore
        self.put()

    def put(self):
        vh, (Rr, D, V) = self.vh, self.sizes
        self.ld = D + self.pad

        def rows(a):
            b = np.full(self.offset + a.shape[0] * self.ld, -777.0, np.float32)
            b[self.offset:].reshape(-1, self.ld)[:, :D] = a
            return vh.DeviceBuffer.from_array(b)

        self.X, self.W_, self.T = rows(self.x), rows(self.w), vh.DeviceBuffer.from_array(self.t)
        self.GO = vh.DeviceBuffer.from_array(np.array([self.go], np.float32))
        self.loss, self.stats = vh.DeviceBuffer(4), vh.DeviceBuffer(8 * Rr)
        self.dx, self.dw = rows(np.full((Rr, D), -777.0)), rows(np.full((V, D), -777.0))

    def call(self, which, scratch=None, stream=None):
        L, o = self.vh.lib, 4 * self.offset
        p, nb = (scratch.ptr, scratch.nbytes) if scratch else (None, 0)
        head = (self.X.ptr + o, self.ld, self.W_.ptr + o, self.ld, self.T.ptr, self.ignore)
        grads = (self.dx.ptr + o, self.ld, self.dw.ptr + o, self.ld)
        mid = {"fwd": (self.loss.ptr, self.stats.ptr), "bwd": (self.stats.ptr, self.GO.ptr, *grads),
               "fwd_bwd": (self.GO.ptr, self.loss.ptr, *grads)}[which]
        self.vh.check(getattr(L, "vh_linear_cross_entropy_" + which)(*head, *mid, *self.sizes, p, nb, stream))

    def rows(self, buf, n):
        D = self.sizes[1]
        b = buf.to_array((self.offset + n * self.ld,))
        m = b[self.offset:].reshape(n, self.ld)
        assert (b[:self.offset] == -777.0).all() and (m[:, D:] == -777.0).all(), "written outside the rows"
        return m[:, :D]

    def results(self):
        self.vh.sync()
        Rr, D, V = self.sizes
        return {"loss": self.loss.to_array((1,)), "stats": self.stats.to_array((Rr, 2)), "dx": self.rows(self.dx, Rr),
                "dw": self.rows(self.dw, V)}

    def check(self):
        val, tol = R.linear_xent(self.x, self.w, self.t, self.ignore, self.go)
        self.call("fwd")
        self.call("bwd")
        R.check(self.results(), val, tol)
        self.put()
        self.call("fwd_bwd")
        R.check(self.results(), val, tol, ["loss", "dx", "dw"])


@pytest.mark.parametrize("Rr,D,V", [(1, 1, 1), (1, 4, 2), (3, 5, 7), (2, 64, 1), (64, 32, 100), (100, 96, 513), (257, 128, 1000),
                                    (300, 129, 2049), (1000, 64, 4099), (33, 768, 5003), (17, 16, 70001),
                                    (700, 768, 1000), (129, 1030, 3001), (1500, 250, 1281), (4100, 40, 2050)])
@pytest.mark.parametrize("ignored", [0.0, 0.4])
def test_sizes(vh, Rr, D, V, ignored):
    Xent(vh, Rr, D, V, ignored, go=0.75, seed=Rr).check()


@pytest.mark.parametrize("pad,offset", [(3, 0), (4, 4), (0, 1), (5, 3)])
def test_strided_rows(vh, pad, offset):
    Xent(vh, 130, 60, 700, 0.2, pad=pad, offset=offset).check()


@pytest.mark.parametrize("sizes,pad", [((1025, 1030, 12001), 3), ((8200, 258, 6000), 0), ((4100, 256, 15000), 1),
                                       ((768, 300, 60001), 0)])
def test_gradient_by_parts(vh, sizes, pad):
    """Sizes past the tiles' by a little, dx or dw in sums of several workgroups or whole, several pieces."""
    Xent(vh, *sizes, 0.2, pad=pad, go=0.7).check()


def test_several_pieces(vh):
    """More rows than a piece holds: 256 rows a piece at this vocabulary."""
    V = 400003
    assert vh.lib.vh_linear_cross_entropy_scratch_bytes(700, 8, V, 1) < 4 * 700 * V
    Xent(vh, 700, 8, V, 0.3).check()


def test_last_piece_with_more_sums(vh):
    """4352 rows of 512 whole tiles and 100 in five sums, then 3948 of 512 and 64 in eight: the larger lot fits the scratch."""
    c = Xent(vh, 8300, 4608, 2560, 0.1, scale=0.02)
    val, tol = R.linear_xent(c.x, c.w, c.t, c.ignore, c.go)
    c.call("fwd_bwd")
    R.check(c.results(), val, tol, ["loss", "dx", "dw"])


@pytest.mark.parametrize("ignore", [-100.0, 3.0, math.nan])
def test_ignored(vh, ignore):
    t = np.array([3, 1, 4, 1, 5, 3, 2, 6, 3, 5], np.float32)
    if ignore == -100.0:
        t[2] = -100
    Xent(vh, 10, 12, 9, ignore=ignore, t=t).check()


@pytest.mark.parametrize("sizes", [(20, 8, 30), (400, 512, 2000), BIG])
def test_no_row_counted(vh, sizes):
    c = Xent(vh, *sizes, t=[-100.0] * sizes[0])
    c.check()
    got = c.results()
    assert got["loss"][0] == 0 and not got["dx"].any() and not got["dw"].any()


@pytest.mark.parametrize("scale", [1e-6, 30.0])
@pytest.mark.parametrize("sizes", [(120, 64, 900), (400, 512, 2000), BIG])
def test_flat_and_sharp(vh, scale, sizes):
    Xent(vh, *sizes, scale=scale).check()


@pytest.mark.parametrize("sizes", [(500, 600, 1500), BIG])
def test_rows_of_very_different_size(vh, sizes):
    c = Xent(vh, *sizes, 0.1, scale=0.05)
    r = np.random.default_rng(4)
    c.x *= (10.0 ** r.uniform(-12, 0, (sizes[0], 1))).astype(np.float32)
    c.w *= (10.0 ** r.uniform(-12, 0, (sizes[2], 1))).astype(np.float32)
    c.x[7] = c.w[9] = 0
    c.put()
    c.check()


@pytest.mark.parametrize("value,text", [(-1.0, "Target class cannot be negative: -1"),
                                        (50.0, "Target class 50 out of vocab bounds 50")])
def test_bad_targets(vh, value, text):
    for which, sizes in (("fwd", (40, 8, 50)), ("fwd_bwd", (40, 8, 50)), ("fwd", (2000, 3000, 50)), ("fwd_bwd", (2000, 3000, 50))):
        c = Xent(vh, *sizes)
        c.t[[11, 30]] = value
        c.put()
        c.call(which)
        with pytest.raises(vh.DevicePanic, match=text):
            vh.sync()
    vh.sync()


@pytest.mark.parametrize("sizes", [(40, 16, 200), (400, 512, 2000), BIG])
def test_bad_values_stay_in_their_row(vh, sizes):
    c = Xent(vh, *sizes)
    c.call("fwd")
    c.call("bwd")
    clean = c.results()
    c.x[7, 3] = np.nan
    c.put()
    c.call("fwd")
    c.call("bwd")
    got = c.results()
    keep = np.arange(sizes[0]) != 7
    assert np.isnan(got["loss"][0]) and np.isnan(got["dx"][7]).all() and np.isnan(got["dw"]).all()
    np.testing.assert_array_equal(got["dx"][keep], clean["dx"][keep])
    np.testing.assert_array_equal(got["stats"][keep], clean["stats"][keep])


@pytest.mark.parametrize("sizes", [(40, 16, 200), (400, 512, 2000), BIG])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_ignored_rows_reach_nothing(vh, sizes, bad):
    """What a row that is not counted holds reaches neither the loss nor dw, and its dx is zero."""
    c = Xent(vh, *sizes, 0.3)
    c.t[-1] = -100
    off = c.t == -100
    val, tol = R.linear_xent(c.x, c.w, c.t, c.ignore, c.go)
    c.x[off] = bad
    for calls in (("fwd", "bwd"), ("fwd_bwd",)):
        c.put()
        for which in calls:
            c.call(which)
        got = c.results()
        assert not got["dx"][off].any()
        R.check(got, val, tol, ["loss", "dx", "dw"])


@pytest.mark.parametrize("sizes", [(40, 16, 200), (400, 512, 2000), BIG])
@pytest.mark.parametrize("power", [-100, 100])
def test_large_weights_of_small_rows(vh, sizes, power):
    """Logits of a usual size whose factors are far from one."""
    c = Xent(vh, *sizes, 0.1)
    c.x = np.ldexp(c.x, power).astype(np.float32)
    c.w = np.ldexp(c.w, -power).astype(np.float32)
    c.put()
    c.call("fwd")
    R.check(c.results(), *R.linear_xent(c.x, c.w, c.t, c.ignore, c.go), ["loss", "stats"])


@pytest.mark.parametrize("go", [0.0, -3.0, 1e-20, 1e15])
def test_gradients_of_the_loss(vh, go):
    Xent(vh, *BIG, 0.1, go=go).check()


def test_entries_of_small_probability(vh):
    """Entries that no row gives weight: each row of dw to its own size, not to the largest one's."""
    c = Xent(vh, *BIG)
    V, rare = BIG[2], np.arange(5000, 5100)
    c.w[:] *= 0.1
    c.x[:, 0], c.w[:, 0] = 1, 0
    c.w[rare, 0] = -np.linspace(20, 60, 100)
    c.t = (c.t + 200 * ((c.t >= 5000) & (c.t < 5100))).astype(np.float32)
    c.put()
    val, tol = R.linear_xent(c.x, c.w, c.t, c.ignore, c.go)
    # No entry here is a target, so dz is p / R with no difference taken: p to 4 e + (V + 16) u
    # of itself, e the logit's error, and the sum over rows as everywhere.
    x, w = R.f64(c.x), R.f64(c.w[rare])
    p = torch.exp(x @ w.T - R.f64(val["stats"][:, :1])) / R.f64(val["stats"][:, 1:]) / BIG[0]
    e = ((x.abs() @ w.abs().T) * (R.W + (BIG[1] + 4) * R.U)).amax()
    small = (p.T @ x.abs()).numpy() * float(4 * e + (V + 16) * R.U + R.W + (BIG[0] + 4) * R.U)
    assert (small < 0.1 * tol["dw"][rare]).all()
    for calls in (("fwd", "bwd"), ("fwd_bwd",)):
        c.put()
        for which in calls:
            c.call(which)
        got = c.results()
        R.check(got, val, tol, ["loss", "dx", "dw"])
        assert (np.abs(got["dw"][rare] - val["dw"][rare]) <= small).all()


@pytest.mark.parametrize("sizes", [(700, 64, 3001), BIG])
def test_same_bits_and_streams(vh, sizes):
    c = Xent(vh, *sizes, 0.1)
    c.call("fwd_bwd")
    want = c.results()
    st = Streams(2)
    try:
        d = [Xent(vh, *sizes, 0.1) for _ in range(2)]
        vh.sync()
        for rep in range(2):
            for x, s in zip(d, st.s):
                x.call("fwd_bwd", stream=s)
        st.sync()
        for x in d:
            got = x.results()
            for n in ("loss", "dx", "dw"):
                np.testing.assert_array_equal(got[n], want[n], err_msg=n)
    finally:
        st.close()
    with pytest.raises(vh.VhError, match="too small"):
        c.call("fwd", vh.DeviceBuffer(64))
    scratch = vh.DeviceBuffer(vh.lib.vh_linear_cross_entropy_scratch_bytes(*sizes, 1))
    c.call("fwd_bwd", scratch)
    np.testing.assert_array_equal(c.results()["dw"], want["dw"])


def test_no_capture(vh):
    c = Xent(vh, 10, 8, 20)
    scratch = vh.DeviceBuffer(vh.lib.vh_linear_cross_entropy_scratch_bytes(10, 8, 20, 1))

    def body(s):
        for which in ("fwd", "bwd", "fwd_bwd"):
            with pytest.raises(vh.VhError, match="capture"):
                c.call(which, scratch, s)

    Graph(body).close()


def test_run_together(vh):
    """Projection's q and k through the norm and rotation, packed attention, the loss, and all the way
    back, against torch's autograd in 64 bits."""
    lens, Hq, Hk, D, V = [70, 1, 50], 4, 2, 32, 300
    T, scale = sum(lens), 32 ** -0.5
    r = np.random.default_rng(99)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.float32)
    rope = Call(vh, T, Hq, Hk, D, D, 0, pos=pos, seed=5)
    v = r.standard_normal((T, Hk, D)).astype(np.float32)
    att = R.Attention(vh, rope.x[0], rope.x[1], v, rope.x[0], R.starts_of(lens), scale, True)
    xe = Xent(vh, T, Hq * D, V, 0.2, seed=6)
    # Each operator's buffers are the one's before: rope.Y -> attention -> x of the loss, and back.
    att.q, att.k = rope.Y
    xe.X = att.o.dev
    off = (att.o.ptr - att.o.dev.ptr) // 4
    assert off == 0
    rope.forward()
    att.forward()
    xe.call("fwd_bwd")
    vh.sync()
    att.do = R.Buf(vh, xe.rows(xe.dx, T).reshape(T, Hq, D))
    att.backward()
    rope.DY = [att.dq, att.dk]
    rope.backward()
    got = rope.results()
    P = {n: R.f64(a).requires_grad_() for n, a in (("q", rope.x[0]), ("k", rope.x[1]), ("v", v), ("w", xe.w),
                                                     ("wq", rope.w[0]), ("wk", rope.w[1]))}
    z = torch.polar(torch.ones(T, D // 2, dtype=torch.float64),
                    R.f64(pos)[:, None] * 1e4 ** (-2 * torch.arange(D // 2, dtype=torch.float64) / D))[:, None]

    def turned(x, w):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        u = torch.complex(y[..., :D // 2], y[..., D // 2:]) * z
        return torch.cat([u.real, u.imag], -1)

    q, k, outs, t0 = turned(P["q"], P["wq"]), turned(P["k"], P["wk"]), [], 0
    for n in lens:
        s = slice(t0, t0 + n)
        t0 += n
        a = torch.einsum("ihd,jhd->hij", q[s], k[s].repeat_interleave(2, 1)) * scale
        a = torch.softmax(a.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf), -1)
        outs.append(torch.einsum("hij,jhd->ihd", a, P["v"][s].repeat_interleave(2, 1)))
    loss = torch.nn.functional.cross_entropy(torch.cat(outs).reshape(T, -1) @ P["w"].T, torch.as_tensor(xe.t).long(),
                                             ignore_index=-100)
    want = dict(zip(P, torch.autograd.grad(loss, list(P.values()))))
    own = {"q": got[0]["dx"], "k": got[1]["dx"], "wq": got[0]["dw"], "wk": got[1]["dw"], "v": att.dv.get(),
           "w": xe.rows(xe.dw, V)}
    assert abs(xe.loss.to_array((1,))[0] - loss.item()) <= 1e-6 * loss.item()
    for n, x in own.items():
        x, y = x.astype(np.float64), want[n].numpy()
        # Every step's roundings stay far below 2^-16 of the gradient's norm at these sizes.
        assert np.linalg.norm(x - y) <= 2.0 ** -16 * np.linalg.norm(y), n
