"""vh_qk_norm_rope_fwd / _bwd against the 64-bit reference and its bounds (packed_ref.py)."""
import numpy as np
import pytest

import packed_ref as R
from test_packed_attention_gpu import Graph
from test_streams_gpu import Streams

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, vh, T, Hq, Hk, D, rot, inter, base=1e4, eps=1e-6, far=0.0, kind="plain", scale=1.0, seed=0, pos=None):
        r = np.random.default_rng(40 + seed)
        g = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.vh, self.par = vh, (eps, base, rot, inter)
        self.x = [np.float32(scale) * g(T, Hq, D), np.float32(scale) * g(T, Hk, D)]
        self.w = [1 + np.float32(0.1) * g(D), 1 + np.float32(0.1) * g(D)]
        self.dy = [g(T, Hq, D), g(T, Hk, D)]
        self.pos = (np.float32(far) + np.arange(T, dtype=np.float32)) if pos is None else pos
        self.upload(kind)

    def upload(self, kind):
        vh = self.vh
        self.X, self.DY = [R.Buf(vh, a, kind) for a in self.x], [R.Buf(vh, a, kind) for a in self.dy]
        self.W, self.P = [vh.DeviceBuffer.from_array(a) for a in self.w], vh.DeviceBuffer.from_array(self.pos)
        self.Y, self.DX = ([R.like(vh, a.shape, kind) for a in self.x] for _ in range(2))
        D = self.x[0].shape[2]
        self.DW = [vh.DeviceBuffer(4 * D) for _ in range(2)]

    def head(self):
        e, b, rot, inter = self.par
        q, k = self.X
        return (q.ptr, q.l, k.ptr, k.l, self.W[0].ptr, self.W[1].ptr, self.P.ptr, e, b, rot, inter)

    def forward(self, stream=None):
        q, k = self.Y
        self.vh.check(self.vh.lib.vh_qk_norm_rope_fwd(*self.head(), q.ptr, q.l, k.ptr, k.l, stream))

    def backward(self, scratch=None, stream=None):
        a = []
        for b in (*self.DY, *self.DX):
            a += [b.ptr, b.l]
        p, nb = (scratch.ptr, scratch.nbytes) if scratch else (None, 0)
        self.vh.check(self.vh.lib.vh_qk_norm_rope_bwd(*self.head(), *a, self.DW[0].ptr, self.DW[1].ptr, p, nb, stream))

    def results(self):
        self.vh.sync()
        D = self.x[0].shape[2]
        return [{"y": y.get(), "dx": d.get(), "dw": w.to_array((D,))} for y, d, w in zip(self.Y, self.DX, self.DW)]

    def run(self):
        self.forward()
        self.backward()
        return self.results()

    def check(self, got=None):
        for g, x, w, dy in zip(got or self.run(), self.x, self.w, self.dy):
            val, tol = R.rope(x, w, dy, self.pos, np.float64(np.float32(self.par[0])), *self.par[1:])
            R.check(g, val, tol)


@pytest.mark.parametrize("inter", [0, 1])
@pytest.mark.parametrize("D,rot", [(1, 0), (2, 2), (6, 4), (7, 6), (8, 8), (16, 8), (32, 32), (40, 40), (64, 64), (64, 32),
                                   (64, 0), (65, 64), (80, 40), (80, 80), (80, 16), (96, 96), (96, 24), (112, 112), (112, 42), (112, 0), (100, 56), (127, 126), (128, 128), (128, 12),
                                   (130, 130), (192, 64), (256, 256), (255, 130), (252, 248)])
def test_head_sizes(vh, D, rot, inter):
    Call(vh, 37, 3, 2, D, rot, inter, seed=D).check()


@pytest.mark.parametrize("T", [1, 2, 63, 65, 1000, 5000])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (12, 4), (9, 1), (0, 3), (5, 0)])
def test_tokens_and_heads(vh, T, Hq, Hk):
    if T * (Hq + Hk) > 30000:
        T = 1900
    Call(vh, T, Hq, Hk, 64, 64, 0, seed=T).check()


@pytest.mark.parametrize("kind", ["cols", "odd", "heads_first"])
@pytest.mark.parametrize("D", [40, 64, 66, 80, 112])
def test_layouts(vh, kind, D):
    Call(vh, 50, 4, 2, D, D // 4 * 2, 0, kind=kind).check()


@pytest.mark.parametrize("far", [1e5, 1e6, 16777000.0, -500.0])
@pytest.mark.parametrize("base", [1e4, 5e5, 2.0])
def test_far_positions(vh, far, base):
    Call(vh, 130, 2, 1, 128, 128, 1, base=base, far=far).check()


def test_fractional_and_large_positions(vh):
    r = np.random.default_rng(2)
    Call(vh, 100, 2, 1, 64, 64, 0, pos=r.uniform(-1e4, 1e4, 100).astype(np.float32)).check()
    Call(vh, 100, 2, 1, 64, 64, 0, pos=r.integers(2 ** 24, 2 ** 30, 100).astype(np.float32)).check()


@pytest.mark.parametrize("scale,eps", [(1e-12, 1e-6), (1e12, 1e-6), (1e-3, 0.0), (0.0, 1e-5)])
def test_ranges(vh, scale, eps):
    Call(vh, 40, 2, 2, 64, 64, 0, scale=scale, eps=eps).check()


def test_bad_values_stay_in_their_row(vh):
    c = Call(vh, 40, 3, 2, 64, 64, 0)
    clean = c.run()
    c.x[0][7, 1, 5] = np.nan
    c.x[1][9, 0, 6] = np.inf
    c.upload("plain")
    c.pos[20] = np.nan
    c.P = vh.DeviceBuffer.from_array(c.pos)
    got = c.run()
    for i, (t, h) in enumerate(((7, 1), (9, 0))):
        keep = np.ones((40, c.x[i].shape[1]), bool)
        keep[t, h] = keep[20] = False
        for n in ("y", "dx"):
            np.testing.assert_array_equal(got[i][n][keep], clean[i][n][keep])
            assert np.isnan(got[i][n][20]).all()
        assert np.isnan(got[i]["dw"]).all()


@pytest.mark.parametrize("D", [64, 66])
def test_in_place(vh, D):
    """Results in the inputs' place."""
    c = Call(vh, 300, 4, 2, D, D // 4 * 2, 0)
    want = c.run()
    c.upload("plain")
    c.DX = c.DY  # dq over dqo, dk over dko
    c.backward()
    vh.sync()
    for w, d, wd in zip(want, c.DX, c.DW):
        np.testing.assert_array_equal(d.get(), w["dx"])
        np.testing.assert_array_equal(wd.to_array((D,)), w["dw"])
    c.Y = c.X
    c.forward()
    vh.sync()
    for w, y in zip(want, c.Y):
        np.testing.assert_array_equal(y.get(), w["y"])


def test_same_bits_other_stream_and_graph(vh):
    c = Call(vh, 3000, 4, 2, 64, 64, 0)
    want = c.run()
    st = Streams(1)
    d = Call(vh, 3000, 4, 2, 64, 64, 0)
    vh.sync()
    d.forward(st.s[0])
    d.backward(stream=st.s[0])
    st.close()
    scratch = vh.DeviceBuffer(vh.lib.vh_qk_norm_rope_bwd_scratch_bytes(3000, 64))
    e = Call(vh, 3000, 4, 2, 64, 64, 0)
    e.run()
    with pytest.raises(vh.VhError, match="too small"):
        e.backward(vh.DeviceBuffer(16))

    def body(s):
        e.forward(s)
        e.backward(scratch, s)
        with pytest.raises(vh.VhError, match="capture"):
            e.backward(None, s)

    g = Graph(body)
    try:
        for rep in range(3):
            for b in (*e.Y, *e.DX):
                b.dev.upload(b.host)
            vh.sync()
            g.replay()
            for got in (d.results(), e.results()):
                for a, b in zip(got, want):
                    for n in a:
                        np.testing.assert_array_equal(a[n], b[n], err_msg=n)
    finally:
        g.close()


def test_nothing_to_do(vh):
    c = Call(vh, 0, 2, 1, 8, 8, 0)
    c.forward()
    c.backward()
    vh.sync()
    for w in c.DW:
        assert (w.to_array((8,)) == 0).all()  # sums over no row
