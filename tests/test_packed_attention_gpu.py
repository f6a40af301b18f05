"""vh_packed_attention_fwd / _bwd against the 64-bit reference and its bounds
(packed_ref.py): lengths from none and one token on, head sizes of every kind, layouts,
unseen values, ranges, bad starts, streams and graphs."""
import ctypes

import numpy as np
import pytest

import packed_ref as R
from test_streams_gpu import Streams

pytestmark = pytest.mark.gpu


def inputs(lens, Hq, Hk, D, seed=0, first=0, tail=0, scale=1.0):
    r = np.random.default_rng(1000 + seed)
    T = first + sum(lens) + tail
    g = lambda H: (scale * r.standard_normal((T, H, D))).astype(np.float32)  # noqa: E731
    return g(Hq), g(Hk), g(Hk), g(Hq)


def run_and_check(vh, lens, Hq, Hk, D, causal, first=0, tail=0, kinds=("plain",) * 4, okind="plain", arrays=None, scale=None,
                  seed=0):
    arrays = arrays or inputs(lens, Hq, Hk, D, seed, first, tail)
    scale = scale or D ** -0.5
    c = R.Attention(vh, *arrays, R.starts_of(lens, first), scale, causal, kinds, okind)
    got = c.run()
    val, tol = R.attention(*arrays, lens, np.float32(scale), causal, first)
    R.check(got, val, tol)
    return got


LENS = [[1], [2, 1, 3], [64], [63, 65, 1, 0, 128], [0, 0, 5], [31, 32, 33, 129], [257], [300, 7, 700]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_lengths(vh, lens, causal):
    run_and_check(vh, lens, 4, 2, 64, causal)


@pytest.mark.parametrize("D", [1, 2, 7, 16, 31, 32, 33, 40, 64, 65, 80, 96, 112, 127, 128, 129, 160, 192, 193, 255, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_head_sizes(vh, D, causal):
    run_and_check(vh, [150, 1, 70], 2, 1, D, causal, seed=D)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (3, 3), (6, 2), (8, 1), (12, 4), (5, 1), (16, 16)])
def test_head_groups(vh, Hq, Hk):
    run_and_check(vh, [90, 200], Hq, Hk, 32, True, seed=Hq)


@pytest.mark.parametrize("D", [48, 64])
@pytest.mark.parametrize("kinds,okind", [
    (("cols",) * 4, "cols"), (("odd",) * 4, "odd"), (("heads_first",) * 4, "heads_first"),
    (("plain", "cols", "odd", "heads_first"), "plain"), (("odd", "plain", "plain", "cols"), "heads_first"),
])
def test_layouts(vh, kinds, okind, D):
    run_and_check(vh, [100, 33, 130], 4, 2, D, True, kinds=kinds, okind=okind)


@pytest.mark.parametrize("D", [64, 160])
def test_rows_in_no_sequence_stay(vh, D):
    run_and_check(vh, [70, 3], 4, 2, D, True, first=37, tail=90)
    run_and_check(vh, [70, 3], 4, 2, D, False, first=64, tail=1)
    run_and_check(vh, [0, 0], 2, 2, D, False, first=3, tail=4)


@pytest.mark.parametrize("D", [32, 128])
def test_long_sequence(vh, D):
    run_and_check(vh, [2500], 2, 1, D, True, seed=5)


def test_many_short_sequences(vh):
    lens = [int(x) for x in np.random.default_rng(3).integers(0, 9, 700)]
    run_and_check(vh, lens, 2, 1, 32, True)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_many_workgroups(vh, D):
    """Enough blocks that dq and dk / dv go out as launches of their own."""
    run_and_check(vh, [40] * 100, 8, 4, D, True, seed=D)


@pytest.mark.parametrize("Hq,Hk,L", [(12, 4, 16), (16, 8, 32)])
def test_parts_of_the_query_heads(vh, Hq, Hk, L):
    """Enough key blocks that three query heads go to two workgroups unevenly, or two to one."""
    run_and_check(vh, [L] * (16384 // L), Hq, Hk, 32, True, seed=L)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hk,D", [([1100], 1, 1, 32), ([257, 1, 900], 2, 1, 48), ([1000, 129], 3, 1, 64), ([513], 3, 3, 80),
                                          ([640, 384], 4, 2, 112), ([700], 2, 1, 128), ([600], 2, 2, 192), ([385], 1, 1, 250)])
def test_few_rows(vh, lens, Hq, Hk, D, causal):
    """Blocks whose keys, and whose queries, are divided over workgroups, with blocks too short for it beside them."""
    run_and_check(vh, lens, Hq, Hk, D, causal, seed=D, first=5, tail=7, kinds=("plain",) * 4)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_with_bad_values(vh, bad, D):
    """A key that only later rows see, of a block divided over workgroups: rows before it as without it."""
    lens, at = [900], 610
    a = inputs(lens, 2, 1, D, 23)
    b = [x.copy() for x in a]
    b[1][at], b[2][at] = bad, bad
    got = R.Attention(vh, *b, R.starts_of(lens), 0.1, True).run()
    val, tol = R.attention(*(x[:at] for x in a), [at], 0.1, True)
    for n in ("o", "dq"):
        assert (np.abs(got[n][:at] - val[n]) <= tol[n]).all(), n
    assert (np.abs(got["lse"][:, :at] - val["lse"]) <= tol["lse"]).all()
    if np.isnan(bad):
        assert np.isnan(got["o"][at:]).all() and np.isnan(got["dq"][at:]).all()


def test_few_rows_one_chunk_of_no_weight(vh):
    """Scores of -infinity through one whole chunk: its keys have no weight, and nothing of them is seen."""
    lens, D = [600], 64
    q, k, v, do = inputs(lens, 1, 1, D, 25)
    q[..., 0] = 1.0
    k[:200, 0, 0] = -np.inf
    val, tol = R.attention(q[200:], k[200:], v[200:], do[200:], [400], 0.1, False)
    got = R.Attention(vh, q, k, v, do, R.starts_of(lens), 0.1, False).run()
    assert (np.abs(got["o"][200:] - val["o"]) <= tol["o"]).all()
    assert (np.abs(got["lse"][:, 200:] - val["lse"]) <= tol["lse"]).all()


def test_broadcast_keys(vh):
    """Every token and head reading one key row (zero strides): its gradient comes out per row."""
    lens, Hq, Hk, D = [40, 90], 4, 2, 64
    q, k, v, do = inputs(lens, Hq, Hk, D)
    k = np.broadcast_to(k[:1, :1], k.shape).copy()
    c = R.Attention(vh, q, k, v, do, R.starts_of(lens), 0.125, True)
    row = vh.DeviceBuffer.from_array(k[0, 0])
    c.k.ptr, c.k.lay = row.ptr, vh.layout(k.shape, [0, 0, 1])
    c.k.l = ctypes.byref(c.k.lay)
    val, tol = R.attention(q, k, v, do, lens, 0.125, True)
    R.check(c.run(), val, tol)


# ------------------------------------------------------------------ unseen values --

@pytest.mark.parametrize("D", [64, 128, 160])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3.4e38, 1e30])
def test_unseen_values_reach_nothing(vh, bad, D):
    """What other sequences, later tokens and tokens in no sequence hold does not reach a row."""
    lens, first, tail, at = [100, 90, 80], 10, 20, 150  # token 150 is row 40 of the second sequence
    arrays = inputs(lens, 2, 1, D, 3, first, tail)
    clean = R.Attention(vh, *arrays, R.starts_of(lens, first), 0.1, True).run()
    q, k, v, do = (x.copy() for x in arrays)
    for x in (q, k, v, do):
        x[:first] = x[first + sum(lens):] = bad
    k[at], v[at] = bad, -bad
    got = R.Attention(vh, q, k, v, do, R.starts_of(lens, first), 0.1, True).run()
    s, second = first + lens[0], slice(first + lens[0], first + lens[0] + lens[1])
    others = np.r_[0:s, s + lens[1]:first + sum(lens) + tail]
    for n in ("o", "dq", "dk", "dv"):  # whole sequences that do not hold the token: the same bits
        np.testing.assert_array_equal(got[n][others], clean[n][others], err_msg=n)
    # Earlier rows of the same sequence: what a sequence cut off before the token gives.
    cut = [lens[0], at - s]
    val, tol = R.attention(*arrays, cut, 0.1, True, first)
    for n in ("o", "dq"):
        R.check({n: np.where(np.isnan(val[n]), -777.0, got[n])}, val, tol, [n])
    if not np.isfinite(bad):
        assert np.isnan(got["o"][at]).all() and not np.isfinite(got["o"][second][at - s:]).any()


@pytest.mark.parametrize("D", [64, 128])
def test_nan_in_a_query_stays_in_its_row(vh, D):
    lens = [130]
    q, k, v, do = inputs(lens, 2, 2, D)
    clean = R.Attention(vh, q, k, v, do, R.starts_of(lens), 0.1, True).run()
    q[77, 1, 3] = np.nan
    got = R.Attention(vh, q, k, v, do, R.starts_of(lens), 0.1, True).run()
    assert np.isnan(got["o"][77, 1]).all() and np.isnan(got["lse"][1, 77]) and np.isnan(got["dq"][77, 1]).all()
    keep = np.arange(130) != 77
    np.testing.assert_array_equal(got["o"][keep], clean["o"][keep])
    np.testing.assert_array_equal(got["o"][:, 0], clean["o"][:, 0])
    assert np.isnan(got["dk"][:78, 1]).all() and np.isnan(got["dv"][:78, 1]).all()
    val, tol = R.attention(*inputs(lens, 2, 2, D), lens, np.float32(0.1), True)
    for n in ("dk", "dv"):  # keys that the row does not see
        far = np.where(np.arange(130)[:, None, None] > 77, got[n], val[n])
        assert (np.abs(far - val[n]) <= tol[n]).all(), n


def test_key_that_no_query_weighs(vh):
    """A key of -inf scores weighs nothing: the other keys' result, not NaN."""
    lens, D = [40], 32
    q, k, v, do = inputs(lens, 1, 1, D)
    q = np.abs(q)
    k[5] = -np.inf
    c = R.Attention(vh, q, k, v, do, R.starts_of(lens), 0.1, False)
    c.forward()
    vh.sync()
    got = c.o.get()
    keep = np.arange(40) != 5
    val, tol = R.attention(q[keep], k[keep], v[keep], do[keep], [39], np.float32(0.1), False)
    assert (np.abs(got[keep] - val["o"]) <= tol["o"]).all()


# ------------------------------------------------------------------------- ranges --

@pytest.mark.parametrize("name,factor", [
    ("q", 1e-6), ("k", 1e-12), ("v", 1e-20), ("do", 1e-12), ("v", 1e15), ("do", 1e10), ("k", 3.0), ("do", 0.0), ("v", 0.0),
    ("k", 0.0),
])
@pytest.mark.parametrize("D", [64, 160])
def test_scaled_inputs(vh, name, factor, D):
    lens = [100, 60]
    a = dict(zip(("q", "k", "v", "do"), inputs(lens, 2, 1, D, 9)))
    a[name] = (a[name] * np.float32(factor)).astype(np.float32)
    run_and_check(vh, lens, 2, 1, D, True, arrays=tuple(a.values()))


@pytest.mark.parametrize("name", ["q", "k", "v", "do"])
@pytest.mark.parametrize("spread", [1e3, 1e8, 1e14])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_very_different_size(vh, name, spread, causal):
    """Rows 1 / spread of their neighbours: each output within its own bound, but for keys' gradients, whose
    bound the largest query of a tile sets."""
    lens, D = [200], 64
    a = dict(zip(("q", "k", "v", "do"), inputs(lens, 2, 1, D, 11)))
    rows = np.ones(200, np.float32)
    rows[::3] = 1 / spread
    if name == "k":  # scores of a usual size at most
        rows *= 1.0
    a[name] = (a[name] * rows[:, None, None]).astype(np.float32)
    run_and_check(vh, lens, 2, 1, D, causal, arrays=tuple(a.values()))


@pytest.mark.parametrize("lens,Hq,Hk,D", [([700], 8, 1, 32), ([300], 6, 2, 64), ([40] * 100, 8, 4, 128), ([150], 4, 1, 160),
                                          ([200], 2, 1, 256),
                                          ([700], 1, 1, 64), ([1100, 40], 2, 2, 128)])
def test_rows_of_very_different_size_in_every_launch(vh, lens, Hq, Hk, D):
    """The row forms beside the matrix kernels: query heads in parts, dq with dk and dv, each alone, elements in halves."""
    for n in range(4):
        a = list(inputs(lens, Hq, Hk, D, 21))
        rows = np.ones(sum(lens), np.float32)
        rows[5:60:7] = 1e-11
        a[n] = (a[n] * rows[:, None, None]).astype(np.float32)
        run_and_check(vh, lens, Hq, Hk, D, True, arrays=tuple(a))


def test_rising_tiles(vh):
    """Values that grow or shrink a thousandfold from tile to tile (running scales)."""
    lens, D = [400], 64
    for sign in (1, -1):
        q, k, v, do = inputs(lens, 1, 1, D, 13)
        f = (10.0 ** (sign * (np.arange(400) // 64) * 3)).astype(np.float32)[:, None, None]
        run_and_check(vh, lens, 1, 1, D, True, arrays=(q, k, v * f, do))
        run_and_check(vh, lens, 1, 1, D, True, arrays=(q, k, v, do * f))
        run_and_check(vh, lens, 1, 1, D, False, arrays=(q, k, v * f, do / f))


def test_sharp_scores(vh):
    """Scores of hundreds: one key takes nearly all weight."""
    lens, D = [150, 40], 64
    q, k, v, do = inputs(lens, 2, 1, D, 15, scale=4.0)
    run_and_check(vh, lens, 2, 1, D, True, arrays=(q, k, v, do), scale=1.0)


# ----------------------------------------------------- same bits, packing, differences --

@pytest.mark.parametrize("D", [64, 128, 160])
def test_same_bits_and_no_neighbours(vh, D):
    """Twice the same bits, whatever the tokens of other sequences are. (How sums are grouped goes by the batch's sizes.)"""
    lens = [130, 77, 200]
    a = inputs(lens, 4, 2, D, 17)
    one = R.Attention(vh, *a, R.starts_of(lens), 0.1, True).run()
    two = R.Attention(vh, *a, R.starts_of(lens), 0.1, True).run()
    s = slice(130, 207)
    others = [x.copy() for x in a]
    for x in others:
        x[:130], x[207:] = x[:130][::-1] * 3, x[207:][::-1] * 0.5
    among = R.Attention(vh, *others, R.starts_of(lens), 0.1, True).run()
    val, tol = R.attention(*(x[s] for x in a), [77], 0.1, True)
    R.check(R.Attention(vh, *(x[s] for x in a), [0, 77], 0.1, True).run(), val, tol)
    for n in one:
        np.testing.assert_array_equal(one[n], two[n], err_msg=n)
        cut = (lambda y: y[:, s]) if n == "lse" else (lambda y: y[s])
        np.testing.assert_array_equal(cut(one[n]), cut(among[n]), err_msg=n)


def test_gradients_against_differences(vh):
    """Directional differences of the 64-bit forward against the kernels' gradients."""
    lens, D, scale = [60, 90], 32, 0.3
    q, k, v, do = inputs(lens, 4, 2, D, 19)
    got = R.Attention(vh, q, k, v, do, R.starts_of(lens), scale, True).run()
    r = np.random.default_rng(5)
    f = lambda *x: (R.attention(*x, do, lens, scale, True)[0]["o"] * do).sum()  # noqa: E731
    for n, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        x = [y.astype(np.float64) for y in (q, k, v)]
        d, h = r.standard_normal(x[i].shape), 1e-5
        plus, minus = list(x), list(x)
        plus[i], minus[i] = x[i] + h * d, x[i] - h * d
        num, own = (f(*plus) - f(*minus)) / (2 * h), (got[n] * d).sum()
        assert abs(num - own) <= 1e-5 * np.linalg.norm(got[n]) * np.linalg.norm(d), n


# ------------------------------------------------------- starts, streams, graphs, errors --

@pytest.mark.parametrize("starts,at,value", [([0, 40, 30, 100], 2, 30), ([0, 50, 101], 2, 101), ([-1, 50, 100], 0, -1),
                                             ([0, 2 ** 31 - 1, 100], 1, 2 ** 31 - 1), ([120, 130], 0, 120),
                                             ([0, -5, 100], 1, -5), ([0, 100] * 300, 2, 0)])
@pytest.mark.parametrize("D", [64, 160])
def test_bad_starts(vh, starts, at, value, D):
    a = inputs([100], 2, 1, D)
    c = R.Attention(vh, *a, starts, 0.1, True)
    for call in (c.forward, c.backward):
        call()
        with pytest.raises(vh.DevicePanic, match=rf"Sequence start {value} at index {at} .* 100 packed tokens"):
            vh.sync()
    vh.sync()  # reported once
    for n, x in c.results().items():
        assert (x == -777.0).all(), f"{n} written"


def test_other_streams(vh):
    lens = [300, 100]
    a = [inputs(lens, 2, 1, 64, s) for s in (1, 2, 3, 4)]
    want = [R.Attention(vh, *x, R.starts_of(lens), 0.1, True).run() for x in a]
    st = Streams(2)
    try:
        calls = [R.Attention(vh, *x, R.starts_of(lens), 0.1, True) for x in a]
        vh.sync()
        for rep in range(2):
            for i, c in enumerate(calls):
                c.forward(stream=st.s[i % 2])
                c.backward(stream=st.s[i % 2])
        st.sync()
        for c, w in zip(calls, want):
            for n, x in c.results().items():
                np.testing.assert_array_equal(x, w[n], err_msg=n)
    finally:
        st.close()


class Graph:
    """A captured and instantiated HIP graph of what `body(stream)` launches."""

    def __init__(self, body):
        self.st = Streams(1)
        h = self.h = self.st.h
        for f, n in (("hipStreamBeginCapture", 2), ("hipStreamEndCapture", 2), ("hipGraphInstantiate", 5),
                     ("hipGraphLaunch", 2), ("hipGraphExecDestroy", 1), ("hipGraphDestroy", 1)):
            getattr(h, f).argtypes = [ctypes.c_void_p] * n if f != "hipStreamBeginCapture" else [ctypes.c_void_p, ctypes.c_int]
        h.hipGraphInstantiate.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_size_t]
        self.graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        s = self.st.s[0]
        assert h.hipStreamBeginCapture(s, 2) == 0  # relaxed
        try:
            body(s)
        finally:
            assert h.hipStreamEndCapture(s, ctypes.byref(self.graph)) == 0
        assert h.hipGraphInstantiate(ctypes.byref(self.exec), self.graph, None, None, 0) == 0

    def replay(self):
        assert self.h.hipGraphLaunch(self.exec, self.st.s[0]) == 0
        self.st.sync()

    def close(self):
        self.h.hipGraphExecDestroy(self.exec)
        self.h.hipGraphDestroy(self.graph)
        self.st.close()


@pytest.mark.parametrize("D,lens,second", [(64, [200, 60], [60, 130]), (160, [200, 60], [60, 130]), (64, [900, 100], [330, 650]),
                                           (128, [900, 100], [330, 650])])
def test_captured_and_replayed(vh, D, lens, second):
    a = [inputs(lens, 2, 1, D, s) for s in (1, 2)]
    starts = [R.starts_of(lens), R.starts_of(second)]  # the second batch's sequences are others
    want = [R.Attention(vh, *x, s, 0.1, True).run() for x, s in zip(a, starts)]
    c = R.Attention(vh, *a[0], starts[0], 0.1, True)
    nb = [vh.lib.vh_packed_attention_scratch_bytes(*c.sizes, b) for b in (0, 1)]
    scratch = [vh.DeviceBuffer(n) for n in nb]
    c.forward(scratch[0])  # (kernels looked up before the capture)
    c.backward(scratch[1])
    vh.sync()
    g = Graph(lambda s: (c.forward(scratch[0], s), c.backward(scratch[1], s)))
    try:
        for i in (0, 1, 0, 1):
            for b, x in zip((c.q, c.k, c.v, c.do), a[i]):
                b.dev.upload(x)
            c.starts.upload(starts[i])
            for b in (c.o, c.dq, c.dk, c.dv):
                b.dev.upload(b.host)
            c.lse.upload(np.full(c.lse_shape, -777.0, np.float32))
            vh.sync()
            g.replay()
            for n, x in c.results().items():
                np.testing.assert_array_equal(x, want[i][n], err_msg=n)
            R.Attention(vh, *a[1 - i], starts[1 - i], 0.1, True).run()  # eager work between the replays
    finally:
        g.close()


def test_capture_needs_scratch(vh):
    c = R.Attention(vh, *inputs([30], 1, 1, 32), [0, 30], 0.1, True)

    def body(s):
        for f in (c.forward, c.backward):
            with pytest.raises(vh.VhError, match="capture"):
                f(stream=s)

    Graph(body).close()


def test_scratch_is_checked(vh):
    c = R.Attention(vh, *inputs([30], 1, 1, 32), [0, 30], 0.1, True)
    small = vh.DeviceBuffer(64)
    for f in (c.forward, c.backward):
        with pytest.raises(vh.VhError, match="too small"):
            f(small)


def test_nothing_to_do(vh):
    e = np.zeros((0, 2, 8), np.float32)
    R.Attention(vh, e, e, e, e, [0, 0], 0.1, True).run()
    x = np.ones((5, 2, 8), np.float32)
    got = R.Attention(vh, x, x, x, x, [3], 0.1, True).run()
    assert all((y == -777.0).all() for y in got.values())
