"""The sequence operators on a B200 against their 64-bit definitions (sequence_ref), with
tolerances derived there; then the ways a program uses them: views and broadcasts, several
streams, captured graphs, chunks and single tokens, and a training run of them together."""

import numpy as np
import pytest

import sequence_ref as R
import tinytensor_b200 as tt

pytestmark = pytest.mark.gpu


def _f32(a):
    return np.asarray(a, np.float32)


# ---- gated_scan --------------------------------------------------------------------------


def _scan_data(shape, axis, init, seed, gate_shape=None):
    rng = np.random.default_rng(seed)
    gate = 1 / (1 + np.exp(-(2.5 + 1.5 * rng.standard_normal(gate_shape or shape))))
    gate[rng.random(gate.shape) < 0.02] = 0.0
    gate[rng.random(gate.shape) < 0.02] *= -1.0
    lane = list(shape)
    del lane[axis]
    return (_f32(gate), _f32(rng.standard_normal(shape)), _f32(rng.standard_normal(lane)) if init else None,
            _f32(rng.standard_normal(shape)), _f32(rng.standard_normal(lane)))


def _check_scan(cache_dir, shape, axis, init=True, seed=0, gate_shape=None, flags=0):
    gate, x, s, dh, dl = _scan_data(shape, axis, init, seed, gate_shape)
    g = tt.Graph()
    na, nx, nd, nl = g.input(gate.shape), g.input(shape), g.input(shape), g.input(dl.shape)
    ns = g.input(s.shape) if init else None
    h = tt.gated_scan(na, nx, init=ns, axis=axis)
    last = tt.scan_last(h)
    feed = {na: gate, nx: x, nd: dh, nl: dl}
    if init:
        feed[ns] = s
    wrt = [na, nx] + ([ns] if init else [])
    # d/dh of sum(h*dh) is dh and d/dlast of sum(last*dl) is dl: both enter one backward scan
    loss = tt.sum(h * nd) + tt.sum(last * nl)
    out = [o.numpy() for o in tt.compile_gradients(g, loss, wrt, outputs=[h, last], cache_dir=cache_dir,
                                                   flags=flags).run(feed)]
    (rh, rlast), rg = R.scan(gate, x, s, axis), R.scan_grad(gate, x, s, axis, dh, dl)
    R.assert_within(out[0], rh)
    R.assert_within(out[1], rlast)
    if gate_shape is None:
        R.assert_within(out[2], rg[0])
    else:  # summed over the axes the gate was broadcast along: adjacent lanes 32 at a time by a tree (five
        # additions deep), the rest in double, each rounded to float32 once: at most 7 roundings a term
        v, tol = rg[0]
        ax = tuple(i for i in range(len(shape)) if gate_shape[i] != shape[i])
        sv = v.sum(ax, keepdims=True)
        R.assert_within(out[2], (sv, tol.sum(ax, keepdims=True) + 7 * R.U * np.abs(v).sum(ax, keepdims=True)))
    R.assert_within(out[3], rg[1])
    if init:
        R.assert_within(out[4], rg[2])


@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 31, 33, 127, 129, 255, 257, 513, 1023, 2049])
@pytest.mark.parametrize("D", [1, 5, 32, 70])
def test_scan_lengths(cache_dir, T, D):
    _check_scan(cache_dir, [2, T, D], 1, init=T % 2 == 1, seed=T * 100 + D)


# Several blocks of lanes a CTA: far more blocks than run at the same time, so that the ring of tiles runs on from
# one block to the next: columns of 4, 2 and 1 lanes a thread, one tile and several a block, rows of whole warps,
# short rows several a warp, and a gate a head.
@pytest.mark.parametrize("shape,axis,gate_shape", [
    ([4, 200, 30016], 1, None), ([4, 40, 60002], 1, None), ([3, 130, 30011], 1, None), ([1000, 700], 1, None),
    ([700, 4099], 1, None), ([20000, 33], 1, None), ([9000, 130], 1, None), ([6, 70, 400, 64], 1, [6, 70, 400, 1]),
    ([30, 33, 90, 24], 1, [30, 33, 90, 1])])
def test_scan_of_many_blocks_a_cta(cache_dir, shape, axis, gate_shape):
    _check_scan(cache_dir, shape, axis, seed=sum(shape), gate_shape=gate_shape)
    if gate_shape is None:
        _check_scan(cache_dir, shape, axis, init=False, seed=sum(shape) + 1)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 31, 127, 128, 129, 511, 513, 1000, 2047, 4099])
@pytest.mark.parametrize("rows", [1, 7, 40])
def test_scan_time_last(cache_dir, T, rows):
    _check_scan(cache_dir, [rows, T], 1, init=T % 2 == 0, seed=T + rows)


@pytest.mark.parametrize("shape,axis", [([6, 3, 5], 0), ([3, 4, 40, 2, 3], 2), ([2, 300, 4], 1), ([1, 20000, 3], 1),
                                        ([2, 9000, 64], 1), ([300, 200], 0), ([1, 1, 1], 1), ([3, 30000], 1),
                                        ([40, 6, 130], 1), ([1, 70000, 40], 1), ([700, 3, 128], 1), ([2, 33, 1030], 1)])
def test_scan_shapes(cache_dir, shape, axis):
    _check_scan(cache_dir, shape, axis, seed=sum(shape))


@pytest.mark.parametrize("gate_shape", [[3, 50, 4, 1], [1, 1, 4, 8], [3, 50, 1, 8], [1, 1, 1, 1], [3, 1, 4, 1], [1, 50, 1, 1]])
def test_scan_broadcast_gates(cache_dir, gate_shape):
    _check_scan(cache_dir, [3, 50, 4, 8], 1, gate_shape=gate_shape, seed=5)


@pytest.mark.parametrize("shape,gate_shape,axis", [
    ([2, 40, 3, 32], [2, 40, 3, 1], 1), ([2, 300, 2, 64], [2, 300, 2, 1], 1), ([1, 17, 5, 96], [1, 17, 5, 1], 1),
    ([2, 33, 3, 2], [2, 33, 3, 1], 1), ([2, 33, 3, 4], [2, 33, 3, 1], 1), ([3, 33, 1, 16], [3, 33, 1, 1], 1),
    ([2, 50, 128], [2, 50, 1], 1), ([2, 50, 2, 2, 16], [2, 50, 2, 1, 1], 1), ([2, 50, 3, 5], [2, 50, 3, 1], 1),
    ([50, 3, 64], [50, 3, 1], 0), ([2, 5, 3, 64], [2, 5, 3, 1], 1), ([1, 9000, 64], [1, 9000, 1], 1),
    ([2, 40, 3, 7], [2, 40, 3, 1], 1), ([2, 33, 1, 100], [2, 33, 1, 1], 1), ([2, 5, 3, 3], [2, 5, 3, 1], 1), ([1, 2, 2, 130], [1, 2, 2, 1], 1),
    ([1, 9000, 2, 37], [1, 9000, 2, 1], 1), ([1, 40, 2, 1139], [1, 40, 2, 1], 1), ([1, 20, 4128], [1, 20, 1], 1)])
def test_scan_shared_gates(cache_dir, shape, gate_shape, axis):
    _check_scan(cache_dir, shape, axis, gate_shape=gate_shape, seed=sum(shape))


def test_scan_without_fusion(cache_dir):
    _check_scan(cache_dir, [2, 300, 40], 1, flags=tt.FLAG_NO_FUSION)


def test_scan_transposed_and_constant_operands(cache_dir):
    rng = np.random.default_rng(8)
    xv, sv = _f32(rng.standard_normal([6, 50, 3])), _f32(rng.standard_normal([3, 2]))
    g = tt.Graph()
    x, s = g.input([6, 50, 3]), g.input([3, 2])
    # x read as [3, 50, 6]: neither time nor channels adjacent; a scalar gate; init broadcast
    h = tt.gated_scan(0.75, tt.transpose(x, 0, 2), init=tt.sum(s, [1], keepdims=True))
    out = [o.numpy() for o in tt.compile(g, [h, tt.scan_last(h)], cache_dir=cache_dir).run({x: xv, s: sv})]
    init = np.repeat(_f32(sv.astype(np.float64).sum(1, keepdims=True)), 6, 1)
    rh, rl = R.scan(np.float32([[[0.75]]]), xv.transpose(2, 1, 0), init, 1)
    R.assert_within(out[0], rh)
    R.assert_within(out[1], rl)


@pytest.mark.parametrize("shape,axis", [([2, 0, 3], 1), ([0, 4, 3], 1), ([2, 4, 0], 1), ([2, 0], 1)])
def test_scan_empty(cache_dir, shape, axis):
    g = tt.Graph()
    lane = shape[:axis] + shape[axis + 1:]
    a, x, s = g.input(shape), g.input(shape), g.input(lane)
    sv = _f32(np.arange(int(np.prod(lane)))).reshape(lane)
    z = np.zeros(shape, np.float32)
    h = tt.gated_scan(a, x, init=s, axis=axis)
    last = tt.scan_last(h)
    out = [o.numpy() for o in tt.compile_gradients(g, tt.sum(last), [x, s], outputs=[h, last], cache_dir=cache_dir)
           .run({a: z, x: z, s: sv})]
    assert out[0].shape == tuple(shape) and out[2].shape == tuple(shape)
    if shape[axis] == 0:
        assert np.array_equal(out[1], sv) and np.array_equal(out[3], np.ones(lane, np.float32))
    assert out[1].shape == tuple(lane)


@pytest.mark.parametrize("dh", [2, 3, 4, 5, 8, 16, 32, 64, 96])
def test_scan_without_steps_and_a_shared_gate(cache_dir, dh):
    """No steps: dinit is the last state's gradient, also where the launch is one that sums groups of lanes."""
    lane = [2, 3, dh]
    g = tt.Graph()
    a, x, s, w = g.input([2, 0, 3, 1]), g.input([2, 0, 3, dh]), g.input(lane), g.input(lane)
    last = tt.scan_last(tt.gated_scan(a, x, init=s, axis=1))
    prog = tt.compile_gradients(g, last, [a, s], outputs=[last], seed=w, cache_dir=cache_dir)
    rng = np.random.default_rng(dh)
    sv, wv = _f32(rng.standard_normal(lane)), _f32(rng.standard_normal(lane))
    ins = [tt.DeviceBuffer.from_numpy(v) for v in (np.zeros([2, 0, 3, 1]), np.zeros([2, 0, 3, dh]), sv, wv)]
    outs = [tt.DeviceBuffer.from_numpy(np.full(v, 7.0)) for v in prog.output_shapes]
    prog.run_device(ins, outs)
    got = [b.numpy() for b in outs]
    assert np.array_equal(got[0], sv) and got[1].size == 0 and np.array_equal(got[2], wv)


def test_scan_last_without_states(cache_dir):
    gate, x, s, _, _ = _scan_data([2, 900, 40], 1, True, 3)
    g = tt.Graph()
    a, b, c = g.input([2, 900, 40]), g.input([2, 900, 40]), g.input([2, 40])
    prog = tt.compile(g, [tt.scan_last(tt.gated_scan(a, b, init=c))], cache_dir=cache_dir)
    R.assert_within(prog.run({a: gate, b: x, c: s}).numpy(), R.scan(gate, x, s, 1)[1])


def test_scan_only_some_gradients(cache_dir):
    gate, x, s, dh, _ = _scan_data([2, 300, 40], 1, True, 4)
    rg = R.scan_grad(gate, x, s, 1, dh, None)
    for which in range(3):
        g = tt.Graph()
        n = [g.input(gate.shape), g.input(x.shape), g.input(s.shape)]
        d = g.input(dh.shape)
        h = tt.gated_scan(n[0], n[1], init=n[2])
        prog = tt.compile_gradients(g, h, [n[which]], outputs=[], seed=d, cache_dir=cache_dir)
        R.assert_within(prog.run({n[0]: gate, n[1]: x, n[2]: s, d: dh}).numpy(), rg[which])


def test_scan_special_values(cache_dir):
    """Zero gates start anew; a NaN addend stays, and 0 * inf is NaN as in the recurrence; an
    infinite state stays infinite or NaN (the gates behind it may underflow, and 0 * inf is
    NaN); growing gates do not disturb a state of 0 when their product overflows."""
    T, D = 700, 40
    gate, x = np.full([1, T, D], 0.5, np.float32), np.zeros([1, T, D], np.float32)
    x[0, 100, 3] = np.nan
    x[0, 100, 4] = np.inf
    gate[0, 300, :] = 0.0
    gate[0, :, 5] = 3.0  # the product of 700 gates overflows; the state stays 0
    x[0, 650, 6] = 1.0
    with np.errstate(all="ignore"):
        want = np.zeros([1, T, D])
        s = np.zeros([1, D])
        for t in range(T):
            s = gate[:, t] * s + x[:, t]
            want[:, t] = s
    g = tt.Graph()
    a, b = g.input(gate.shape), g.input(x.shape)
    got = tt.compile(g, [tt.gated_scan(a, b)], cache_dir=cache_dir).run({a: gate, b: x}).numpy()
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin) and np.isnan(got[np.isnan(want)]).all()
    assert np.array_equal(got[fin], _f32(want)[fin])  # powers of two: exact


def _wild_scan(shape, axis, kind, seed, gate_shape=None):
    """Gates whose products leave float32's range many times over, on states that do not: every lane's state
    follows a path of magnitudes within 1e-30 .. 1e30, and the upstream gradient the inverse of it."""
    rng = np.random.default_rng(seed)
    lanes = list(gate_shape or shape)
    T = lanes.pop(axis)
    u = np.linspace(0.0, 1.0, T + 1).reshape([-1] + [1] * len(lanes))
    if kind == "paths":  # a reflected random walk
        p = np.cumsum(3.0 * rng.standard_normal([T + 1] + lanes), 0) + 28
        p = np.abs(p - 112.0 * np.round(p / 112.0)) - 28
    else:
        p = {"grow": 60 * u - 30, "decay": 30 - 60 * u, "there and back": 58 * np.sin(2 * np.pi * u) / 2,
             "up and down": 29 - 58 * np.abs(2 * u - 1)}[kind] + rng.uniform(-0.5, 0.5, lanes)
    sign = np.where(rng.random([T + 1] + lanes) < 0.1, -1.0, 1.0)
    gate = _f32(10.0 ** (p[1:] - p[:-1]) * sign[1:])
    size = 10.0 ** np.broadcast_to(p, [T + 1] + [d for i, d in enumerate(shape) if i != axis])
    noise = [0.1 * rng.standard_normal(size[1:].shape) * (rng.random(size[1:].shape) < 0.5) for _ in range(2)]
    if kind != "paths":
        noise = [0.0 * n for n in noise]
    back = lambda v: np.moveaxis(v, 0, axis)  # noqa: E731
    return (back(gate), _f32(back(noise[0] * size[1:])), _f32(size[0] * rng.choice([-1, 1], size[0].shape)),
            _f32(back(noise[1] / size[1:])), _f32(1 / size[-1]))


_WILD = [([7, 60], 1, None), ([9, 130], 1, None), ([5, 600], 1, None), ([5, 4001], 1, None), ([3, 30000], 1, None),
         ([1, 70001], 1, None), ([300, 4100], 1, None), ([2, 12, 40], 1, None), ([2, 50, 7], 1, None), ([2, 300, 5], 1, None),
         ([2, 301, 6], 1, None), ([2, 900, 40], 1, None), ([1, 5000, 40], 1, None), ([1, 20000, 64], 1, None),
         ([1, 70000, 3], 1, None), ([1, 70000, 40], 1, None), ([1, 300, 3584], 1, None), ([2, 200, 12000], 1, None),
         ([300, 10, 7], 0, None), ([2, 300, 3, 64], 1, [2, 300, 3, 1]), ([1, 9000, 2, 24], 1, [1, 9000, 2, 1])]


@pytest.mark.parametrize("kind", ["paths", "grow", "decay", "there and back", "up and down"])
@pytest.mark.parametrize("shape,axis,gate_shape", _WILD)
def test_scan_where_products_of_gates_leave_the_range(cache_dir, shape, axis, gate_shape, kind):
    """A tile's map cannot hold such a product, the states are ordinary: at every cut of the axis (threads, warps,
    clusters, segments), forward and backward."""
    gate, x, s, dh, dl = _wild_scan(shape, axis, kind, sum(shape), gate_shape)
    g = tt.Graph()
    na, nx, ns, nd, nl = (g.input(v.shape) for v in (gate, x, s, dh, dl))
    h = tt.gated_scan(na, nx, init=ns, axis=axis)
    last = tt.scan_last(h)
    loss = tt.sum(h * nd) + tt.sum(last * nl)
    out = [o.numpy() for o in tt.compile_gradients(g, loss, [na, nx, ns], outputs=[h, last], cache_dir=cache_dir)
           .run({na: gate, nx: x, ns: s, nd: dh, nl: dl})]
    full = np.broadcast_to(gate, shape)
    (rh, rlast), rg = R.scan(full, x, s, axis), R.scan_grad(full, x, s, axis, dh, dl)
    assert np.isfinite(rh[0]).all() and np.abs(rh[0]).max() < 1e37 and np.abs(rg[1][0]).max() < 1e37
    R.assert_within(out[0], rh)
    R.assert_within(out[1], rlast)
    if gate_shape is None:
        R.assert_within(out[2], rg[0])
    else:  # (the bound of a shared gate's sum: see _check_scan)
        ax = tuple(i for i in range(len(shape)) if gate_shape[i] != shape[i])
        v, tol = rg[0]
        R.assert_within(out[2], (v.sum(ax, keepdims=True), tol.sum(ax, keepdims=True) + 7 * R.U * np.abs(v).sum(ax, keepdims=True)))
    R.assert_within(out[3], rg[1])
    R.assert_within(out[4], rg[2])
    # the last state alone: the states are not stored, the maps are the same
    g = tt.Graph()
    na, nx, ns = (g.input(v.shape) for v in (gate, x, s))
    alone = tt.compile(g, [tt.scan_last(tt.gated_scan(na, nx, init=ns, axis=axis))], cache_dir=cache_dir)
    R.assert_within(alone.run({na: gate, nx: x, ns: s}).numpy(), rlast)


@pytest.mark.parametrize("shape,axis", [([3, 20], 1), ([3, 100], 1), ([2, 900], 1), ([5, 9000], 1), ([1, 70001], 1), ([2, 50, 7], 1),
                                        ([2, 700, 40], 1), ([1, 5000, 40], 1), ([1, 70000, 3], 1)])
@pytest.mark.parametrize("gate", [1.0, -1.0])
def test_scan_of_states_near_the_largest_float(cache_dir, shape, axis, gate):
    """A run of addends that overflows by itself, on a state that it brings from one end of the range to the other."""
    T = shape[axis]
    lane = list(shape)
    del lane[axis]
    sign = np.where(np.arange(T) // 6 % 2 == 0, 1.0, -1.0) * np.where(np.arange(T) % 2 == 1, np.sign(gate), 1.0)
    if gate < 0:  # h[t] = -h[t-1] + x[t]: the same path with every other state's sign turned
        sign = -sign
    x = _f32(np.broadcast_to((1e38 * sign).reshape([T if i == axis else 1 for i in range(len(shape))]), shape))
    init = np.full(lane, -3e38, np.float32)
    g = tt.Graph()
    nx, ns = g.input(shape), g.input(lane)
    h = tt.gated_scan(gate, nx, init=ns, axis=axis)
    out = [o.numpy() for o in tt.compile(g, [h, tt.scan_last(h)], cache_dir=cache_dir).run({nx: x, ns: init})]
    rh, rlast = R.scan(np.full([1] * len(shape), gate), x, init, axis)
    assert np.abs(rh[0]).max() < 3.1e38
    R.assert_within(out[0], rh)
    R.assert_within(out[1], rlast)


@pytest.mark.parametrize("shape,axis", [([3, 640], 1), ([2, 700, 40], 1), ([1, 70000, 5], 1), ([1, 70001], 1)])
def test_scan_in_windows_equals_the_whole_where_gates_grow(cache_dir, shape, axis):
    """Single windows, and their states handed on: no cut of the axis changes a state."""
    gate, x, s, _, _ = _wild_scan(shape, axis, "paths", 3)
    (rh, tol), _ = R.scan(gate, x, s, axis)
    T, at = shape[axis], 0
    cut = lambda v, i, j: np.ascontiguousarray(np.moveaxis(np.moveaxis(v, axis, 0)[i:j], 0, axis))  # noqa: E731
    for n in (T // 2 + 1, T - T // 2 - 4, 1, 1, 1):
        w = [cut(v, at, at + n) for v in (gate, x)]
        g = tt.Graph()
        a, b, c = g.input(w[0].shape), g.input(w[1].shape), g.input(s.shape)
        h = tt.gated_scan(a, b, init=c, axis=axis)
        got, s = (o.numpy() for o in tt.compile(g, [h, tt.scan_last(h)], cache_dir=cache_dir).run({a: w[0], b: w[1], c: s}))
        R.assert_within(got, (cut(rh, at, at + n), cut(tol, at, at + n)))
        at += n
    assert at == T


def test_scan_in_windows_and_tokens_equals_the_whole(cache_dir):
    """Windows that hand their last state on, then single tokens: the states of one long scan."""
    gate, x, _, _, _ = _scan_data([3, 64, 20], 1, False, 6)
    (rh, tol), _ = R.scan(gate, x, None, 1)
    progs = {}
    s, at = np.zeros([3, 20], np.float32), 0
    for n in [40, 17] + [1] * 7:
        if n not in progs:
            g = tt.Graph()
            a, b, c = g.input([3, n, 20]), g.input([3, n, 20]), g.input([3, 20])
            h = tt.gated_scan(a, b, init=c)
            progs[n] = (a, b, c, tt.compile(g, [h, tt.scan_last(h)], cache_dir=cache_dir))
        a, b, c, p = progs[n]
        h, last = (o.numpy() for o in p.run({a: gate[:, at:at + n], b: x[:, at:at + n], c: s}))
        # a handed-over state is one more rounding of every term, within the bound's slack of 16
        R.assert_within(h, (rh[:, at:at + n], tol[:, at:at + n]))
        assert np.array_equal(h[:, -1], last)
        s, at = last, at + n


def test_scan_is_deterministic(cache_dir):
    gate, x, s, dh, _ = _scan_data([2, 5000, 40], 1, True, 9)
    g = tt.Graph()
    a, b, c, d = g.input(gate.shape), g.input(x.shape), g.input(s.shape), g.input(dh.shape)
    h = tt.gated_scan(a, b, init=c)
    p = tt.compile_gradients(g, h, [a, b, c], outputs=[h], seed=d, cache_dir=cache_dir)
    first = [o.numpy().tobytes() for o in p.run({a: gate, b: x, c: s, d: dh})]
    for _ in range(5):
        assert [o.numpy().tobytes() for o in p.run({a: gate, b: x, c: s, d: dh})] == first


@pytest.mark.parametrize("dense_first", [True, False])
def test_scans_that_share_an_expanded_operand(cache_dir, dense_first):
    """One scan takes the expanded node as a dense x, the other as its gate beside a transposed x."""
    rng = np.random.default_rng(16)
    av, yv, dv = _f32(rng.random([2, 5, 3, 1])), _f32(rng.standard_normal([2, 5, 4, 3])), _f32(rng.random([2, 5, 3, 4]))
    for steps in (5, 50):  # (the thread-a-lane kernel and the tiled one)
        n = steps // 5
        av2, yv2, dv2 = (np.tile(v, [1, n, 1, 1]) for v in (av, yv, dv))
        g = tt.Graph()
        a, y, d = g.input(av2.shape), g.input(yv2.shape), g.input(dv2.shape)
        if dense_first:
            h1 = tt.gated_scan(d, a, axis=1)
            h2 = tt.gated_scan(a, tt.transpose(y, 2, 3), axis=1)
        else:
            h2 = tt.gated_scan(a, tt.transpose(y, 2, 3), axis=1)
            h1 = tt.gated_scan(d, a, axis=1)
        out = [o.numpy() for o in tt.compile_gradients(g, tt.sum(h1) + tt.sum(h2), [y, d], outputs=[h1, h2], cache_dir=cache_dir)
               .run({a: av2, y: yv2, d: dv2})]
        full = np.broadcast_to(av2, dv2.shape)
        yt = yv2.transpose(0, 1, 3, 2)
        R.assert_within(out[0], R.scan(dv2, full, None, 1)[0])
        R.assert_within(out[1], R.scan(av2, yt, None, 1)[0])
        dx = R.scan_grad(av2, yt, None, 1, np.ones(yt.shape), None)[1]
        R.assert_within(out[2], tuple(v.transpose(0, 1, 3, 2) for v in dx))
        R.assert_within(out[3], R.scan_grad(dv2, full, None, 1, np.ones(yt.shape), None)[0])


@pytest.mark.parametrize("shape,axis", [([2, 5, 3], 1), ([2, 40, 5], 1), ([3, 50], 1), ([50, 3, 2], 0), ([4], 0), ([2, 1, 3], 1)])
def test_gradient_of_the_states_themselves(cache_dir, shape, axis):
    """d loss / d h takes in what the loss reads through scan_last, at the last step."""
    gate, x, s, w, wl = _scan_data(shape, axis, True, 5)
    for direct in (False, True):
        for targets in (1, 2):  # (2: the target named twice, and x beside it)
            g = tt.Graph()
            a, b, c, nw, nl = g.input(shape), g.input(shape), g.input(s.shape), g.input(shape), g.input(wl.shape)
            h = tt.gated_scan(a, b, init=c, axis=axis)
            loss = tt.sum(tt.scan_last(h) * nl)
            if direct:
                loss = loss + tt.sum(h * nw)
            wrt = [h] if targets == 1 else [h, b, h]
            out = [o.numpy() for o in tt.compile_gradients(g, loss, wrt, outputs=[tt.scan_last(h)], cache_dir=cache_dir)
                   .run({a: gate, b: x, c: s, nw: w, nl: wl})][1:]
            want = w.astype(np.float64) if direct else np.zeros(shape)
            np.moveaxis(want, axis, 0)[-1] += wl
            for o in out[::2]:
                R.assert_within(o, (want, R.U * np.abs(want)))
            if targets == 2:
                R.assert_within(out[1], R.scan_grad(gate, x, s, axis, w if direct else None, wl)[1])


# ---- token operators ---------------------------------------------------------------------------


def _tokens(rng, shape, V, empty=True):
    k = rng.integers(0, V, shape).astype(np.int32)
    k[rng.random(shape) < 0.2] = -1
    flat = k.reshape(-1)
    if flat.size > 0:
        flat[0] = V - 1
    if flat.size > 1:
        flat[1] = 0
    if flat.size > 2:
        flat[2] = -2**31  # any negative id is padding
    if empty and len(shape) > 1 and shape[0] > 2:
        k[1] = -1  # a sequence without a token
    return k


def _logits(rng, shape, V):
    x = _f32(2.5 * rng.standard_normal(list(shape) + [V]))
    if V > 3:
        x[..., V // 2] = -np.inf  # a token the sampler forbids
    return x


def _run_tokens(cache_dir, build, x, k, data, g, flags=0):
    """[values, dlogits, values] of build(logits, tokens, *data nodes): with the gradient, seeded
    with g, and in a program without one.  The two sum in different orders, so each is held
    to the definition."""
    gr = tt.Graph()
    nx, nk = gr.input(x.shape), gr.input(k.shape, dtype=tt.int32)
    nd = [gr.input(d.shape) for d in data]
    ng = gr.input(g.shape)
    y = build(nx, nk, *nd)
    feed = {nx: x, nk: k, ng: g, **dict(zip(nd, data))}
    prog = tt.compile_gradients(gr, y, [nx], outputs=[y], seed=ng, cache_dir=cache_dir, flags=flags)
    out = [o.numpy() for o in prog.run(feed)]
    g2 = tt.Graph()
    nx, nk = g2.input(x.shape), g2.input(k.shape, dtype=tt.int32)
    nd = [g2.input(d.shape) for d in data]
    alone = tt.compile(g2, [build(nx, nk, *nd)], cache_dir=cache_dir, flags=flags).run({nx: x, nk: k, **dict(zip(nd, data))})
    return out + [alone.numpy()]


def _check(out, want):
    R.assert_within(out[0], want[0])
    R.assert_within(out[1], want[1])
    R.assert_within(out[2], want[0])


VOCABULARIES = [1, 2, 3, 4, 5, 31, 33, 127, 256, 257, 1000, 1023, 1025, 4096, 8191, 8195, 32001, 50000, 131072, 200003]


@pytest.mark.parametrize("V", VOCABULARIES)
def test_token_logprob(cache_dir, V):
    rng = np.random.default_rng(V)
    shape = [3, 5] if V < 20000 else [3, 2]
    x, k, g = _logits(rng, shape, V), _tokens(rng, shape, V), _f32(rng.standard_normal(shape))
    k[k == V // 2] = 0
    x[1] = np.nan  # padding: not read
    out = _run_tokens(cache_dir, tt.token_logprob, x, k, [], g)
    x[1] = 0
    _check(out, R.logprob(x, k, g))


@pytest.mark.parametrize("V, rows", [(9200, 300), (9216, 300), (9217, 150), (35001, 80), (73728, 40), (73725, 3), (73729, 3),
                                     (2049, 600), (2560, 592), (2561, 600), (3069, 592), (3077, 600)])
def test_token_logprob_at_most_vectors_a_thread(cache_dir, V, rows):
    """Rows that just fit a cluster's threads, or just do not, and enough of them for the fewest CTAs."""
    rng = np.random.default_rng(V)
    x, k, g = _f32(rng.standard_normal([rows, V])), _tokens(rng, [rows], V), _f32(rng.standard_normal([rows]))
    out = _run_tokens(cache_dir, tt.token_logprob, x, k, [], g)
    _check(out, R.logprob(x, k, g))


# Rows that a gradient's clusters (1 to 8 CTAs of 256 or 512 threads) and small CTAs walk about ten or more each: ring
# stages and row records come round several times, barriers and mbarriers go through their phases, and padding
# rows shift the exchange's parity against the rows'.  Rows that all start on 16 bytes, and rows that do not.
@pytest.mark.parametrize("V, rows", [(2500, 6500), (3001, 6500), (5000, 3000), (9217, 1500), (9220, 1500), (18501, 1000),
                                     (35001, 720), (50004, 500), (73725, 380), (80003, 300)])
def test_token_gradient_of_many_rows_a_cluster(cache_dir, V, rows):
    rng = np.random.default_rng(V)
    x = 2 * rng.standard_normal([rows, V], dtype=np.float32)
    k, g = rng.integers(0, V, [rows]).astype(np.int32), _f32(rng.standard_normal([rows]))
    # single padding rows, a run of them, and a stretch without any
    k[rng.random(rows) < 0.15] = -1
    k[rows // 3:rows // 3 + rows // 20] = -1
    k[rows // 2:rows // 2 + rows // 5] = np.abs(k[rows // 2:rows // 2 + rows // 5])
    x[k < 0] = np.nan
    gr = tt.Graph()
    nx, nk, ng = gr.input(x.shape), gr.input([rows], dtype=tt.int32), gr.input([rows])
    y = tt.token_logprob(nx, nk)
    out = [o.numpy() for o in tt.compile_gradients(gr, y, [nx], outputs=[y], seed=ng, cache_dir=cache_dir)
           .run({nx: x, nk: k, ng: g})]
    x[k < 0] = 0
    for i in range(0, rows, 250):  # (the definition in blocks of rows, for its 64-bit copies)
        b = slice(i, i + 250)
        want = R.logprob(x[b], k[b], g[b])
        R.assert_within(out[0][b], want[0])
        R.assert_within(out[1][b], want[1])


@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_policy_gradient_of_many_rows_a_cluster(cache_dir, kl):
    """The joining warp's operands of the rows ahead, over many rows of a cluster."""
    rng = np.random.default_rng(3)
    rows, V, clip = 1400, 9300, (0.2, 0.3)
    x = rng.standard_normal([rows, V], dtype=np.float32)
    k = rng.integers(0, V, [rows]).astype(np.int32)
    k[rng.random(rows) < 0.2] = -1
    p = R.logprob(x, k)[0][0]
    ratio = np.exp(0.3 * rng.standard_normal(rows))
    for border in (0.8, 1.3):
        ratio = np.where(np.abs(ratio - border) < 1e-3, border + 5e-3, ratio)
    old, adv, g = _f32(p - np.log(ratio)), _f32(rng.standard_normal(rows)), _f32(rng.standard_normal(rows))
    ref = _f32(p + 0.3 * rng.standard_normal(rows))
    data = [old, adv] + ([ref] if kl else [])
    out = _run_tokens(cache_dir, lambda a, b, o, d, r=None: tt.policy_loss(a, b, o, d, ref_logp=r, clip=clip, kl=kl),
                      x, k, data, g)
    _check(out, R.policy(x, k, old, adv, ref if kl else None, clip, kl, g))


@pytest.mark.parametrize("rows", [1, 2, 9, 149, 600, 3000])
@pytest.mark.parametrize("V", [7, 300])
def test_token_logprob_rows(cache_dir, rows, V):
    rng = np.random.default_rng(rows)
    x, k, g = _logits(rng, [rows], V), _tokens(rng, [rows], V), _f32(rng.standard_normal([rows]))
    k[k == V // 2] = 0
    out = _run_tokens(cache_dir, tt.token_logprob, x, k, [], g)
    _check(out, R.logprob(x, k, g))


def test_token_logprob_single_row(cache_dir):
    rng = np.random.default_rng(1)
    x, k, g = _f32(rng.standard_normal([50])), np.array(7, np.int32), _f32(rng.standard_normal([]))
    _check(_run_tokens(cache_dir, tt.token_logprob, x, k, [], g), R.logprob(x, k, g))


@pytest.mark.parametrize("V", [8, 257, 5000, 40001])
@pytest.mark.parametrize("kl", [0.0, 0.25])
def test_policy_loss(cache_dir, V, kl):
    rng = np.random.default_rng(V)
    shape, clip = [4, 6], (0.2, 0.3)
    x, k = _logits(rng, shape, V), _tokens(rng, shape, V)
    k[k == V // 2] = 1
    p = R.logprob(x, k)[0][0]
    ratio = np.exp(0.3 * rng.standard_normal(shape))
    for border in (0.8, 1.3):  # off the borders by more than any rounding of p
        ratio = np.where(np.abs(ratio - border) < 1e-3, border + 5e-3, ratio)
    old, adv = _f32(p - np.log(ratio)), _f32(rng.standard_normal(shape))
    adv[0, 0] = 0.0
    ref = _f32(p + 0.3 * rng.standard_normal(shape))
    g = _f32(rng.standard_normal(shape))
    for d in (old, adv, ref):
        d[k < 0] = np.nan  # padding: not used
    data = [old, adv] + ([ref] if kl else [])
    out = _run_tokens(cache_dir, lambda a, b, o, d, r=None: tt.policy_loss(a, b, o, d, ref_logp=r, clip=clip, kl=kl),
                      x, k, data, g)
    _check(out, R.policy(x, k, old, adv, ref if kl else None, clip, kl, g))


def test_policy_loss_at_equal_policies(cache_dir):
    """r = 1 exactly: the value is -advantage and the gradient passes."""
    rng = np.random.default_rng(2)
    x = np.zeros([2, 3, 16], np.float32)
    k = rng.integers(0, 16, [2, 3]).astype(np.int32)
    old, adv, g = np.full([2, 3], -np.log(16.0), np.float32), _f32(rng.standard_normal([2, 3])), np.ones([2, 3], np.float32)
    out = _run_tokens(cache_dir, lambda a, b, o, d: tt.policy_loss(a, b, o, d, clip=(0.0625, 0.0625)), x, k, [old, adv], g)
    _check(out, R.policy(x, k, old, adv, None, (0.0625, 0.0625), 0.0, g))


@pytest.mark.parametrize("T", [0, 1, 2, 40, 300])
@pytest.mark.parametrize("V", [9, 1500])
def test_preference_loss(cache_dir, T, V):
    rng = np.random.default_rng(T * V)
    shape, beta = [3, 2, T], 0.3
    x, k = _logits(rng, shape, V), _tokens(rng, shape, V, empty=False)
    if T:
        k[k == V // 2] = 1
        k[1, 1] = -1  # an answer without a token
        k[2] = -1     # a pair without one
        x[2] = np.nan
    ref, g = _f32(R.logprob(np.nan_to_num(x, neginf=-np.inf), k)[0][0] + 0.3 * rng.standard_normal(shape)), _f32(rng.standard_normal([3]))
    for smoothing in (0.0, 0.125):
        out = _run_tokens(cache_dir, lambda a, b, r: tt.preference_loss(a, b, r, beta=beta, smoothing=smoothing),
                          x, k, [ref], g)
        _check(out, R.preference(np.nan_to_num(x, neginf=-np.inf), k, ref, beta, smoothing, g))


@pytest.mark.parametrize("N, T, V", [(200, 4, 300), (150, 5, 1025), (149, 1, 77), (40, 40, 1500), (2, 300, 701), (2, 290, 701), (33, 40, 2049)])
def test_preference_loss_of_many_short_rows(cache_dir, N, T, V):
    """Sizes around which the gradient's form changes."""
    rng = np.random.default_rng(N + T + V)
    shape, beta = [N, 2, T], 0.2
    x, k = _f32(3 * rng.standard_normal(shape + [V])), _tokens(rng, shape, V, empty=False)
    k[1, 0], k[N - 1, 1] = -1, -1
    x[1, 0] = np.nan
    x0 = np.nan_to_num(x)
    ref, g = _f32(R.logprob(x0, k)[0][0] + 0.3 * rng.standard_normal(shape)), _f32(rng.standard_normal([N]))
    out = _run_tokens(cache_dir, lambda a, b, r: tt.preference_loss(a, b, r, beta=beta, smoothing=0.125), x, k, [ref], g)
    _check(out, R.preference(x0, k, ref, beta, 0.125, g))


@pytest.mark.parametrize("N, T, V", [(32, 32, 1281), (31, 32, 1281), (33, 31, 1283), (300, 32, 1301), (32, 128, 1290), (32, 129, 1290),
                                     (32, 32, 6144), (32, 32, 6145), (400, 33, 1280)])
def test_preference_loss_of_many_pairs(cache_dir, N, T, V):
    """Sizes around which pairs go to a cluster each or to three launches."""
    rng = np.random.default_rng(N + T + V)
    shape = [N, 2, T]
    x, k = 3 * rng.standard_normal(shape + [V], dtype=np.float32), _tokens(rng, shape, V, empty=False)
    k[1, 0], k[N - 1, 1] = -1, -1
    ref, g = _f32(R.logprob(x, k)[0][0] + 0.3 * rng.standard_normal(shape)), _f32(rng.standard_normal([N]))
    out = _run_tokens(cache_dir, lambda a, b, r: tt.preference_loss(a, b, r, beta=0.2, smoothing=0.125), x, k, [ref], g)
    _check(out, R.preference(x, k, ref, 0.2, 0.125, g))


def test_preference_loss_saturates(cache_dir):
    """Sums far apart: the loss is -z or 0 and its slope -beta or 0, without overflow."""
    x = np.zeros([2, 2, 1, 4], np.float32)
    k = np.zeros([2, 2, 1], np.int32)
    ref = np.zeros([2, 2, 1], np.float32)
    ref[0, 0], ref[1, 1] = 1e4, 1e4  # z = -+1e4
    g = np.ones([2], np.float32)
    for smoothing in (0.0, 0.25):
        out = _run_tokens(cache_dir, lambda a, b, r: tt.preference_loss(a, b, r, beta=1.0, smoothing=smoothing), x, k, [ref], g)
        _check(out, R.preference(x, k, ref, 1.0, smoothing, g))


@pytest.mark.parametrize("V", [300, 3000, 40000, 140000])
def test_forbidden_and_overflowing_logits(cache_dir, V):
    """A chosen token at -inf has log-probability -inf; a row of -inf, or one with +inf or NaN,
    is NaN, as log softmax is; large logits do not overflow."""
    x = np.zeros([7, V], np.float32)
    x[0, 5] = -np.inf
    x[1] = -np.inf
    x[2, 9] = np.inf
    x[3, 10] = np.nan
    x[4] = 3e38
    x[5] = np.finfo(np.float32).min
    x[6] = np.finfo(np.float32).min
    x[6, 7] = 5.0
    k = np.array([5, 5, 5, 5, 5, 5, 7], np.int32)
    out = _run_tokens(cache_dir, tt.token_logprob, x, k, [], np.ones([7], np.float32))
    for y in (out[0], out[2]):
        assert y[0] == -np.inf and np.isnan(y[1:4]).all()
    assert np.isfinite(out[1][0]).all() and np.isnan(out[1][1]).all()
    _check([o[4:] for o in out], R.logprob(x[4:], k[4:], np.ones([3])))


def test_preference_loss_of_an_impossible_answer(cache_dir):
    x = np.zeros([2, 2, 1, 4], np.float32)
    x[0, 0, 0, 1] = -np.inf  # the chosen answer cannot be sampled: loss inf
    x[1, 1, 0, 1] = -np.inf  # the rejected one cannot: loss 0
    k = np.ones([2, 2, 1], np.int32)
    out = _run_tokens(cache_dir, lambda a, b, r: tt.preference_loss(a, b, r, beta=1.0), x, k,
                      [np.zeros([2, 2, 1], np.float32)], np.ones([2], np.float32))
    for y in (out[0], out[2]):
        assert y[0] == np.inf and y[1] == 0.0
    assert np.isfinite(out[1]).all() and (out[1][1] == 0.0).all()


@pytest.mark.parametrize("V", [5, 3000, 70000])
def test_token_outside_the_vocabulary(cache_dir, V):
    rng = np.random.default_rng(0)
    x, k = _f32(rng.standard_normal([1, 2, 2, V])), np.zeros([1, 2, 2], np.int32)
    k[0, 0, 1] = V
    for make in (lambda a, b: tt.token_logprob(a, b), lambda a, b: tt.policy_loss(a, b, 0.0, 1.0),
                 lambda a, b: tt.preference_loss(a, b, 0.0)):
        g = tt.Graph()
        nx, nk = g.input(x.shape), g.input(k.shape, dtype=tt.int32)
        y = make(nx, nk)
        prog = tt.compile_gradients(g, tt.sum(y), [nx], outputs=[y], cache_dir=cache_dir)
        with pytest.raises(tt.DeviceStatusError, match="token id"):
            prog.run({nx: x, nk: k})
        k2 = k.copy()
        k2[0, 0, 1] = 2**31 - 1
        dx, dk = tt.DeviceBuffer.from_numpy(x), tt.DeviceBuffer.from_numpy(k2, dtype=tt.int32)
        outs = [tt.DeviceBuffer(s) for s in prog.output_shapes]
        prog.run_device([dx, dk], outs)
        with pytest.raises(tt.DeviceStatusError, match="token id"):
            prog.status()
        assert np.isnan(outs[1].numpy()[0, 0, 1]).all() and np.isnan(outs[0].numpy()).any()
        # the status is cleared, and the same program answers the next batch
        out = prog.run({nx: x, nk: np.zeros_like(k)})
        assert np.isfinite(out[1].numpy()).all() and prog.status() == 0


def test_a_reports_clear_does_not_hide_the_next_one(cache_dir):
    """The status is cleared when its report is raised, whatever the default stream is busy with (streams of
    the framework are not ordered with it): the next run's report is not lost."""
    from tinytensor_b200 import _lib

    V = 64
    g = tt.Graph()
    nx, nk = g.input([4, V]), g.input([4], dtype=tt.int32)
    prog = tt.compile(g, [tt.token_logprob(nx, nk)], cache_dir=cache_dir)
    x, k = np.zeros([4, V], np.float32), np.array([0, V, 1, 2], np.int32)
    ins = [tt.DeviceBuffer.from_numpy(x), tt.DeviceBuffer.from_numpy(k, dtype=tt.int32)]
    out, st = tt.DeviceBuffer([4]), tt.Stream()
    big = [tt.DeviceBuffer([1 << 28]) for _ in range(2)]
    for _ in range(3):
        for _ in range(40):  # some 30 ms of copies on the default stream
            _lib.check(_lib.lib.tt_memcpy(big[0].ptr, big[1].ptr, big[0].nbytes, _lib.D2D, None))
        prog.run_device(ins, [out], st)
        with pytest.raises(tt.DeviceStatusError, match="token id"):
            prog.status()
        prog.run_device(ins, [out], st)
        st.synchronize()
        _lib.check(_lib.lib.tt_stream_sync(None))
        with pytest.raises(tt.DeviceStatusError, match="token id"):
            prog.status()
        assert prog.status() == 0


def test_token_operands_as_views(cache_dir):
    """Transposed rows, a broadcast advantage, logits whose vocabulary is not adjacent."""
    rng = np.random.default_rng(4)
    V, T, B = 40, 6, 3
    xv, kv = _f32(rng.standard_normal([T, B, V])), rng.integers(0, V, [T, B]).astype(np.int32)
    advv, oldv = _f32(rng.standard_normal([B, 1])), _f32(R.logprob(xv, kv)[0][0])
    g = tt.Graph()
    x, k, adv, old = g.input([T, B, V]), g.input([T, B], dtype=tt.int32), g.input([B, 1]), g.input([T, B])
    y = tt.policy_loss(tt.transpose(x, 0, 1), tt.transpose(k, 0, 1), tt.transpose(old, 0, 1), adv, clip=(0.5, 0.5))
    out = [o.numpy() for o in tt.compile_gradients(g, tt.sum(y), [x], outputs=[y], cache_dir=cache_dir)
           .run({x: xv, k: kv, adv: advv, old: oldv})]
    want = R.policy(xv.transpose(1, 0, 2), kv.T, oldv.T, advv, None, (0.5, 0.5), 0.0, np.ones([B, T]))
    R.assert_within(out[0], want[0])
    R.assert_within(out[1], tuple(np.transpose(v, (1, 0, 2)) for v in want[1]))
    g = tt.Graph()
    x, k = g.input([V, T]), g.input([T], dtype=tt.int32)
    y = tt.token_logprob(tt.transpose(x, 0, 1), k)
    xv2, kv2 = _f32(rng.standard_normal([V, T])), rng.integers(0, V, [T]).astype(np.int32)
    out = [o.numpy() for o in tt.compile_gradients(g, tt.sum(y), [x], outputs=[y], cache_dir=cache_dir).run({x: xv2, k: kv2})]
    want = R.logprob(xv2.T, kv2, np.ones([T]))
    R.assert_within(out[0], want[0])
    R.assert_within(out[1], tuple(np.transpose(v, (1, 0)) for v in want[1]))


@pytest.mark.parametrize("V", [41, 1501, 3001, 9001, 40003, 140001])
def test_rows_that_lie_differently_than_their_gradient(cache_dir, V):
    """Rows in another order than the gradient's, an odd vocabulary: the two start differently within
    16 bytes.  Tokens whose order no two strides describe are copied."""
    rng = np.random.default_rng(V)
    xv, kv = _f32(2 * rng.standard_normal([3, 2, 2, V])), rng.integers(0, V, [3, 2, 2]).astype(np.int32)
    kv[1, 0, 1] = -1
    gv = _f32(rng.standard_normal([2, 3, 2]))
    g = tt.Graph()
    x, k, s = g.input(xv.shape), g.input(kv.shape, dtype=tt.int32), g.input(gv.shape)
    y = tt.token_logprob(tt.transpose(x, 0, 1), tt.transpose(k, 0, 1))  # rows [2, 3, 2]
    out = [o.numpy() for o in tt.compile_gradients(g, y, [x], outputs=[y], seed=s, cache_dir=cache_dir).run({x: xv, k: kv, s: gv})]
    want = R.logprob(xv.transpose(1, 0, 2, 3), kv.transpose(1, 0, 2), gv)
    R.assert_within(out[0], want[0])
    R.assert_within(out[1], tuple(np.transpose(v, (1, 0, 2, 3)) for v in want[1]))
    # rows [3, 2] transposed: two strides, read in place
    g = tt.Graph()
    x, k, s = g.input([3, 2, V]), g.input([3, 2], dtype=tt.int32), g.input([2, 3])
    y = tt.token_logprob(tt.transpose(x, 0, 1), tt.transpose(k, 0, 1))
    xv, kv, gv = xv[:, :, 0], kv[:, :, 0], gv[:, :, 0]
    out = [o.numpy() for o in tt.compile_gradients(g, y, [x], outputs=[y], seed=s, cache_dir=cache_dir).run({x: xv, k: kv, s: gv})]
    want = R.logprob(xv.transpose(1, 0, 2), kv.T, gv)
    R.assert_within(out[0], want[0])
    R.assert_within(out[1], tuple(np.transpose(v, (1, 0, 2)) for v in want[1]))


def test_scan_of_one_sequence(cache_dir):
    rng = np.random.default_rng(0)
    for T in (5, 1000, 70001):
        av, xv = _f32(rng.random([T])), _f32(rng.standard_normal([T]))
        g = tt.Graph()
        a, x, s = g.input([T]), g.input([T]), g.input([])
        h = tt.gated_scan(a, x, init=s, axis=0)
        out = [o.numpy() for o in tt.compile_gradients(g, tt.sum(h), [a, x, s], outputs=[h], cache_dir=cache_dir)
               .run({a: av, x: xv, s: 2.0})]
        R.assert_within(out[0], R.scan(av, xv, np.float32(2.0), 0)[0])
        for o, r in zip(out[1:], R.scan_grad(av, xv, np.float32(2.0), 0, np.ones([T]), None)):
            R.assert_within(o, r)


def test_scan_last_twice_without_cse(cache_dir):
    gate, x, s, _, _ = _scan_data([2, 100, 40], 1, True, 3)
    g = tt.Graph()
    a, b, c = g.input(gate.shape), g.input(x.shape), g.input(s.shape)
    h = tt.gated_scan(a, b, init=c)
    l1, l2 = tt.scan_last(h), tt.scan_last(h)
    out = [o.numpy() for o in tt.compile(g, [l1 * 1.0, l2, l1], optimize=False, cache_dir=cache_dir).run({a: gate, b: x, c: s})]
    want = R.scan(gate, x, s, 1)[1]
    for o in out:
        R.assert_within(o, want)


def test_gradient_of_an_expanded_gate_itself(cache_dir):
    gate, x, _, dh, _ = _scan_data([2, 50, 3, 64], 1, False, 3, [2, 50, 3, 1])
    g = tt.Graph()
    a, b, d = g.input(gate.shape), g.input(x.shape), g.input(dh.shape)
    h = tt.gated_scan(a, b, axis=1)
    out = [o.numpy() for o in tt.compile_gradients(g, h, [h.inputs[0], a], outputs=[], seed=d, cache_dir=cache_dir)
           .run({a: gate, b: x, d: dh})]
    v, tol = R.scan_grad(gate, x, None, 1, dh, None)[0]
    R.assert_within(out[0], (v, tol))
    R.assert_within(out[1], (v.sum(-1, keepdims=True), tol.sum(-1, keepdims=True) + 2 * R.U * np.abs(v).sum(-1, keepdims=True)))


def test_gradient_that_needs_the_loss(cache_dir):
    """A loss that is not linear in the values: the gradient has its own launch."""
    rng = np.random.default_rng(5)
    xv, kv = _f32(rng.standard_normal([4, 30])), rng.integers(0, 30, [4]).astype(np.int32)
    g = tt.Graph()
    x, k = g.input([4, 30]), g.input([4], dtype=tt.int32)
    y = tt.token_logprob(x, k)
    out = [o.numpy() for o in tt.compile_gradients(g, tt.sum(y * y), [x], outputs=[y], cache_dir=cache_dir).run({x: xv, k: kv})]
    p = R.logprob(xv, kv)[0]
    # the seed 2*y is y + y of the stored y: its own error is y's bound twice
    v, tol = R.logprob(xv, kv, 2 * p[0])[1]
    R.assert_within(out[1], (v, tol + 2.02 * (p[1] + R.U * np.abs(p[0]))[:, None] * np.abs(v / (2 * p[0][:, None]))))


def test_tt_gradients_skips_token_ids(cache_dir):
    rng = np.random.default_rng(5)
    xv, kv = _f32(rng.standard_normal([4, 30])), rng.integers(0, 30, [4]).astype(np.int32)
    g = tt.Graph()
    x, k = g.input([4, 30]), g.input([4], dtype=tt.int32)
    got = tt.gradients(g, tt.sum(tt.token_logprob(x, k)), {x: xv, k: kv}, cache_dir=cache_dir)
    assert list(got) == [x]
    R.assert_within(got[x].numpy(), R.logprob(xv, kv, np.ones([4]))[1])


def test_host_tokens_are_checked(cache_dir):
    g = tt.Graph()
    x, k = g.input([4, 30]), g.input([4], dtype=tt.int32)
    p = tt.compile(g, [tt.token_logprob(x, k)], cache_dir=cache_dir)
    xv = np.zeros([4, 30], np.float32)
    assert np.isfinite(p.run({x: xv, k: np.zeros([4], np.int64)}).numpy()).all()
    for bad in (np.zeros([4], np.float32), np.full([4], 2**40), [0.5] * 4):
        with pytest.raises(tt.TypeError):
            p.run({x: xv, k: bad})
    with pytest.raises(tt.ShapeError):
        p.run({x: xv, k: np.zeros([5], np.int32)})
    buf = [tt.DeviceBuffer.from_numpy(xv), tt.DeviceBuffer.from_numpy(np.zeros([4], np.float32))]
    with pytest.raises(tt.TypeError):
        p.run_device(buf, [tt.DeviceBuffer([4])])


# ---- streams, graphs, several programs ------------------------------------------------------------


def _token_program(cache_dir, V=3000, N=4, T=32):
    rng = np.random.default_rng(7)
    x, k, ref = _logits(rng, [N, 2, T], V), _tokens(rng, [N, 2, T], V, empty=False), None
    k[k == V // 2] = 0
    ref, w = _f32(R.logprob(x, k)[0][0] + 0.1), _f32(rng.standard_normal([N]))
    g = tt.Graph()
    n = [g.input(x.shape), g.input(k.shape, dtype=tt.int32), g.input(ref.shape), g.input(w.shape)]
    y = tt.preference_loss(n[0], n[1], n[2])
    prog = tt.compile_gradients(g, y, [n[0]], outputs=[y], seed=n[3], cache_dir=cache_dir)
    bufs = [tt.DeviceBuffer.from_numpy(x), tt.DeviceBuffer.from_numpy(k, dtype=tt.int32), tt.DeviceBuffer.from_numpy(ref),
            tt.DeviceBuffer.from_numpy(w)]
    assert np.array_equal(bufs[1].numpy(), k) and bufs[1].numpy().dtype == np.int32
    return prog, bufs, R.preference(x, k, ref, 0.1, 0.0, w)


def _scan_program(cache_dir, shape=(3, 3000, 48), axis=1, seed=11):
    gate, x, s, dh, _ = _scan_data(list(shape), axis, True, seed)
    g = tt.Graph()
    n = [g.input(v.shape) for v in (gate, x, s, dh)]
    h = tt.gated_scan(n[0], n[1], init=n[2], axis=axis)
    prog = tt.compile_gradients(g, h, n[:3], outputs=[h], seed=n[3], cache_dir=cache_dir)
    want = [R.scan(gate, x, s, axis)[0]] + R.scan_grad(gate, x, s, axis, dh, None)
    return prog, [tt.DeviceBuffer.from_numpy(v) for v in (gate, x, s, dh)], want


def test_equal_outputs_and_gradients_keep_their_places(cache_dir):
    rng = np.random.default_rng(17)
    av, bv, cv = (_f32(rng.standard_normal([2, 3])) for _ in range(3))
    g = tt.Graph()
    a, b = g.input([2, 3]), g.input([2, 3])
    out = tt.compile(g, [tt.relu(a + b), a + b, a * b, a + b], cache_dir=cache_dir).run({a: av, b: bv})
    for o, w in zip(out, (np.maximum(av + bv, 0), av + bv, av * bv, av + bv), strict=True):
        assert np.array_equal(o.numpy(), w)
    g = tt.Graph()
    a, b, c = g.input([2, 3]), g.input([2, 3]), g.input([2, 3])
    grads = tt.gradients(g, tt.sum(c * c), {a: av, b: bv, c: cv}, cache_dir=cache_dir)
    assert not grads[a].numpy().any() and not grads[b].numpy().any() and np.array_equal(grads[c].numpy(), 2 * cv)
    # equal gradients of different targets: the two initial states of a scan over equal gates
    g = tt.Graph()
    gate, x, s1, s2 = g.input([2, 3]), g.input([2, 3]), g.input([3]), g.input([3])
    h1, h2 = (tt.gated_scan(gate, x, init=s, axis=0) for s in (s1, s2))
    res = tt.compile_gradients(g, tt.sum(tt.scan_last(h1)) + tt.sum(tt.scan_last(h2)), [s1, x, s2], outputs=[], cache_dir=cache_dir)
    got = [o.numpy() for o in res.run({gate: av, x: bv, s1: cv[0], s2: cv[1]})]
    want = av[0].astype(np.float64) * av[1]
    assert [o.shape for o in got] == [(3,), (2, 3), (3,)]
    for o in (got[0], got[2]):
        R.assert_within(o, (want, 2 * R.U * np.abs(want)))


def test_random_graphs_of_scans(cache_dir):
    """Scans, last states and losses over one pool of views, in random roles, against torch's autodiff in 64 bits:
    operands and launches shared in every way the schedule knows.  Gates are at most 1, so a step of
    at most 40 adds a few roundings: 100 in all, 6e-6 of a result's norm."""
    import torch

    def scan(a, x, s, axis):
        a, x = torch.broadcast_tensors(a, x)
        a, x = a.movedim(axis, 0), x.movedim(axis, 0)
        c = torch.zeros_like(x[0]) if s is None else torch.broadcast_to(s, x[0].shape)
        h = []
        for t in range(x.shape[0]):
            c = a[t] * c + x[t]
            h.append(c)
        return torch.stack(h).movedim(0, axis), c

    rng = np.random.default_rng(11)
    for case in range(40):
        T, H, D = int(rng.choice([3, 18, 40])), int(rng.integers(1, 4)), int(rng.choice([1, 3, 4, 8]))
        full = [2, T, H, D]
        shapes = [[2, T, H, 1], [2, T, D, H], full, [1, T, 1, D], [2, H, T, D], [T, H, 1]]
        vals = [_f32(rng.uniform(-1, 1, s)) for s in shapes]
        g = tt.Graph()
        leaves = [g.input(s) for s in shapes]
        ref = [torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in vals]
        pool = [leaves[0], tt.transpose(leaves[1], 2, 3), leaves[2], leaves[3], tt.transpose(leaves[4], 1, 2), leaves[5]]
        rpool = [ref[0], ref[1].transpose(2, 3), ref[2], ref[3], ref[4].transpose(1, 2), ref[5]]
        loss, rloss, outs, routs = 0.0, 0.0, [], []
        for _ in range(3):
            i, j = (int(v) for v in rng.integers(0, len(pool), 2))
            if pool[i].shape != full and pool[j].shape != full:
                j = int(rng.choice([1, 2, 4]))
            init = None
            if rng.random() < 0.5:
                init = int(rng.integers(0, len(outs) + 1)) if outs else None
            s, rs = (None, None) if init is None or init >= len(outs) else (outs[init], routs[init])
            h = tt.gated_scan(pool[i], pool[j], init=s, axis=1)
            rh, rlast = scan(rpool[i], rpool[j], rs, 1)
            if rng.random() < 0.6:
                loss, rloss = tt.sum(h * pool[2]) + loss, (rh * rpool[2]).sum() + rloss
            last = tt.scan_last(h)
            loss, rloss = tt.sum(last * last) + loss, (rlast * rlast).sum() + rloss
            outs.append(last)
            routs.append(rlast)
            if rng.random() < 0.4 and T > 1:  # (the states as another scan's operand)
                pool.append(h)
                rpool.append(rh)
        for flags in (0, tt.FLAG_NO_FUSION):
            got = [o.numpy() for o in tt.compile_gradients(g, loss, leaves, outputs=[loss], cache_dir=cache_dir, flags=flags)
                   .run(dict(zip(leaves, vals)))]
            want = [rloss] + list(torch.autograd.grad(rloss, ref, allow_unused=True, retain_graph=True))
            for o, r in zip(got, want):
                r = np.zeros(o.shape) if r is None else r.detach().numpy()
                assert o.shape == r.shape
                assert np.linalg.norm(o - r) <= 6e-6 * max(np.linalg.norm(r), 1e-30), (case, flags)


def test_on_streams_captured_and_replayed(cache_dir):
    runs = [_token_program(cache_dir), _scan_program(cache_dir), _scan_program(cache_dir, (5, 4000), 1, 12)]
    streams = [tt.Stream() for _ in runs]
    outs = [[tt.DeviceBuffer(s) for s in p.output_shapes] for p, _, _ in runs]
    for _ in range(3):  # side by side, each program on its own stream
        for (p, ins, _), o, st in zip(runs, outs, streams):
            p.run_device(ins, o, st)
    for (p, _, want), o, st in zip(runs, outs, streams):
        st.synchronize()
        assert p.status() == 0
        for b, r in zip(o, want):
            R.assert_within(b.numpy(st), r)
    # all three in one graph, replayed over outputs that were overwritten in between
    graph, st = tt.CudaGraph(), streams[0]
    with graph.capture(st):
        for (p, ins, _), o in zip(runs, outs):
            p.run_device(ins, o, st)
    for _ in range(3):
        for o in outs:
            for b in o:
                b.copy_from(np.full(b.shape, np.nan, np.float32), st)
        graph.replay(st)
        st.synchronize()
        for (p, _, want), o in zip(runs, outs):
            for b, r in zip(o, want):
                R.assert_within(b.numpy(st), r)
    # the inputs of a replay are read then: a changed seed changes the gradient
    runs[0][1][3].copy_from(np.zeros([4], np.float32), st)
    graph.replay(st)
    st.synchronize()
    assert not outs[0][1].numpy(st).any()


def test_nothing_behind_the_results_is_written(cache_dir):
    """Results in the middle of a larger allocation leave what lies behind them as it was."""
    for prog, ins, want in (_token_program(cache_dir, V=1001, N=2, T=3), _scan_program(cache_dir, (2, 333, 33)),
                            _scan_program(cache_dir, (3, 777), 1)):
        big = []
        for s in prog.output_shapes:
            b = tt.DeviceBuffer([int(np.prod(s)) + 512])
            b.copy_from(np.full(b.shape, 7.0, np.float32))
            big.append(b)
        prog.run_device(ins, big)
        prog.status()
        for b, s, r in zip(big, prog.output_shapes, want):
            v, n = b.numpy(), int(np.prod(s))
            R.assert_within(v[:n].reshape(s), r)
            assert (v[n:] == 7.0).all()


# ---- together -----------------------------------------------------------------------------------


def _model(g, B2, T, F, D, V, batch):
    """A gated recurrent token model: features -> gates and inputs -> states -> logits."""
    x = g.input([*batch, T, F], name="features")
    wg, wx, wo = g.input([F, D]), g.input([F, D]), g.input([D, V])
    h = tt.gated_scan(tt.sigmoid(x @ wg + 2.0), x @ wx, axis=-2)
    return x, [wg, wx, wo], h, h @ wo


def _model_reference(x, w, loss_grad):
    """Loss and weight gradients in 64 bits; loss_grad(logits) -> (loss, dlogits)."""
    wg, wx, wo = (v.astype(np.float64) for v in w)
    x = x.astype(np.float64)
    gate, v = 1 / (1 + np.exp(-(x @ wg + 2.0))), x @ wx
    ax = x.ndim - 2
    h = R.scan(gate, v, None, ax)[0][0]
    loss, dl = loss_grad(h @ wo)
    dh = dl @ wo.T
    (da, _), (dv, _), _ = R.scan_grad(gate, v, None, ax, dh, None)
    dz = da * gate * (1 - gate)
    flat = lambda q: q.reshape(-1, q.shape[-1])  # noqa: E731
    return loss, [flat(x).T @ flat(dz), flat(x).T @ flat(dv), flat(h).T @ flat(dl)]


def _gemm_close(got, ref):
    e = np.linalg.norm(got - ref) / np.linalg.norm(ref)
    assert e <= 1e-5, e  # the framework's matmul contract


@pytest.mark.parametrize("kind", ["cross_entropy", "policy", "preference"])
def test_model_gradients(cache_dir, kind):
    """Matmuls, gates, the scan, the head and each loss in one compiled training program."""
    rng = np.random.default_rng(13)
    T, F, D, V = 24, 40, 48, 300
    batch = [3, 2] if kind == "preference" else [4]
    g = tt.Graph()
    x, w, h, logits = _model(g, 0, T, F, D, V, batch)
    k = g.input([*batch, T], dtype=tt.int32)
    kv = _tokens(rng, [*batch, T], V, empty=False)
    xv, wv = _f32(rng.standard_normal([*batch, T, F])), [_f32(rng.standard_normal(n.shape) / 6) for n in w]
    feed = {x: xv, k: kv, **dict(zip(w, wv))}
    if kind == "cross_entropy":
        wt = _f32(rng.random([*batch, T]))
        nw = g.input(wt.shape)
        loss = -tt.sum(tt.token_logprob(logits, k) * nw)
        feed[nw] = wt
        ref = lambda lg: (lambda y, d: (-(y * wt).sum(), d))(R.logprob(lg, kv)[0][0], R.logprob(lg, kv, -wt)[1][0])  # noqa: E731
    elif kind == "policy":
        old, adv, rl = (_f32(rng.standard_normal(s)) for s in ([*batch, T], [*batch, 1], [*batch, T]))
        old, rl = old - np.float32(6), rl - np.float32(6)
        no, na, nr = (g.input(v.shape) for v in (old, adv, rl))
        loss = tt.mean(tt.policy_loss(logits, k, no, na, ref_logp=nr, kl=0.1))
        feed.update({no: old, na: adv, nr: rl})
        n = kv.size
        args = (kv, old, adv, rl, (0.2, 0.2), 0.1)
        ref = lambda lg: (R.policy(lg, *args)[0][0].mean(), R.policy(lg, *args, np.full(kv.shape, 1 / n))[1][0])  # noqa: E731
    else:
        rl = _f32(rng.standard_normal([*batch, T]) - 6)
        nr = g.input(rl.shape)
        loss = tt.mean(tt.preference_loss(logits, k, nr, beta=0.5, smoothing=0.1))
        feed[nr] = rl
        args = (kv, rl, 0.5, 0.1)
        ref = lambda lg: (R.preference(lg, *args)[0][0].mean(), R.preference(lg, *args, np.full(3, 1 / 3))[1][0])  # noqa: E731
    out = [o.numpy() for o in tt.compile_gradients(g, loss, w, cache_dir=cache_dir).run(feed)]
    rloss, rgrads = _model_reference(xv, wv, ref)
    assert abs(out[0] - rloss) <= 2e-5 * max(1.0, abs(rloss))
    for o, r in zip(out[1:], rgrads):
        _gemm_close(o, r)


def test_training_steps_with_sgd_and_host_batches(cache_dir):
    """Data-parallel SGD steps (one process) over a cross-entropy program with int32 batches from
    pinned memory move the weights as the reference gradients say, step after step."""
    rng = np.random.default_rng(14)
    B, T, F, D, V, lr = 3, 16, 24, 32, 70, 0.05
    g = tt.Graph()
    x = g.input([B, T, F])
    k = g.input([B, T], dtype=tt.int32)
    w = [g.input([F, D]), g.input([F, D]), g.input([D, V])]
    h = tt.gated_scan(tt.sigmoid(x @ w[0] + 2.0), x @ w[1])
    loss = -tt.mean(tt.token_logprob(h @ w[2], k))
    prog = tt.compile_gradients(g, loss, w, cache_dir=cache_dir)
    wv = [_f32(rng.standard_normal(n.shape) / 5) for n in w]
    params = [tt.DeviceBuffer.from_numpy(v) for v in wv]
    trainer = tt.DataParallelSGD(prog, params, lr=lr)
    stream = tt.Stream()
    hosts = [(tt.PinnedBuffer([B, T, F]), tt.PinnedBuffer([B, T], dtype=tt.int32)) for _ in range(3)]
    ref = [v.astype(np.float64) for v in wv]
    for px, pk in hosts:
        px.array[...] = _f32(rng.standard_normal([B, T, F]))
        pk.array[...] = _tokens(rng, [B, T], V)
    for px, pk in hosts:
        trainer.step_host([px, pk], stream)
        seed = np.full([B, T], -1.0 / (B * T))
        _, grads = _model_reference(px.array, ref, lambda lg: (0.0, R.logprob(lg, pk.array, seed)[1][0]))
        ref = [v - lr * d for v, d in zip(ref, grads)]
    stream.synchronize()
    assert prog.status() == 0
    for p, v0, r in zip(params, wv, ref):
        _gemm_close(p.numpy() - v0, r - v0)
