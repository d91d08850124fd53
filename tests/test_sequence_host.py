"""The sequence operators without a GPU: shapes and refusals, IR text, the schedule (which
nodes share a launch, which operands are copied), and the 64-bit definitions the GPU tests
compare with, checked against differences."""

import ctypes

import numpy as np
import pytest

import sequence_ref as R
import tinytensor_b200 as tt
from tinytensor_b200 import _lib

HOST = tt.FLAG_HOST_ONLY


def _plan(prog):
    return prog.execution_plan()


def _launches(prog):
    text = _plan(prog)
    n = int(text.split("Kernel Launches (")[1].split(")")[0])
    return n, [line.strip() for line in text.splitlines() if line.startswith("  [")]


def _loss_graph(V=7, N=2, T=3):
    g = tt.Graph()
    x = g.input([N, T, V], name="logits")
    k = g.input([N, T], dtype=tt.int32, name="tokens")
    return g, x, k


# ---- shapes and refusals -----------------------------------------------------------------


def test_scan_shapes():
    g = tt.Graph()
    a, x, s = g.input([5, 1]), g.input([2, 5, 3]), g.input([3])
    h = tt.gated_scan(a, x, init=s)
    assert h.shape == [2, 5, 3] and tt.scan_last(h).shape == [2, 3]
    assert tt.gated_scan(0.5, x, axis=-1).shape == [2, 5, 3]
    assert tt.scan_last(tt.gated_scan(x, x, axis=0)).shape == [5, 3]
    assert "gated_scan" in g.to_ir() and "axis=1" in g.to_ir()


def test_scan_refusals():
    g = tt.Graph()
    x = g.input([2, 5, 3])
    with pytest.raises(tt.DimensionError):
        tt.gated_scan(x, x, axis=3)
    with pytest.raises(tt.DimensionError):
        tt.gated_scan(g.input([4]), g.input([4]))  # rank 1 has no axis -2
    with pytest.raises(tt.BroadcastError):
        tt.gated_scan(g.input([4, 3]), x)
    with pytest.raises(tt.BroadcastError):
        tt.gated_scan(x, x, init=g.input([2, 5, 3]))
    with pytest.raises(tt.TypeError):
        tt.gated_scan(x, g.input([2, 5, 3], dtype=tt.int32))
    with pytest.raises(tt.TypeError):
        tt.gated_scan(g.input([2, 5, 3], dtype=tt.float64), x)
    with pytest.raises(tt.IRError):
        tt.scan_last(x)
    with pytest.raises(tt.IRError):
        tt.gated_scan(x, tt.Graph().input([2, 5, 3]))


def test_token_refusals():
    g, x, k = _loss_graph()
    f = g.input([2, 3])
    with pytest.raises(tt.TypeError):
        tt.token_logprob(x, f)
    with pytest.raises(tt.TypeError):
        tt.token_logprob(x, np.zeros((2, 3), np.int32))  # token ids are graph inputs
    with pytest.raises(tt.ShapeError):
        tt.token_logprob(x, g.input([3, 2], dtype=tt.int32))
    with pytest.raises(tt.ShapeError):
        tt.token_logprob(g.input([2, 0]), g.input([2], dtype=tt.int32))
    with pytest.raises(tt.ShapeError):
        tt.token_logprob(g.input([0, 2**30 + 1]), g.input([0], dtype=tt.int32))
    with pytest.raises(tt.DimensionError):
        tt.token_logprob(g.input([]), g.input([], dtype=tt.int32))
    with pytest.raises(tt.BroadcastError):
        tt.policy_loss(x, k, g.input([4]), f)
    for clip in ((-0.1, 0.2), (1.1, 0.2), (0.2, -1.0), (0.2, float("inf")), (float("nan"), 0.2), (0.2,)):
        with pytest.raises(ValueError):
            tt.policy_loss(x, k, f, f, clip=clip)
    for kw in ({"kl": 0.1}, {"ref_logp": f}, {"kl": -1.0, "ref_logp": f}, {"kl": float("nan"), "ref_logp": f},
               {"kl": 1e-60, "ref_logp": f}):  # 1e-60 is 0 in float32
        with pytest.raises(ValueError):
            tt.policy_loss(x, k, f, f, **kw)
    with pytest.raises(tt.ShapeError):
        tt.preference_loss(x, k, f)
    p, q = g.input([4, 2, 3, 7]), g.input([4, 2, 3], dtype=tt.int32)
    for kw in ({"beta": 0.0}, {"beta": float("inf")}, {"smoothing": 0.6}, {"smoothing": -0.1}):
        with pytest.raises(ValueError):
            tt.preference_loss(p, q, 0.0, **kw)
    with pytest.raises(tt.ShapeError):
        tt.preference_loss(g.input([4, 3, 3, 7]), g.input([4, 3, 3], dtype=tt.int32), 0.0)


def test_int32_goes_to_token_operators_only(cache_dir):
    g = tt.Graph()
    k = g.input([4], dtype=tt.int32)
    with pytest.raises(tt.TypeError):
        tt.add(k, g.input([4]))
    with pytest.raises(tt.TypeError):
        tt.compile(g, [k], cache_dir=cache_dir, flags=HOST)
    g = tt.Graph()
    k = g.input([4], dtype=tt.int32)
    with pytest.raises(tt.TypeError):
        tt.compile(g, [tt.relu(k)], cache_dir=cache_dir, flags=HOST)
    g, x, k = _loss_graph()
    with pytest.raises(tt.TypeError):
        tt.compile_gradients(g, tt.sum(tt.token_logprob(x, k)), [k], cache_dir=cache_dir, flags=HOST)


def test_seed_refusals(cache_dir):
    g, x, k = _loss_graph()
    y = tt.token_logprob(x, k)
    with pytest.raises(tt.ShapeError):
        tt.compile_gradients(g, y, [x], seed=g.input([3]), cache_dir=cache_dir, flags=HOST)
    with pytest.raises(tt.TypeError):
        tt.compile_gradients(g, y, [x], seed=k, cache_dir=cache_dir, flags=HOST)
    with pytest.raises(tt.IRError):
        tt.compile_gradients(g, y, [x], seed=tt.Graph().input([2, 3]), cache_dir=cache_dir, flags=HOST)


def _verify(nodes, n_inputs):
    arr = (_lib.TTNode * len(nodes))(*nodes)
    ins = (ctypes.c_int32 * n_inputs)(*range(n_inputs))
    g = _lib.TTGraph(len(nodes), arr, n_inputs, ins, 0, (ctypes.c_int32 * 1)())
    _lib.check(_lib.lib.tt_graph_verify(ctypes.byref(g)))


def _node(op, shape, inputs=(), dtype=0, attrs=None):
    n = _lib.TTNode()
    n.op, n.dtype, n.rank, n.num_inputs = op, dtype, len(shape), len(inputs)
    for i, d in enumerate(shape):
        n.shape[i] = d
    for i, q in enumerate(inputs[:2]):
        n.inputs[i] = q
    if attrs is not None:
        for i, q in enumerate(inputs[2:]):
            attrs.more_inputs[i] = q
        n.data = ctypes.addressof(attrs)
    return n


def test_c_abi_refuses_bad_nodes():
    """What the Python builders never send: the C entry answers with a status."""
    IN = _lib.OP_INPUT
    f23, f237, k23 = _node(IN, [2, 3]), _node(IN, [2, 3, 7]), _node(IN, [2, 3], dtype=2)
    at = _lib.TTOpAttrs()
    at.f[0], at.f[1] = 0.2, 0.2
    ok = [f237, k23, f23, f23, _node(_lib.OP_POLICY_LOSS, [2, 3], [0, 1, 2, 3], attrs=at)]
    _verify(ok, 4)
    bad = _lib.TTOpAttrs()
    bad.more_inputs[0], bad.more_inputs[1] = 9, 9
    n = _node(_lib.OP_POLICY_LOSS, [2, 3], [0, 1, 2, 3])
    with pytest.raises(tt.IRError):  # no attributes
        _verify(ok[:4] + [n], 4)
    n.data = ctypes.addressof(bad)
    with pytest.raises(tt.IRError):  # an operand that does not exist
        _verify(ok[:4] + [n], 4)
    at2 = _lib.TTOpAttrs()
    at2.f[0] = float("nan")
    with pytest.raises(ValueError):
        _verify(ok[:4] + [_node(_lib.OP_POLICY_LOSS, [2, 3], [0, 1, 2, 3], attrs=at2)], 4)
    with pytest.raises(tt.TypeError):  # float tokens
        _verify([f237, f23, _node(_lib.OP_TOKEN_LOGPROB, [2, 3], [0, 1])], 2)
    with pytest.raises(tt.IRError):  # scan_last of an input
        _verify([f237, _node(_lib.OP_SCAN_LAST, [2, 7], [0])], 1)
    n = _node(_lib.OP_GATED_SCAN, [2, 3, 7], [0, 0])
    n.dim0 = 3
    with pytest.raises(tt.DimensionError):
        _verify([f237, n], 1)
    with pytest.raises(tt.ShapeError):
        _verify([f237, f23, _node(_lib.OP_GATED_SCAN, [2, 3, 7], [0, 1])], 2)
    for op in (26, 64, 65, 69, 1000):  # backward nodes are not for callers
        with pytest.raises(tt.IRError):
            _verify([f237, _node(op, [2, 3, 7], [0])], 1)


def test_device_buffer_refuses_other_dtypes():
    with pytest.raises(tt.TypeError):
        tt.DeviceBuffer([2], dtype=tt.float64)
    with pytest.raises(tt.TypeError):
        tt.PinnedBuffer([2], dtype="int64")


class _FakeDevice:
    """The library with an allocator that hands out the addresses it is told to, and runs that do nothing."""

    def __init__(self, lib):
        self.lib, self.next, self.runs = lib, None, 0

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def tt_device_alloc(self, nbytes, p):
        p._obj.value = self.next
        return 0

    def tt_device_free(self, p):
        return 0

    def tt_program_run(self, *args):
        self.runs += 1
        return 0


def test_device_runs_refuse_buffers_of_the_other_dtype(cache_dir, monkeypatch):
    """Also where a buffer lies at the address of one that an earlier run had."""
    g, x, k = _loss_graph()
    prog = tt.compile(g, outputs=[tt.token_logprob(x, k)], cache_dir=cache_dir, flags=HOST)
    fake = _FakeDevice(_lib.lib)
    monkeypatch.setattr(_lib, "lib", fake)

    def buffer(address, shape, dtype=tt.float32):
        fake.next = address
        return tt.DeviceBuffer(shape, dtype=dtype)

    xb, kb, y = buffer(0x1000, [2, 3, 7]), buffer(0x2000, [2, 3], tt.int32), buffer(0x3000, [2, 3])
    for _ in range(2):
        prog.run_device([xb, kb], [y])
    prog.run_device([0x1000, 0x2000], [0x3000])
    assert fake.runs == 3
    kb.free()
    with pytest.raises(tt.TypeError):
        prog.run_device([xb, buffer(0x2000, [2, 3])], [y])
    kb = buffer(0x2000, [2, 3], tt.int32)
    prog.run_device([xb, kb], [y])
    xb.free()
    with pytest.raises(tt.TypeError):
        prog.run_device([buffer(0x1000, [2, 3, 7], tt.int32), kb], [y])
    xb = buffer(0x1000, [2, 3, 7])
    prog.run_device([xb, kb], [y])
    y.free()
    with pytest.raises(tt.TypeError):
        prog.run_device([xb, kb], [buffer(0x3000, [2, 3], tt.int32)])
    assert fake.runs == 5
    xb = kb = None  # (freed through the fake)


def test_int32_tensors():
    k = tt.tensor([[1, 2**31 - 1]], dtype=tt.int32)
    assert k.dtype == tt.int32 and k.numpy().dtype == np.int32 and k.numpy().tolist() == [[1, 2**31 - 1]]
    assert tt.tensor([1, 2]).dtype == tt.float32
    with pytest.raises(tt.TypeError):
        tt.tensor([0.5], dtype=tt.int32)
    with pytest.raises(tt.TypeError):
        tt.tensor([2**31], dtype=tt.int32)


# ---- schedule --------------------------------------------------------------------------------


def test_loss_and_gradient_share_a_launch(cache_dir):
    g, x, k = _loss_graph()
    old, adv, w = g.input([2, 3]), g.input([2, 1]), g.input([2, 3])
    y = tt.policy_loss(x, k, old, adv)
    p = tt.compile_gradients(g, y, [x], outputs=[y], seed=w, cache_dir=cache_dir, flags=HOST)
    n, lines = _launches(p)
    assert n == 1 and "policy_loss+policy_loss_grad" in lines[0]
    p = tt.compile_gradients(g, y, [x], outputs=[y], seed=w, cache_dir=cache_dir, flags=HOST | tt.FLAG_NO_FUSION)
    assert _launches(p)[0] == 2


def test_gradient_that_needs_the_loss_has_its_own_launch(cache_dir):
    g, x, k = _loss_graph()
    y = tt.token_logprob(x, k)
    p = tt.compile_gradients(g, tt.sum(y * y), [x], cache_dir=cache_dir, flags=HOST)
    lines = _launches(p)[1]
    assert not any("token_logprob+" in ln for ln in lines)
    assert sum("token_logprob" in ln for ln in lines) == 2


def test_weighted_sum_of_losses_keeps_one_loss_launch(cache_dir):
    g, x, k = _loss_graph()
    w = g.input([2, 3])
    p = tt.compile_gradients(g, tt.sum(tt.token_logprob(x, k) * w), [x], cache_dir=cache_dir, flags=HOST)
    assert any("token_logprob+token_logprob_grad" in ln for ln in _launches(p)[1])


def test_scan_gradients_share_a_launch(cache_dir):
    g = tt.Graph()
    a, x, s, d = g.input([2, 5, 3]), g.input([2, 5, 3]), g.input([2, 3]), g.input([2, 5, 3])
    h = tt.gated_scan(a, x, init=s)
    p = tt.compile_gradients(g, h, [a, x, s], outputs=[h], seed=d, cache_dir=cache_dir, flags=HOST)
    n, lines = _launches(p)
    assert n == 2 and "gated_scan_dgate+gated_scan_dx+gated_scan_dinit" in lines[1]
    # the states and their last one, both in the loss: one backward scan takes both gradients
    g2 = tt.Graph()
    a, x = g2.input([2, 5, 3]), g2.input([2, 5, 3])
    h = tt.gated_scan(a, x)
    loss = tt.sum(h * h) + tt.sum(tt.scan_last(h))
    p = tt.compile_gradients(g2, loss, [a, x], cache_dir=cache_dir, flags=HOST)
    assert sum("gated_scan_d" in ln for ln in _launches(p)[1]) == 1


def test_a_shared_gates_gradient_is_summed_in_the_scan(cache_dir):
    for gate, dh, sums in (([2, 50, 3, 1], 64, True), ([2, 50, 3, 1], 5, True), ([2, 50, 1, 64], 64, False)):
        g = tt.Graph()
        a, x, d = g.input(gate), g.input([2, 50, 3, dh]), g.input([2, 50, 3, dh])
        p = tt.compile_gradients(g, tt.gated_scan(a, x, axis=1), [a, x], outputs=[], seed=d, cache_dir=cache_dir, flags=HOST)
        assert any("reduce_sum" in ln for ln in _launches(p)[1]) != sums
        assert p.output_shapes == [gate, [2, 50, 3, dh]]


def test_states_only_scan_last_reads_are_not_stored(cache_dir):
    g = tt.Graph()
    a, x = g.input([2, 500, 3]), g.input([2, 500, 3])
    p = tt.compile(g, [tt.scan_last(tt.gated_scan(a, x))], cache_dir=cache_dir, flags=HOST)
    n, lines = _launches(p)
    assert n == 1 and lines[0].split("->")[1].split()[0] == "output:0"
    assert int(_plan(p).split("Peak ")[1].split()[0]) < 4 * 2 * 500 * 3  # joins of the axis's segments at most


def test_broadcast_and_transposed_operands_are_not_copied(cache_dir):
    g = tt.Graph()
    a, x, s = g.input([4, 6, 3, 1]), g.input([4, 3, 6, 5]), g.input([3, 5])
    h = tt.gated_scan(a, tt.transpose(x, 1, 2), init=s, axis=1)
    p = tt.compile(g, [h], cache_dir=cache_dir, flags=HOST)
    # x's dims behind the axis, (heads, channels), are not one arithmetic sequence after the
    # transpose, but the gate's split (heads | channels) fits them
    assert _launches(p)[0] == 1
    g = tt.Graph()
    x, k, adv = g.input([3, 2, 9]), g.input([2, 3], dtype=tt.int32), g.input([1, 3])
    y = tt.policy_loss(tt.transpose(x, 0, 1), k, 0.0, adv)
    assert _launches(tt.compile(g, [y], cache_dir=cache_dir, flags=HOST))[0] == 1
    g = tt.Graph()
    x, k = g.input([9, 4]), g.input([4], dtype=tt.int32)
    y = tt.token_logprob(tt.transpose(x, 0, 1), k)  # the vocabulary is not adjacent: copied
    assert _launches(tt.compile(g, [y], cache_dir=cache_dir, flags=HOST))[0] == 2


def test_steps_of_scan_and_loss_outputs(cache_dir):
    g = tt.Graph()
    a, x, w = g.input([2, 50, 8]), g.input([2, 50, 8]), g.input([8, 40])
    k, s = g.input([2, 50], dtype=tt.int32), g.input([2, 50])
    h = tt.gated_scan(a, x)
    y = tt.token_logprob(h @ w, k)
    p = tt.compile_gradients(g, y, [w, a], outputs=[y, tt.scan_last(h)], seed=s, cache_dir=cache_dir, flags=HOST)
    n = _launches(p)[0]
    out, ins = p.output_steps(), p.input_steps()
    assert out[1] == 0 and 0 < out[0] < min(out[2], out[3]) and max(out) == n - 1
    assert ins[3] == ins[4] == out[0] and ins[1] == 0 and ins[0] == out[3]  # tokens, seed, x, gate


def test_scan_last_twice_without_cse(cache_dir):
    g = tt.Graph()
    a, x = g.input([2, 50, 3]), g.input([2, 50, 3])
    h = tt.gated_scan(a, x)
    l1, l2 = tt.scan_last(h), tt.scan_last(h)
    p = tt.compile(g, [l1 + 1.0, l2, l1], optimize=False, cache_dir=cache_dir, flags=HOST)
    lines = _launches(p)[1]
    assert sum("gated_scan" in ln for ln in lines) == 1 and lines[0].count("scan_last") == 1


def test_gradient_of_an_expanded_gate_itself(cache_dir):
    """A gate that is broadcast is a gradient target too (the C ABI can name the expand node)."""
    g = tt.Graph()
    a, x, d = g.input([2, 50, 3, 1]), g.input([2, 50, 3, 64]), g.input([2, 50, 3, 64])
    h = tt.gated_scan(a, x, axis=1)
    p = tt.compile_gradients(g, h, [h.inputs[0], a], outputs=[], seed=d, cache_dir=cache_dir, flags=HOST)
    assert any("gated_scan_dgate" in ln for ln in _launches(p)[1])
    assert p.output_shapes == [[2, 50, 3, 64], [2, 50, 3, 1]]


def test_equal_nodes_merge_only_with_equal_numbers(cache_dir):
    g, x, k = _loss_graph()
    f = g.input([2, 3])
    y = [tt.policy_loss(x, k, f, f, clip=c) for c in ((0.2, 0.2), (0.2, 0.2), (0.2, 0.3))]
    p = tt.compile(g, [y[0] + y[1] + y[2]], cache_dir=cache_dir, flags=HOST)
    assert sum("policy_loss" in ln for ln in _launches(p)[1]) == 2


def test_existing_schedules_hold_a_scan_between_regions(cache_dir):
    """Elementwise nodes before and behind a scan do not merge around it."""
    g = tt.Graph()
    x = g.input([2, 5, 3])
    a = tt.sigmoid(x)
    h = tt.gated_scan(a, x * 2.0)
    p = tt.compile(g, [h * a + tt.relu(x)], cache_dir=cache_dir, flags=HOST)
    n, lines = _launches(p)
    assert [("gated_scan" in ln) for ln in lines].index(True) == n - 2


def test_the_last_states_gradient_is_the_states_own_too(cache_dir):
    """d loss / d h where the loss reads h through scan_last alone, and beside it."""
    def plan(loss, wrt):
        g = tt.Graph()
        a, x, w = g.input([2, 5, 3]), g.input([2, 5, 3]), g.input([2, 3])
        h = tt.gated_scan(a, x)
        nodes = {"h": h, "x": x}
        p = tt.compile_gradients(g, loss(h, w), [nodes[n] for n in wrt], outputs=[], cache_dir=cache_dir, flags=HOST)
        assert p.output_shapes == [[2, 5, 3]] * len(wrt)
        return _launches(p)[1]

    last = lambda h, w: tt.sum(tt.scan_last(h) * w)  # noqa: E731
    both = lambda h, w: tt.sum(tt.scan_last(h) * w) + tt.sum(h * h)  # noqa: E731
    for loss in (last, both):
        lines = plan(loss, ["h"])
        assert "mul" in lines[-1] and "output:0" in lines[-1] and not any("gated_scan_d" in ln for ln in lines)
    lines = plan(both, ["h", "x", "h"])
    assert sum("gated_scan_d" in ln for ln in lines) == 1


# ---- the definitions themselves -----------------------------------------------------------------


def _differences(f, v, eps=1e-6):
    d = np.zeros(v.shape)
    for i in np.ndindex(v.shape):
        hi, lo = v.copy(), v.copy()
        hi[i] += eps
        lo[i] -= eps
        d[i] = (f(hi) - f(lo)) / (2 * eps)
    return d


@pytest.mark.parametrize("axis", [0, 1, 2])
@pytest.mark.parametrize("init", [False, True])
def test_scan_definition_against_differences(axis, init):
    rng = np.random.default_rng(axis)
    a, x, g = rng.uniform(-1, 1, (2, 4, 3)), rng.standard_normal((2, 4, 3)), rng.standard_normal((2, 4, 3))
    lane = np.delete(np.array(x.shape), axis)
    s, gl = (rng.standard_normal(lane) if init else None), rng.standard_normal(lane)

    def f(a, x, s):
        (h, _), (last, _) = R.scan(a, x, s, axis)
        return (h * g).sum() + (last * gl).sum()

    got = R.scan_grad(a, x, s, axis, g, gl)
    assert np.allclose(got[0][0], _differences(lambda v: f(v, x, s), a), atol=1e-7)
    assert np.allclose(got[1][0], _differences(lambda v: f(a, v, s), x), atol=1e-7)
    if init:
        assert np.allclose(got[2][0], _differences(lambda v: f(a, x, v), s), atol=1e-7)


@pytest.mark.parametrize("kind", ["logprob", "policy", "policy_kl", "preference"])
def test_loss_definitions_against_differences(kind):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 2, 3, 5))
    k = rng.integers(0, 5, (2, 2, 3))
    k[0, 1, 2] = -1
    p = R.logprob(x, k)[0][0]
    old, ref, adv = p + 0.3 * rng.standard_normal(k.shape), p + 0.3, rng.standard_normal(k.shape)
    g = rng.standard_normal(2 if kind == "preference" else k.shape)
    f = {
        "logprob": lambda v, g=None: R.logprob(v, k, g),
        "policy": lambda v, g=None: R.policy(v, k, old, adv, None, (0.2, 0.3), 0.0, g),
        "policy_kl": lambda v, g=None: R.policy(v, k, old, adv, ref, (0.2, 0.3), 0.25, g),
        "preference": lambda v, g=None: R.preference(v, k, ref, 0.5, 0.125, g),
    }[kind]
    got = f(x, g)[1][0]
    want = _differences(lambda v: (f(v)[0][0] * g).sum(), x)
    assert np.allclose(got, want, atol=1e-7)


# ---- operands as the kernels address them --------------------------------------------------------


def _addressed(line):
    """(extents, {operand: (strides, offset)}) of a scan's line in the plan."""
    def ints(t):
        return [int(v) for v in t.split(",")]

    over = ints(line.split("over=[")[1].split("]")[0])
    words = line.split("over=")[1].split(" ->")[0].split()[1:]
    ops = {w.split("=")[0]: (ints(w.split("[")[1].split("]")[0]), int(w.split("+")[1])) for w in words}
    return over, ops


def _last_index(over, strides, offset):
    return offset + sum((n - 1) * s for n, s in zip(over, strides) if n > 0)


@pytest.mark.parametrize("dense_first", [True, False])
def test_scans_that_share_an_expanded_operand(cache_dir, dense_first):
    """One scan needs a dense copy of the expanded node (as its x: no split of the dense gate's dims fits it),
    the other reads it in place as its gate: neither's split or strides depend on the other."""
    g = tt.Graph()
    a, y, d = g.input([2, 5, 3, 1]), g.input([2, 5, 4, 3]), g.input([2, 5, 3, 4])

    def dense():
        return tt.gated_scan(d, a, axis=1)

    def shared():
        return tt.gated_scan(a, tt.transpose(y, 2, 3), axis=1)

    h = [dense(), shared()] if dense_first else [shared(), dense()][::-1]
    lines = [ln for ln in _launches(tt.compile(g, h, cache_dir=cache_dir, flags=HOST))[1] if "gated_scan" in ln]
    seen = {}
    for ln in lines:
        over, ops = _addressed(ln)
        seen[ln.split("output:")[1].split()[0]] = (over, ops)
        assert int(np.prod(over)) == 120
        assert all(_last_index(over, s, o) < 120 for s, o in ops.values())
    assert seen["0"] == ([2, 5, 1, 12], {"gate": ([60, 12, 0, 1], 0), "x": ([60, 12, 0, 1], 0)})
    assert seen["1"] == ([2, 5, 3, 4], {"gate": ([15, 3, 1, 0], 0), "x": ([60, 12, 1, 3], 0)})


def test_scans_over_shared_views_stay_inside_their_operands(cache_dir):
    """Scans and their gradients over one pool of expanded and transposed nodes, in random roles and orders."""
    rng = np.random.default_rng(0)
    for _ in range(40):
        g = tt.Graph()
        full = [2, 5, 3, 4]
        leaves = [g.input([2, 5, 3, 1]), g.input([2, 5, 4, 3]), g.input(full), g.input([1, 5, 1, 4]), g.input([2, 3, 5, 4])]
        pool = [leaves[0], tt.transpose(leaves[1], 2, 3), leaves[2], leaves[3], tt.transpose(leaves[4], 1, 2)]
        hs = []
        for _ in range(4):
            i, j = rng.integers(0, len(pool), 2)
            if pool[i].shape != full and pool[j].shape != full:
                j = 2
            hs.append(tt.gated_scan(pool[i], pool[j], axis=int(rng.integers(0, 4))))
        loss = hs[0] * hs[1]
        for h in hs[2:]:
            loss = loss + h
        p = tt.compile_gradients(g, tt.sum(loss), leaves, outputs=hs, cache_dir=cache_dir, flags=HOST)
        lines = [ln for ln in _launches(p)[1] if "gated_scan" in ln]
        assert lines
        for ln in lines:
            over, ops = _addressed(ln)
            assert int(np.prod(over)) == 120
            for name, (s, o) in ops.items():
                extents = [over[0], 1, over[2], over[3]] if name in ("carry", "init") else over
                assert _last_index(extents, s, o) < 120, ln
