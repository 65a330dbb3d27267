"""CPU: the 64-bit oracle of the sequence, norm and update operators against differences, and the calls that
HipHandler refuses before anything reaches the library."""
import numpy as np
import pytest

from oracle import sequence_ops as ops


def slopes_by_differences(f, arrays, step=1e-6):
    """Central differences of the scalar f(*arrays) by every element of every array."""
    out = []
    for n, a in enumerate(arrays):
        d = np.zeros(a.shape)
        for i in np.ndindex(*a.shape):
            values = []
            for sign in (1, -1):
                moved = [x.copy() for x in arrays]
                moved[n][i] += sign * step
                values.append(f(*moved))
            d[i] = (values[0] - values[1]) / (2 * step)
        out.append(d)
    return out


@pytest.mark.parametrize("lengths", [None, [4.0, 0.0, 2.9]])
def test_linear_attention_gradients_are_the_differences(lengths):
    rng = np.random.RandomState(1)
    time, batch, heads, dk, dv = 4, 3, 2, 2, 3
    q, k = (rng.standard_normal((time, batch, heads * dk)) for _ in range(2))
    v, dout = (rng.standard_normal((time, batch, heads * dv)) for _ in range(2))
    decay, state = np.array([0.8, 0.3]), rng.standard_normal((batch, heads, dk, dv))
    dnew = rng.standard_normal(state.shape)

    def loss(q, k, v, decay, state):
        out, new = ops.linear_attention(q, k, v, decay, 0.7, state, lengths)
        return (out * dout).sum() + (new * dnew).sum()

    want = slopes_by_differences(loss, [q, k, v, decay, state])
    got = ops.linear_attention_gradients(q, k, v, decay, dout, 0.7, state, dnew, lengths)
    for a, b in zip(got, want):
        np.testing.assert_allclose(a, b, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("activation", ["linear", "sigmoid", "tanh", "rel", "el", "swish", None])
def test_gated_residual_gradients_are_the_differences(activation):
    rng = np.random.RandomState(2)
    block, gate, x, dy, dh = (rng.standard_normal((3, 5)) for _ in range(5))
    post, pre = 1 + 0.3 * rng.standard_normal((2, 5))
    with_gate = gate if activation else None

    def loss(block, gate, x, post, pre):
        y, h = ops.gated_residual(activation, block, gate if activation else None, x, post, pre, 0.9, 1e-3)
        return (y * dy).sum() + (h * dh).sum()

    want = slopes_by_differences(loss, [block, gate, x, post, pre])
    y, _ = ops.gated_residual(activation, block, with_gate, x, post, pre, 0.9, 1e-3)
    got = ops.gated_residual_gradients(activation, block, with_gate, post, pre, y, dy, dh, 0.9, 1e-3)
    for name, d in zip(("dblock", "dgate", "dx", "dpost", "dpre"), want):
        if name in got:
            np.testing.assert_allclose(got[name], d, rtol=1e-6, atol=1e-7, err_msg=name)


def test_orthogonalize_brings_singular_values_to_about_one():
    rng = np.random.RandomState(3)
    for shape in ((6, 6), (4, 9), (9, 4), (1, 5), (5, 1)):
        s = np.linalg.svd(ops.orthogonalize(rng.standard_normal(shape) * 1e-3), compute_uv=False)
        assert s.max() < 1.21 and s.max() > 0.6
    assert not ops.orthogonalize(np.zeros((3, 2))).any()


def refused(h):
    A = lambda *shape: h.allocate(shape)
    q, k, v, out = A(6, 2, 8), A(6, 2, 8), A(6, 2, 12), A(6, 2, 12)
    decay, state, lengths = A(4), A(2, 4, 2, 3), A(2)
    wide = A(3, 1, 516)
    m, n, w = A(4, 6), A(4, 7), A(6)
    dq, dk, dv = A(6, 2, 8), A(6, 2, 8), A(6, 2, 12)
    fwd, bwd = h.linear_attention_forward, h.linear_attention_backward
    gate, gate_back = h.gated_residual_forward, h.gated_residual_backward
    stack = A(3, 4, 6)
    flat = A(200)
    near = lambda at: flat[at:at + 144].reshape((6, 2, 12))
    return [
        ("k of another length", lambda: fwd(q, A(5, 2, 8), v, decay, out)),
        ("v of another batch", lambda: fwd(q, k, A(6, 3, 12), decay, out)),
        ("out of another size", lambda: fwd(q, k, v, decay, A(6, 2, 8))),
        ("features that are not whole heads", lambda: fwd(q, k, v, A(3), out)),
        ("no heads", lambda: fwd(q, k, v, A(0), out)),
        ("matrices", lambda: fwd(A(6, 8), A(6, 8), A(6, 12), decay, A(6, 12))),
        ("a state of another size", lambda: fwd(q, k, v, decay, out, state=A(2, 4, 3, 3))),
        ("a new state of another size", lambda: fwd(q, k, v, decay, out, new_state=A(2, 4, 2, 2))),
        ("lengths of another batch", lambda: fwd(q, k, v, decay, out, lengths=A(3))),
        ("heads wider than 128", lambda: fwd(wide, wide, wide, decay, A(3, 1, 516))),
        ("out is v", lambda: fwd(q, k, v, decay, v)),
        ("out overlaps v", lambda: fwd(q, k, near(0), decay, near(4))),
        ("new_state is decay", lambda: fwd(A(6, 1, 2), A(6, 1, 2), A(6, 1, 2), decay[:2], A(6, 1, 2), new_state=decay[:2])),
        ("a state that is not the new one overlaps it",
         lambda: fwd(q, k, v, decay, out, state=flat[0:48], new_state=flat[4:52])),
        ("step of another batch", lambda: h.linear_attention_step(q[0], k[0], v[0], decay, A(1, 4, 2, 3), out[0])),
        ("step on a sequence's arrays", lambda: h.linear_attention_step(q, k, v, decay, state, out)),
        ("dq of another size", lambda: bwd(q, k, v, decay, out, A(6, 2, 7), dk, dv)),
        ("ddecay of another size", lambda: bwd(q, k, v, decay, out, dq, dk, dv, A(3))),
        ("dout of another size", lambda: bwd(q, k, v, decay, A(6, 2, 8), dq, dk, dv)),
        ("dstate of another size", lambda: bwd(q, k, v, decay, out, dq, dk, dv, dstate=A(2, 4, 2, 2))),
        ("dq is q", lambda: bwd(q, k, v, decay, out, q, dk, dv)),
        ("dq is dk", lambda: bwd(q, k, v, decay, out, dq, dq, dv)),
        ("dstate is state", lambda: bwd(q, k, v, decay, out, dq, dk, dv, state=state, dstate=state)),
        ("gate of another width", lambda: gate("linear", m, n, m, w, w, m, m)),
        ("post weight of another width", lambda: gate("linear", m, m, m, A(7), w, m, m)),
        ("no h with a pre weight", lambda: gate("linear", m, m, m, w, w, m, None)),
        ("three axes", lambda: gate("linear", stack, None, stack, w, w, stack, stack)),
        ("no dgate", lambda: gate_back("linear", m, m, w, w, m, m, m, m, None, m, w, w)),
        ("no dh", lambda: gate_back("linear", m, m, w, w, m, m, None, m, m, m, w, w)),
        ("y is h", lambda: gate("linear", m, m, m, w, w, m, m)),
        ("dblock is dgate", lambda: gate_back("linear", m, m, w, w, m, m, m, m, m, A(4, 6), A(6), A(6))),
        ("dgate overlaps dx",
         lambda: gate_back("linear", m, m, w, w, m, m, m, m, flat[0:24].reshape((4, 6)), flat[6:30].reshape((4, 6)), A(6), A(6))),
        ("dpost is dpre", lambda: gate_back("linear", m, m, w, w, m, m, m, m, A(4, 6), A(4, 6), w, w)),
        ("norm weight", lambda: h.rms_norm_forward(m, A(7), m)),
        ("norm out", lambda: h.rms_norm_forward(m, w, n)),
        ("norm gradient", lambda: h.rms_norm_backward(m, w, n, m, w)),
        ("orthogonalize into another shape", lambda: h.orthogonalize(m, A(6, 4))),
        ("orthogonalize a vector", lambda: h.orthogonalize(w, A(6))),
        ("orthogonalize four axes", lambda: h.orthogonalize(A(1, 2, 3, 4), A(1, 2, 3, 4))),
        ("orthogonalize into an overlapping matrix",
         lambda: h.orthogonalize(flat[0:24].reshape((4, 6)), flat[6:30].reshape((4, 6)))),
        ("update of another shape", lambda: h.orthogonal_update(0.9, -0.1, m, n, m)),
        ("update with velocity in the gradients", lambda: h.orthogonal_update(0.9, -0.1, m, m, A(4, 6))),
        ("update with velocity in the parameters", lambda: h.orthogonal_update(0.9, -0.1, A(4, 6), m, m)),
    ]


def test_calls_that_do_not_fit_are_refused(trace):
    from brainstorm_amd import HipHandler
    h = HipHandler(seed=1)
    for what, call in refused(h):
        with pytest.raises(ValueError):
            call()
            pytest.fail("not refused: " + what)


def test_unknown_gate_activation(trace):
    from brainstorm_amd import HipHandler
    h = HipHandler(seed=1)
    m, w = h.allocate((4, 6)), h.allocate((6,))
    with pytest.raises(ValueError):
        h.gated_residual_forward("softplus", m, m, m, w, w, m, m)


def overlapping(h):
    """Calls of the norms whose outputs share memory with an input that they are not."""
    A = lambda *shape: h.allocate(shape)
    flat = A(200)
    at = lambda first: flat[first:first + 24].reshape((4, 6))
    weight = lambda first: flat[first:first + 6]
    m, w = A(4, 6), A(6)
    gate, back = h.gated_residual_forward, h.gated_residual_backward
    fresh = lambda: (A(4, 6), A(4, 6), A(4, 6), A(6), A(6))

    def gradients(where, first):
        grads = list(fresh())
        grads[where] = at(first) if where < 3 else weight(first)
        return grads

    calls = []
    for shift in (1, 6):                        # by an element, by a row; up and down
        for a, b in ((0, shift), (shift, 0)):
            calls += [
                ("y over x", lambda a=a, b=b: gate("tanh", m, m, at(a), w, w, at(b), A(4, 6))),
                ("y over block", lambda a=a, b=b: gate("tanh", at(a), m, m, w, w, at(b), A(4, 6))),
                ("y over gate, no norm behind", lambda a=a, b=b: gate("tanh", m, at(a), m, w, None, at(b), None)),
                ("h over x", lambda a=a, b=b: gate("tanh", m, m, at(a), w, w, A(4, 6), at(b))),
                ("the norm's out over x", lambda a=a, b=b: h.rms_norm_forward(at(a), w, at(b))),
                ("the norm's dx over x", lambda a=a, b=b: h.rms_norm_backward(at(a), w, m, at(b), A(6))),
                ("the norm's dx over dout", lambda a=a, b=b: h.rms_norm_backward(m, w, at(a), at(b), A(6)))]
            for where, name in enumerate(("dblock", "dgate", "dx")):
                for n, of in enumerate(("block", "gate", "y", "dy", "dh")):
                    def call(where=where, n=n, a=a, b=b):
                        x = [m] * 5
                        x[n] = at(a)
                        back("tanh", x[0], x[1], w, w, x[2], x[3], x[4], *gradients(where, b))
                    calls.append(("%s over %s" % (name, of), call))
    calls += [
        ("y over post", lambda: gate("tanh", m, m, m, weight(6), w, at(0), A(4, 6))),
        ("h over pre", lambda: gate("tanh", m, m, m, w, weight(6), A(4, 6), at(0))),
        ("y is post", lambda: gate("tanh", m[:1], m[:1], m[:1], w, A(6), w.reshape((1, 6)), A(1, 6))),
        ("dx over pre", lambda: back("tanh", m, m, w, weight(6), m, m, m, *gradients(2, 0))),
        ("dblock over post", lambda: back("tanh", m, m, weight(6), w, m, m, m, *gradients(0, 0))),
        ("dpost over dy", lambda: back("tanh", m, m, w, w, m, at(0), m, *gradients(3, 6))),
        ("dpre over post", lambda: back("tanh", m, m, weight(1), w, m, m, m, *gradients(4, 0))),
        ("the norm's out over weight", lambda: h.rms_norm_forward(m, weight(6), at(0))),
        ("the norm's dx over weight", lambda: h.rms_norm_backward(m, weight(6), m, at(0), A(6))),
        ("the norm's dweight over x", lambda: h.rms_norm_backward(at(0), w, m, A(4, 6), weight(6))),
    ]
    return calls


def test_outputs_that_overlap_an_input_are_refused(trace):
    from brainstorm_amd import HipHandler
    h = HipHandler(seed=1)
    for what, call in overlapping(h):
        with pytest.raises(ValueError, match="overlap"):
            call()
            pytest.fail("not refused: " + what)


def test_outputs_in_an_inputs_place_reach_the_library(trace):
    # the calls that stay allowed: the stand-in library has none of these entry points, which is how a call that gets there ends
    from brainstorm_amd import HipHandler
    h = HipHandler(seed=1)
    A = lambda *shape: h.allocate(shape)
    for inputs in range(5):
        for output in range(3):
            x, grads = [A(4, 6) for _ in range(5)], [A(4, 6) for _ in range(3)]
            grads[output] = x[inputs]
            w = [A(6), A(6)]
            for accumulate in (False, True):
                with pytest.raises(AttributeError, match="bship_gated_residual_bwd_f32"):
                    h.gated_residual_backward("tanh", x[0], x[1], *w, *x[2:], *grads, *w, accumulate=accumulate)
    for inputs in range(3):
        x = [A(4, 6) for _ in range(3)]
        for outputs in ((x[inputs], A(4, 6)), (A(4, 6), x[inputs]), (x[inputs], x[inputs - 1])):
            with pytest.raises(AttributeError, match="bship_gated_residual_fwd_f32"):
                h.gated_residual_forward("tanh", *x, A(6), A(6), *outputs)
    m, w = A(4, 6), A(6)
    with pytest.raises(AttributeError, match="bship_gated_residual_fwd_f32"):
        h.rms_norm_forward(m, w, m)
    for x, dout in ((m, A(4, 6)), (A(4, 6), m)):
        with pytest.raises(AttributeError, match="bship_gated_residual_bwd_f32"):
            h.rms_norm_backward(x, w, dout, m, w)


def test_apart():
    from brainstorm_amd._fastcall import apart
    from brainstorm_amd.device_array import DeviceArray
    a = lambda ptr, n: DeviceArray(ptr, (n,), None)
    assert apart() and apart(None) and apart(a(1024, 4), None, a(1040, 4), a(1008, 4), a(1028, 0), a(0, 0), a(0, 0))
    for ptr, n in ((1024, 4), (1020, 2), (1036, 1), (1000, 100), (1028, 1)):
        assert not apart(a(1024, 4), a(ptr, n)) and not apart(a(ptr, n), a(5000, 3), None, a(1024, 4))
    with pytest.raises(TypeError, match="at most 24"):
        apart(*[None] * 25)
    with pytest.raises(AttributeError):
        apart(a(1024, 4), 7)


def test_shared_elements_of_row_pitched_views():
    # every pair of a few dense and pitched views of one buffer, against the sets of their elements
    from brainstorm_amd.device_array import DeviceArray, PitchedDeviceArray
    from brainstorm_amd.hip_handler import _share_elements
    views = []
    for first in (0, 1, 3, 5, 7, 12, 20, 29):
        for n in (0, 1, 2, 6, 11):
            views.append((DeviceArray(4096 + 4 * first, (n,), None), set(range(first, first + n))))
        for rows, run, pitch in ((1, 3, 7), (2, 3, 7), (4, 1, 7), (3, 6, 7), (3, 2, 5), (2, 4, 5)):
            elements = {first + r * pitch + c for r in range(rows) for c in range(run)}
            views.append((PitchedDeviceArray(4096 + 4 * first, (rows, run), pitch, None, None), elements))
    for a, of_a in views:
        for b, of_b in views:
            pitches = {v.pitch for v in (a, b) if type(v) is PitchedDeviceArray and v.rows > 1}
            if len(pitches) < 2:
                assert _share_elements(a, b) == bool(of_a & of_b), (a, b)
            else:                                         # may be taken for overlapping, never for apart
                assert _share_elements(a, b) or not of_a & of_b, (a, b)


def test_row_pitched_outputs_that_overlap_are_refused(trace):
    from brainstorm_amd import HipHandler
    h = HipHandler(seed=1, pitched_views=True)
    A = lambda *shape: h.allocate(shape)
    hub, m, w = A(4, 20), A(4, 6), A(6)
    x, s = A(5, 2, 8), A(2, 2, 4, 4)
    wide = A(5, 2, 20)
    with pytest.raises(ValueError, match="two outputs overlap"):
        h.gated_residual_forward("tanh", m, m, m, w, w, hub[:, 2:8], hub[:, 7:13])
    with pytest.raises(ValueError, match="two outputs overlap"):
        h.gated_residual_backward("tanh", m, m, w, w, m, m, m, hub[:, 2:8], A(4, 6), hub[:, 3:9], A(6), A(6))
    with pytest.raises(ValueError, match="two outputs overlap"):
        h.linear_attention_backward(x, x, x, A(2), x, wide[:, :, :8], wide[:, :, 8:16], wide[:, :, 12:20])
    with pytest.raises(ValueError, match="two outputs overlap"):
        h.orthogonal_update(0.9, -0.1, m, hub[:, 1:7], hub[:, :6])
