"""The layers and the stepper built on the sequence, norm and update operators: gradients against differences on the
64-bit oracle (CPU), and the whole network, stepped, on the GPU against the oracle."""
import numpy as np
import pytest

from brainstorm_amd.drivers import configs
from brainstorm_amd.drivers.layers import FullyConnected, GatedResidual, Input, LinearAttention, Loss, Lstm, SoftmaxCE
from brainstorm_amd.drivers.net import MomentumStepper, Net, OrthogonalStepper
from oracle.sequence_ops import SequenceRefHandler

F32 = np.float32
SMALL = dict(time_steps=5, batch=3, symbols=7, hidden=12, heads=3, blocks=2)


def loss_of(net, data, params):
    net.set_parameters(params)
    net.provide_external_data(data)
    net.forward_pass(training_pass=True)
    return float(net.get("loss", "outputs", "loss")[0])


def test_gradients_of_the_network_are_the_differences():
    net, data = configs.build_attention(SequenceRefHandler(np.float64, seed=1), fused=False, **SMALL)
    rng = np.random.RandomState(2)
    params = net.handler.get_numpy_copy(net.parameters) + 0.3 * rng.standard_normal(net.parameters.shape)
    loss_of(net, data, params)
    net.backward_pass()
    grads = net.handler.get_numpy_copy(net.gradients)
    for name, (a, b, _) in net.parameter_slices().items():
        for i in np.unique(np.linspace(a, b - 1, min(b - a, 7)).astype(int)):
            moved = []
            for sign in (1, -1):
                p = params.copy()
                p[i] += sign * 1e-6
                moved.append(loss_of(net, data, p))
            np.testing.assert_allclose(grads[i], (moved[0] - moved[1]) / 2e-6, rtol=1e-4, atol=1e-7, err_msg=name)


def test_backward_pass_adds_to_input_deltas():
    net, data = configs.build_attention(SequenceRefHandler(np.float64, seed=1), fused=False, **SMALL)
    net.provide_external_data(data)
    net.forward_pass(training_pass=True)
    net.backward_pass()
    once = net.get("embed", "output_deltas", "default").copy()
    for name in ("end0", "attend0", "norm"):
        before = {n: d.copy() for n, d in net.buffers[name].input_deltas.items()}
        net.layers[name].backward_pass(net.buffers[name])
        assert any(not np.array_equal(d, before[n]) for n, d in net.buffers[name].input_deltas.items()), name
    assert not np.array_equal(net.get("embed", "output_deltas", "default"), once)


def shared_sources(handler, fused):
    """A network whose GatedResidual layers take two and three of their inputs from one output."""
    layers = [("Input", Input({"default": (9,), "targets": (1,)}), {}),
              ("embed", FullyConnected(12, "tanh", fused=fused), {"default": "Input.default"}),
              ("gate", FullyConnected(12, "linear", fused=fused), {"default": "embed.default"}),
              ("first", GatedResidual("sigmoid", 0.5), {"block": "embed.default", "gate": "gate.default", "x": "embed.default"}),
              ("second", GatedResidual("tanh"), {"block": "first.default", "gate": "first.default", "x": "first.default"}),
              ("third", GatedResidual("swish"), {"block": "second.default", "gate": "second.default", "x": "second.residual"}),
              ("out", FullyConnected(5, "linear", fused=fused), {"default": "third.default"}),
              ("ce", SoftmaxCE(fused=fused), {"default": "out.default", "targets": "Input.targets"}),
              ("loss", Loss(), {"default": "ce.loss"})]
    net = Net(handler, layers)
    rng = np.random.RandomState(4)
    data = {"default": rng.standard_normal((3, 4, 9)).astype(F32), "targets": rng.randint(0, 5, (3, 4, 1)).astype(F32)}
    net.provide_external_data(data)
    return net, data, 0.5 * rng.standard_normal(net.parameter_count()) + 0.2


def test_inputs_from_one_output():
    net, data, params = shared_sources(SequenceRefHandler(np.float64, seed=1), False)
    loss_of(net, data, params)
    net.backward_pass()
    grads = net.handler.get_numpy_copy(net.gradients)
    for name, (a, b, _) in net.parameter_slices().items():
        for i in np.unique(np.linspace(a, b - 1, min(b - a, 5)).astype(int)):
            moved = []
            for sign in (1, -1):
                p = params.copy()
                p[i] += sign * 1e-6
                moved.append(loss_of(net, data, p))
            np.testing.assert_allclose(grads[i], (moved[0] - moved[1]) / 2e-6, rtol=1e-4, atol=1e-7, err_msg=name)


@pytest.mark.gpu
def test_inputs_from_one_output_on_the_gpu(hip):
    # 2e-4 of each array's scale, as for the network below
    got = []
    for handler, fused in ((hip, True), (SequenceRefHandler(np.float64, seed=1), False)):
        net, _, params = shared_sources(handler, fused)
        net.set_parameters(params if handler is not hip else params.astype(F32))
        net.forward_pass(training_pass=True)
        net.backward_pass()
        got.append((net.handler.get_numpy_copy(net.gradients), net.parameter_slices()))
    for name, (a, b, _) in got[1][1].items():
        want = got[1][0][a:b]
        assert np.abs(got[0][0][a:b] - want).max() <= 2e-4 * np.abs(want).max(), name


def test_orthogonal_stepper_groups_equal_neighbours():
    net, data = configs.build_attention(SequenceRefHandler(np.float64, seed=1), fused=False, **SMALL)
    stepper = OrthogonalStepper()
    stepper.start(net)
    covered = np.zeros(net.parameter_count(), int)
    for first, end, matrix in stepper.groups:
        covered[first:end] += 1
        assert matrix is None or (end - first) % (matrix[0] * matrix[1]) == 0
    assert (covered == 1).all()
    a, _, _ = net.parameter_slices()["attend0.Wq"]
    assert [a, a + 3 * 144, (12, 12)] in stepper.groups                # Wq, Wk and Wv in one call
    # one step: every group as the formulas have it
    before = net.handler.get_numpy_copy(net.parameters)
    net.provide_external_data(data)
    stepper.run()
    grads, after = net.handler.get_numpy_copy(net.gradients), net.handler.get_numpy_copy(net.parameters)
    g = grads[a:a + 144].reshape(12, 12)
    from oracle.sequence_ops import orthogonalize
    np.testing.assert_allclose(after[a:a + 144].reshape(12, 12), before[a:a + 144].reshape(12, 12)
                               - 0.02 * orthogonalize(g + 0.95 * g), rtol=1e-12, atol=1e-14)
    b, e, _ = net.parameter_slices()["end0.post"]
    np.testing.assert_allclose(after[b:e], before[b:e] - 0.01 * grads[b:e], rtol=1e-12, atol=1e-14)


def two_nets(hip, **kw):
    kw = dict(dict(time_steps=37, batch=6, symbols=30, hidden=96, heads=4, blocks=2), **kw)
    net_h, data = configs.build_attention(hip, fused=True, **kw)
    net_r, _ = configs.build_attention(SequenceRefHandler(np.float64, seed=1), fused=False, **kw)
    for net in (net_h, net_r):
        net.provide_external_data(data)
    return net_h, net_r


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(time_steps=150, batch=2, hidden=60, heads=5), dict(time_steps=3, hidden=64, heads=1)])
def test_network_on_the_gpu(hip, kw):
    # Tolerance: the matrix products are hipBLASLt's, held to 1e-5 of their scale elsewhere; here a chain of about
    # 20 of them forwards and backwards through two blocks: 20 * 1e-5 = 2e-4 of each array's own scale.
    net_h, net_r = two_nets(hip, **kw)
    for net in (net_h, net_r):
        net.forward_pass(training_pass=True)
        net.backward_pass()
    for layer, group, name in (("attend0", "outputs", "default"), ("end0", "outputs", "residual"),
                               ("end1", "outputs", "default"), ("out", "outputs", "default"),
                               ("attend0", "internals", "dq"), ("end0", "output_deltas", "residual")):
        got, want = net_h.get(layer, group, name), net_r.get(layer, group, name)
        assert np.abs(got - want).max() <= 2e-4 * np.abs(want).max(), (layer, group, name)
    got, want = hip.get_numpy_copy(net_h.gradients), net_r.handler.get_numpy_copy(net_r.gradients)
    for name, (a, b, _) in net_h.parameter_slices().items():
        assert np.abs(got[a:b] - want[a:b]).max() <= 2e-4 * np.abs(want[a:b]).max(), name


@pytest.mark.gpu
def test_steps_on_the_gpu_recorded_and_not(hip):
    # a step from the oracle's own gradients: the update alone, at the update's tolerance
    net_h, net_r = two_nets(hip)
    stepper = OrthogonalStepper()
    stepper.start(net_h)
    before = hip.get_numpy_copy(net_h.parameters)
    stepper.run()
    grads, after = hip.get_numpy_copy(net_h.gradients), hip.get_numpy_copy(net_h.parameters)
    from oracle.sequence_ops import orthogonalize
    for first, end, matrix in stepper.groups:
        if matrix is None:
            continue
        shape = (-1,) + matrix
        g = grads[first:end].astype(np.float64).reshape(shape)
        moved = 0.02 * np.sqrt(max(1.0, matrix[0] / matrix[1])) * orthogonalize(F32(1.95) * g)
        want = before[first:end].reshape(shape) - moved
        off = np.linalg.norm(after[first:end].reshape(shape) - want)
        assert off <= 1.4e-4 * np.linalg.norm(moved) + 2.0 ** -23 * 2 * np.linalg.norm(want)
    # recorded steps give the bits of ordinary ones
    eager = [hip.get_numpy_copy(net_h.parameters)]
    for _ in range(3):
        stepper.run()
        eager.append(hip.get_numpy_copy(net_h.parameters))
    net_2, _ = two_nets(hip)
    second = OrthogonalStepper()
    second.start(net_2)
    second.run()
    assert np.array_equal(hip.get_numpy_copy(net_2.parameters), eager[0])
    for want in eager[1:]:
        second.run_recorded()
        assert np.array_equal(hip.get_numpy_copy(net_2.parameters), want)
    second.release_recorded()


@pytest.mark.gpu
def test_serving_a_trained_layer_token_by_token(hip):
    # the layer's sequence output, again from single steps with the state kept
    net, _ = two_nets(hip)
    net.forward_pass(training_pass=False)
    layer, buffers = net.layers["attend0"], net.buffers["attend0"]
    q, k, v, g = (buffers.internals[n] for n in ("q", "k", "v", "g"))
    want = hip.get_numpy_copy(buffers.outputs["default"])
    state = hip.zeros((6, 4, 24, 24))
    out = hip.zeros((6, 96))
    for t in range(37):
        hip.linear_attention_step(q[t], k[t], v[t], g, state, out, scale=layer.scale)
        assert np.abs(out.get() - want[t]).max() <= 1e-5 * np.abs(want).max()


@pytest.mark.gpu
def test_orthogonal_stepper_trains_any_network(hip):
    # every kind of parameter: matrices, filters, vectors; the step is finite and moves each of them
    for build, kw in ((configs.build_mlp, dict(batch=5, in_size=17, hidden=11)), (configs.build_cnn, dict(batch=2, size=16)),
                      (configs.build_lstm, dict(time_steps=4, batch=3, symbols=9, hidden=8))):
        net, data = build(hip, **kw)
        net.provide_external_data(data)
        stepper = OrthogonalStepper()
        stepper.start(net)
        before = hip.get_numpy_copy(net.parameters)
        stepper.run()
        after, grads = hip.get_numpy_copy(net.parameters), hip.get_numpy_copy(net.gradients)
        assert np.isfinite(after).all()
        for name, (a, b, _) in net.parameter_slices().items():
            assert not grads[a:b].any() or (after[a:b] != before[a:b]).any(), name


def test_momentum_stepper_is_unchanged():
    stepper = MomentumStepper(0.1, 0.5)
    assert (stepper.learning_rate, stepper.momentum, stepper.scale_learning_rate, stepper.fused) == (0.1, 0.5, True, False)


class OutputsApart(SequenceRefHandler):
    """The oracle with HipHandler's refusal of outputs that share memory."""

    def gated_residual_backward(self, activation, block, gate, post_weight, pre_weight, y, dy, dh, dblock, dgate, dx, *args,
                                **kwargs):
        outputs = [a for a in (dblock, dgate, dx) if a is not None]
        if any(np.shares_memory(a, b) for n, a in enumerate(outputs) for b in outputs[:n]):
            raise ValueError("two outputs overlap")
        super().gated_residual_backward(activation, block, gate, post_weight, pre_weight, y, dy, dh, dblock, dgate, dx, *args,
                                        **kwargs)


def recurrent_source(handler, fused, inputs):
    """An Lstm, whose buffers have a context slot, as the source of a GatedResidual's `inputs`."""
    layers = [("Input", Input({"default": (9,), "targets": (1,)}), {}),
              ("lstm", Lstm(12, fused=fused), {"default": "Input.default"}),
              ("other", FullyConnected(12, "linear", fused=fused), {"default": "lstm.default"}),
              ("end", GatedResidual("swish"), {n: ("lstm" if n in inputs else "other") + ".default"
                                               for n in ("block", "gate", "x")}),
              ("out", FullyConnected(5, "linear", fused=fused), {"default": "end.default"}),
              ("ce", SoftmaxCE(fused=fused), {"default": "out.default", "targets": "Input.targets"}),
              ("loss", Loss(), {"default": "ce.loss"})]
    net = Net(handler, layers)
    rng = np.random.RandomState(7)
    data = {"default": rng.standard_normal((3, 4, 9)).astype(F32), "targets": rng.randint(0, 5, (3, 4, 1)).astype(F32)}
    net.provide_external_data(data)
    return net, data, 0.5 * rng.standard_normal(net.parameter_count()) + 0.2


SHARED = [("block", "gate", "x"), ("block", "gate"), ("block", "x"), ("gate", "x")]


@pytest.mark.parametrize("inputs", SHARED)
def test_inputs_from_one_recurrent_output(inputs):
    net, data, params = recurrent_source(OutputsApart(np.float64, seed=1), False, inputs)
    loss_of(net, data, params)
    net.backward_pass()
    want, want_data, _ = recurrent_source(SequenceRefHandler(np.float64, seed=1), False, inputs)
    loss_of(want, want_data, params)
    want.backward_pass()
    np.testing.assert_allclose(net.handler.get_numpy_copy(net.gradients), want.handler.get_numpy_copy(want.gradients),
                               rtol=1e-12, atol=1e-14)


@pytest.mark.gpu
@pytest.mark.parametrize("inputs", SHARED)
def test_inputs_from_one_recurrent_output_on_the_gpu(hip, inputs):
    # 2e-4 of each array's scale, as for the networks above
    got = []
    for handler, fused in ((hip, True), (SequenceRefHandler(np.float64, seed=1), False)):
        net, _, params = recurrent_source(handler, fused, inputs)
        net.set_parameters(params if handler is not hip else params.astype(F32))
        net.forward_pass(training_pass=True)
        net.backward_pass()
        got.append((net.handler.get_numpy_copy(net.gradients), net.parameter_slices()))
    for name, (a, b, _) in got[1][1].items():
        want = got[1][0][a:b]
        assert np.abs(got[0][0][a:b] - want).max() <= 2e-4 * np.abs(want).max(), name


def test_heads_that_the_operator_does_not_take_are_refused_by_the_layer():
    assert LinearAttention(1024, 8).scale == 128 ** -0.5
    for size, heads in ((1032, 8), (129, 1), (10, 3), (0, 2), (8, 0), (-8, -2)):
        with pytest.raises(ValueError):
            LinearAttention(size, heads)
