"""GPU: the norms around a block with gate and residual scale, forward and backward, against 64 bits.

Tolerance (u = 2^-24). A row's sum of squares is formed by at most 4 ceil(width / 256) additions per thread (rows
up to 1024) or 4 ceil(width / 1024), a tree of eight more and a few products: its square root is off by at most
half of that, relative. The gate's value is within 8 u (1 + |value|) for every activation used here (exp, tanh and
expm1 within 2 units, then at most three roundings). So y is off by at most c u (|residual_scale x| + |gate post
n|) with c = 24 + 2 width / 256, and h by its share of that and of the second norm. Gradients: each is a chain of at
most four such factors and three row means, whose terms' absolute values are added up; 4 c bounds the chain, and
the slope of the gate adds 8 u (1 + |z|) absolute.
"""
import numpy as np
import pytest

from oracle import sequence_ops as ops
from util import assert_bit_equal

pytestmark = pytest.mark.gpu
F32 = np.float32
U = 2.0 ** -24
EPS = 1e-5


def inputs(seed, rows, width):
    rng = np.random.RandomState(seed)
    a = {n: rng.standard_normal((rows, width)).astype(F32) for n in ("block", "gate", "x", "dy", "dh")}
    a["post"], a["pre"] = (1 + 0.2 * rng.standard_normal((2, width))).astype(F32)
    return a


def c_of(width):
    return 24 + 2 * width / 256


def close(got, want, bound, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound + 2.0 ** -126)
    assert not bad.any(), "%s: %d of %d elements off, worst by %.3g of its bound" % (
        what, bad.sum(), bad.size, np.max(np.abs(got - want) / (bound + 2.0 ** -126)))


def forward(hip, a, activation, gate=True, pre=True):
    up = {n: hip.create_from_numpy(x) for n, x in a.items()}
    y, h = hip.ones(a["x"].shape), hip.ones(a["x"].shape)
    hip.gated_residual_forward(activation, up["block"], up["gate"] if gate else None, up["x"], up["post"],
                               up["pre"] if pre else None, y, h if pre else None, residual_scale=0.9, epsilon=EPS)
    return y.get(), h.get()


def check_forward(hip, a, activation, gate=True, pre=True):
    y, h = forward(hip, a, activation, gate, pre)
    width = a["x"].shape[1]
    want_y, want_h = ops.gated_residual(activation, a["block"], a["gate"] if gate else None, a["x"], a["post"],
                                        a["pre"] if pre else None, 0.9, EPS)
    n = np.abs(a["post"] * a["block"] * ops.inverse_rms(a["block"], EPS))
    value = np.abs(ops.gate_value(activation, a["gate"])) + 1 if gate else 1.0
    off = c_of(width) * U * (0.9 * np.abs(a["x"]) + value * n)
    close(y, want_y, off, "y")
    if pre:
        r = ops.inverse_rms(want_y, EPS)
        share = np.sqrt((off * off).sum(1, keepdims=True)) / np.maximum(np.sqrt((want_y ** 2).sum(1, keepdims=True)), 1e-30)
        close(h, want_h, np.abs(a["pre"]) * r * (off + np.abs(want_y) * (share + c_of(width) * U)), "h")


def check_backward(hip, a, activation, gate=True, pre=True, accumulate=False):
    up = {n: hip.create_from_numpy(x) for n, x in a.items()}
    rows, width = a["x"].shape
    y = forward(hip, a, activation, gate, pre)[0]
    start = np.full((rows, width), 0.5, F32)
    dblock, dgate, dx = (hip.create_from_numpy(start) for _ in range(3))
    dpost, dpre = hip.ones((width,)), hip.ones((width,))
    hip.gated_residual_backward(activation, up["block"], up["gate"] if gate else None, up["post"],
                                up["pre"] if pre else None, hip.create_from_numpy(y), up["dy"],
                                up["dh"] if pre else None, dblock, dgate if gate else None, dx, dpost,
                                dpre if pre else None, residual_scale=0.9, epsilon=EPS, accumulate=accumulate)
    want = ops.gated_residual_gradients(activation, a["block"], a["gate"] if gate else None, a["post"],
                                        a["pre"] if pre else None, y, a["dy"], a["dh"] if pre else None, 0.9, EPS)
    # the same chain over absolute values
    c = 4 * c_of(width) * U
    block, post = np.abs(a["block"]), np.abs(a["post"])
    rb = ops.inverse_rms(block, EPS)
    total = np.abs(a["dy"]).astype(np.float64)
    if pre:
        ry, ay, e = ops.inverse_rms(y, EPS), np.abs(y), np.abs(a["dh"] * a["pre"])
        total = total + ry * (e + ay * ry * ry * (e * ay).mean(1, keepdims=True))
    value = np.abs(ops.gate_value(activation, a["gate"])) + 1 if gate else np.ones((rows, width))
    d = total * value * post
    extra = 0.5 if accumulate else 0.0
    rounded = lambda w: 2 * U * (np.abs(w) + extra) if accumulate else 0.0
    close(dx.get(), want["dx"] + extra, c * 0.9 * total + rounded(want["dx"]), "dx")
    close(dblock.get(), want["dblock"] + extra,
          c * rb * (d + block * rb * rb * (d * block).mean(1, keepdims=True)) + rounded(want["dblock"]), "dblock")
    close(dpost.get(), want["dpost"], (c + (rows + 8) * U) * (total * value * block * rb).sum(0), "dpost")
    if gate:
        slope = np.abs(ops.gate_slope(activation, a["gate"]))
        close(dgate.get(), want["dgate"] + extra,
              total * post * block * rb * (c * slope + 8 * U * (1 + np.abs(a["gate"]))) + rounded(want["dgate"]), "dgate")
    if pre:
        close(dpre.get(), want["dpre"], (c + (rows + 8) * U) * (np.abs(a["dh"]) * ay * ry).sum(0), "dpre")


SHAPES = [(1, 1), (3, 5), (2, 64), (7, 255), (5, 256), (5, 257), (9, 512), (6, 1000), (4, 1024), (3, 1025), (5, 2048),
          (3, 2050), (4, 4096), (3, 4099), (2, 8192), (3, 8193), (2, 20001), (3000, 33), (700, 1200)]


@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward(hip, rows, width):
    check_forward(hip, inputs(rows + width, rows, width), "swish")


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_backward(hip, rows, width, accumulate):
    check_backward(hip, inputs(rows + width + 1, rows, width), "sigmoid", accumulate=accumulate)


@pytest.mark.parametrize("activation", ["linear", "sigmoid", "tanh", "rel", "el", "swish"])
@pytest.mark.parametrize("width", [30, 1500, 9000])
def test_activations(hip, activation, width):
    a = inputs(5, 4, width)
    a["gate"] *= 4
    check_forward(hip, a, activation)
    check_backward(hip, a, activation)


@pytest.mark.parametrize("width", [30, 1500, 9000])
@pytest.mark.parametrize("gate,pre", [(False, True), (True, False), (False, False)])
def test_parts_can_be_left_out(hip, width, gate, pre):
    a = inputs(6, 5, width)
    check_forward(hip, a, "tanh", gate, pre)
    check_backward(hip, a, "tanh", gate, pre)


@pytest.mark.parametrize("rows,width", [(1, 1), (5, 100), (4, 1024), (3, 3000), (2, 9001)])
def test_the_norm_alone(hip, rows, width):
    a = inputs(7, rows, width)
    x, w, dh = (hip.create_from_numpy(a[n]) for n in ("x", "pre", "dh"))
    out = hip.ones(a["x"].shape)
    hip.rms_norm_forward(x, w, out, epsilon=EPS)
    _, want = ops.gated_residual("linear", None, None, a["x"], None, a["pre"], epsilon=EPS)
    close(out.get(), want, c_of(width) * U * np.abs(want), "norm")
    dx, dw = hip.ones(a["x"].shape), hip.ones((width,))
    hip.rms_norm_backward(x, w, dh, dx, dw, epsilon=EPS)               # adds
    want = ops.gated_residual_gradients("linear", None, None, None, a["pre"], a["x"], None, a["dh"], epsilon=EPS)
    r, ax, e = ops.inverse_rms(a["x"], EPS), np.abs(a["x"]), np.abs(a["dh"] * a["pre"])
    size = r * (e + ax * r * r * (e * ax).mean(1, keepdims=True))
    close(dx.get(), want["dx"] + 1, 4 * c_of(width) * U * (size + 1), "dx")
    close(dw.get(), want["dpre"], (4 * c_of(width) + rows + 8) * U * (np.abs(a["dh"]) * ax * r).sum(0), "dweight")


def test_no_rows(hip):
    none, w = hip.allocate((0, 6)), hip.ones((6,))
    hip.gated_residual_forward("swish", none, none, none, w, w, none, none)
    dpost, dpre = hip.ones((6,)), hip.ones((6,))
    hip.gated_residual_backward("swish", none, none, w, w, none, none, none, none, none, none, dpost, dpre)
    assert not dpost.get().any() and not dpre.get().any()


def test_rows_of_zeros_and_rows_that_are_not_finite(hip):
    a = inputs(8, 6, 300)
    a["block"][1] = a["x"][1] = 0
    clean = forward(hip, a, "swish")
    assert not clean[0][1].any() and not clean[1][1].any()
    a["block"][3, 7] = np.nan
    a["x"][4, 9] = np.inf
    got = forward(hip, a, "swish")
    for x, w in zip(got, clean):
        for row in (0, 1, 2, 5):
            assert_bit_equal(x[row], w[row])
    assert np.isnan(got[0][3]).all() and np.isinf(got[0][4, 9])
    # gates far out: the sigmoid underflows and saturates without a NaN
    a = inputs(9, 2, 64)
    a["gate"][0], a["gate"][1] = -200, 200
    for activation in ("sigmoid", "swish", "tanh", "el"):
        check_forward(hip, a, activation)
        check_backward(hip, a, activation)


@pytest.mark.parametrize("width", [100, 3000, 9000])
def test_outputs_in_the_inputs_places(hip, width):
    a = inputs(10, 5, width)
    y, h = forward(hip, a, "swish")
    up = {n: hip.create_from_numpy(x) for n, x in a.items()}
    hip.gated_residual_forward("swish", up["block"], up["gate"], up["x"], up["post"], up["pre"], up["x"], up["block"],
                               residual_scale=0.9, epsilon=EPS)
    assert_bit_equal(up["x"].get(), y)
    assert_bit_equal(up["block"].get(), h)
    up = {n: hip.create_from_numpy(x) for n, x in a.items()}
    dev = hip.create_from_numpy(y)
    fresh = [hip.ones((5, width)) for _ in range(3)] + [hip.ones((width,)) for _ in range(2)]
    hip.gated_residual_backward("swish", up["block"], up["gate"], up["post"], up["pre"], dev, up["dy"], up["dh"], *fresh,
                                residual_scale=0.9, epsilon=EPS, accumulate=False)
    want = [x.get() for x in fresh]
    hip.gated_residual_backward("swish", up["block"], up["gate"], up["post"], up["pre"], dev, up["dy"], up["dh"],
                                up["dh"], up["gate"], up["dy"], fresh[3], fresh[4], residual_scale=0.9, epsilon=EPS,
                                accumulate=False)
    for x, w in zip((up["dh"], up["gate"], up["dy"], fresh[3], fresh[4]), want):
        assert_bit_equal(x.get(), w)


@pytest.mark.parametrize("rows,width", [(40, 100), (5, 1300), (3, 9001)])
def test_rows_that_start_anywhere(hip, rows, width):
    a = inputs(11, rows, width)
    want = forward(hip, a, "tanh")

    def up(x):
        flat = hip.zeros((x.size + 4,))
        view = flat[1:1 + x.size].reshape(x.shape)
        hip.set_from_numpy(view, x)
        return view, flat

    block, gate, x, post, pre = (up(a[n])[0] for n in ("block", "gate", "x", "post", "pre"))
    (y, y_all), (h, h_all) = up(a["x"] * 0), up(a["x"] * 0)
    hip.gated_residual_forward("tanh", block, gate, x, post, pre, y, h, 0.9, EPS)
    assert_bit_equal(y.get(), want[0])
    assert_bit_equal(h.get(), want[1])
    for flat in (y_all, h_all):                                       # nothing around the rows was written
        got = flat.get()
        assert not got[0] and not got[-3:].any()


def test_the_same_bits_every_time_and_in_a_recording(hip):
    a = inputs(12, 700, 500)
    up = {n: hip.create_from_numpy(x) for n, x in a.items()}
    outs = [hip.ones((700, 500)) for _ in range(5)] + [hip.ones((500,)) for _ in range(2)]
    y, h, dblock, dgate, dx, dpost, dpre = outs

    def run():
        hip.gated_residual_forward("swish", up["block"], up["gate"], up["x"], up["post"], up["pre"], y, h, 0.9, EPS)
        hip.gated_residual_backward("swish", up["block"], up["gate"], up["post"], up["pre"], y, up["dy"], up["dh"],
                                    dblock, dgate, dx, dpost, dpre, 0.9, EPS, accumulate=False)

    run()
    want = [x.get() for x in outs]
    recorded, other = hip.record(run), hip.record(run)
    for step in (recorded, other, recorded):
        for x in outs:
            hip.fill(x, 3.0)
        step.replay()
        for x, w in zip(outs, want):
            assert_bit_equal(x.get(), w)
        run()
        for x, w in zip(outs, want):
            assert_bit_equal(x.get(), w)
    recorded.release()
    other.release()
