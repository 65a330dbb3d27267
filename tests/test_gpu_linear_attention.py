"""GPU: linear attention with a decay, forward, backward and step by step, against the 64-bit recurrence.

Tolerance. Every output is a sum of products w q k v (w a power of the decay, times scale) whose absolute
values add up to what the same formula gives for |q|, |k|, |v|, |decay|. On its way a product meets at most:
the roundings of the dk-deep sum of q.k or of q.S; one addition per position, in the score sum or in the
state; two roundings of powers and products for every chunk of 32 positions that the state passes; and a
fixed number of further products. With n of them and u = 2^-24 the error is at most n u / (1 - n u) times the
sum of absolute values; n = steps + d + 3 (steps / 32 + 1) + 16 counts them generously.
"""
import threading

import numpy as np
import pytest

from brainstorm_amd import _lib
from oracle import sequence_ops as ops
from util import assert_bit_equal

pytestmark = pytest.mark.gpu
F32 = np.float32
U = 2.0 ** -24


def inputs(seed, time, batch, heads, dk, dv, ragged=False):
    rng = np.random.RandomState(seed)
    a = {"q": rng.standard_normal((time, batch, heads * dk)), "k": rng.standard_normal((time, batch, heads * dk)),
         "v": rng.standard_normal((time, batch, heads * dv)), "dout": rng.standard_normal((time, batch, heads * dv)),
         "state": rng.standard_normal((batch, heads, dk, dv)), "dnew": rng.standard_normal((batch, heads, dk, dv)),
         "decay": 1 - 2.0 ** -np.linspace(2, 7, heads)}
    a = {n: x.astype(F32) for n, x in a.items()}
    a["lengths"] = None
    if ragged:
        lengths = rng.randint(0, time + 1, batch).astype(F32)
        lengths[0] = time
        if batch > 1:
            lengths[1] = 0
        a["lengths"] = lengths
    return a


def roundings(time, d):
    n = time + d + 3 * (time // 32 + 1) + 16
    return n * U / (1 - n * U)


def close(got, want, size, rel, what):
    """|got - want| <= rel * size, element by element (plus the smallest normal number for underflow)."""
    bad = ~(np.abs(got.astype(np.float64) - want) <= rel * size + 2.0 ** -126)
    assert not bad.any(), "%s: %d of %d elements off, worst by %.3g of its bound" % (
        what, bad.sum(), bad.size, np.max(np.abs(got - want) / (rel * size + 2.0 ** -126)))


def forward(hip, a, carry, scale=0.3):
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    out = hip.ones(a["v"].shape)
    new = hip.ones(a["state"].shape) if carry else None
    hip.linear_attention_forward(up["q"], up["k"], up["v"], up["decay"], out, scale=scale,
                                 state=up["state"] if carry else None, new_state=new, lengths=up["lengths"])
    return out.get(), new.get() if carry else None


def check_forward(hip, a, carry, scale=0.3):
    got, new = forward(hip, a, carry, scale)
    state = a["state"] if carry else None
    want, want_new = ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], scale, state, a["lengths"])
    size, size_new = ops.linear_attention(*[np.abs(a[n]) for n in ("q", "k", "v", "decay")], abs(scale),
                                          None if state is None else np.abs(state), a["lengths"])
    rel = roundings(a["q"].shape[0], a["state"].shape[2])
    close(got, want, size, rel, "out")
    if carry:
        close(new, want_new, size_new, rel, "new_state")


def backward(hip, a, carry, scale=0.3, with_decay=True):
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    dq, dk, dv = hip.ones(a["q"].shape), hip.ones(a["k"].shape), hip.ones(a["v"].shape)
    ddecay = hip.ones(a["decay"].shape) if with_decay else None
    dstate = hip.ones(a["state"].shape) if carry else None
    hip.linear_attention_backward(up["q"], up["k"], up["v"], up["decay"], up["dout"], dq, dk, dv, ddecay, scale=scale,
                                  state=up["state"] if carry else None, dnew_state=up["dnew"] if carry else None,
                                  dstate=dstate, lengths=up["lengths"])
    return [x.get() if x is not None else None for x in (dq, dk, dv, ddecay, dstate)]


def check_backward(hip, a, carry, scale=0.3, with_decay=True):
    got = backward(hip, a, carry, scale, with_decay)
    state, dnew = (a["state"], a["dnew"]) if carry else (None, None)
    want = ops.linear_attention_gradients(a["q"], a["k"], a["v"], a["decay"], a["dout"], scale, state, dnew, a["lengths"])
    m = {n: None if x is None else np.abs(x) for n, x in a.items()}
    size = ops.linear_attention_gradients(m["q"], m["k"], m["v"], m["decay"], m["dout"], abs(scale),
                                          m["state"] if carry else None, m["dnew"] if carry else None, a["lengths"])
    time, dk, dv = a["q"].shape[0], a["state"].shape[2], a["state"].shape[3]
    for x, w, s, name in zip(got, want, size, ("dq", "dk", "dv", "ddecay", "dstate")):
        if x is None:
            continue
        # the decay's gradient: a product of a derivative of the state (twice the roundings) with q and its sum
        rel = roundings(2 * time, dk + dv) if name == "ddecay" else roundings(time, max(dk, dv))
        close(x, w, s, rel, name)


SHAPES = [(1, 1, 1, 1, 1), (2, 3, 2, 4, 4), (4, 2, 3, 17, 5), (5, 2, 2, 16, 16), (31, 2, 2, 8, 3), (32, 1, 4, 32, 64),
          (33, 3, 1, 33, 65), (64, 2, 3, 40, 72), (100, 3, 2, 125, 125), (65, 1, 2, 128, 128), (97, 2, 1, 128, 1),
          (130, 1, 1, 1, 128), (300, 2, 2, 64, 64), (777, 1, 2, 20, 36)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("carry,ragged", [(False, False), (True, False), (True, True)])
def test_forward(hip, shape, carry, ragged):
    check_forward(hip, inputs(sum(shape), *shape, ragged=ragged), carry)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("carry,ragged", [(False, False), (True, True), (False, True)])
def test_backward(hip, shape, carry, ragged):
    check_backward(hip, inputs(sum(shape) + 1, *shape, ragged=ragged), carry)


def test_backward_without_the_decays_gradient(hip):
    a = inputs(5, 200, 2, 2, 24, 40)
    with_it, without = backward(hip, a, True), backward(hip, a, True, with_decay=False)
    for n in (0, 1, 2, 4):
        assert_bit_equal(without[n], with_it[n])


@pytest.mark.parametrize("decay", [[0.0, 1.0], [-0.5, 1.01], [1e-20, 0.999]])
def test_decays_at_and_beyond_the_ends(hip, decay):
    a = inputs(6, 90, 2, 2, 12, 20, ragged=True)
    a["decay"] = np.array(decay, F32)
    check_forward(hip, a, True)
    check_backward(hip, a, True)


def test_zero_steps_and_zero_sequences(hip):
    a = inputs(7, 3, 2, 2, 4, 5)
    up = {n: hip.create_from_numpy(a[n]) for n in ("state", "decay", "dnew")}
    none = [hip.allocate((0, 2, 8)), hip.allocate((0, 2, 8)), hip.allocate((0, 2, 10))]
    new = hip.ones(a["state"].shape)
    hip.linear_attention_forward(*none, up["decay"], hip.allocate((0, 2, 10)), state=up["state"], new_state=new)
    assert_bit_equal(new.get(), a["state"])
    hip.linear_attention_forward(*none, up["decay"], hip.allocate((0, 2, 10)), new_state=new)
    assert_bit_equal(new.get(), np.zeros(a["state"].shape))
    dstate, ddecay = hip.ones(a["state"].shape), hip.ones((2,))
    hip.linear_attention_backward(*none, up["decay"], hip.allocate((0, 2, 10)), *none, ddecay=ddecay,
                                  dnew_state=up["dnew"], dstate=dstate)
    assert_bit_equal(dstate.get(), a["dnew"])
    assert_bit_equal(ddecay.get(), np.zeros(2))
    empty = [hip.allocate((3, 0, 8)), hip.allocate((3, 0, 8)), hip.allocate((3, 0, 10))]
    ddecay = hip.ones((2,))
    hip.linear_attention_forward(*empty, up["decay"], hip.allocate((3, 0, 10)))
    hip.linear_attention_backward(*empty, up["decay"], hip.allocate((3, 0, 10)), *empty, ddecay=ddecay)
    assert_bit_equal(ddecay.get(), np.zeros(2))


@pytest.mark.parametrize("time", [3, 70, 500])
def test_padding_is_not_read_and_gets_zeros(hip, time):
    a = inputs(8, time, 4, 2, 20, 12)
    a["lengths"] = np.array([time, 0, time // 2 + 0.9, np.nan], F32)
    lengths = ops.sequence_lengths(a["lengths"], time, 4)
    assert list(lengths) == [time, 0, time // 2, 0]
    clean_out, clean_new = forward(hip, a, True)
    clean = backward(hip, a, True)
    for b, n in enumerate(lengths):
        for name in ("q", "k", "v", "dout"):
            a[name][n:, b] = np.nan if b % 2 else np.inf
    out, new = forward(hip, a, True)
    assert_bit_equal(out, clean_out)
    assert_bit_equal(new, clean_new)
    for x, y in zip(backward(hip, a, True), clean):
        assert_bit_equal(x, y)
    for b, n in enumerate(lengths):
        for x in (out, clean[0], clean[1], clean[2]):
            assert not x[n:, b].any()
    assert_bit_equal(new[1], a["state"][1])
    assert_bit_equal(clean[4][3], a["dnew"][3])


@pytest.mark.parametrize("time,at", [(3, 1), (40, 5), (40, 20), (200, 77)])
@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_values_that_are_not_finite_stay_behind_their_position(hip, time, at, name):
    a = inputs(9, time, 2, 2, 20, 24)
    clean, _ = forward(hip, a, True)
    a[name][at, 0, 3] = np.nan
    a[name][at + 1, 0, 5] = np.inf
    out, _ = forward(hip, a, True)
    first, second = (slice(0, 24), slice(24, 48))                        # features 3 and 5 belong to the first head
    assert_bit_equal(out[:at], clean[:at])
    assert_bit_equal(out[:, 1], clean[:, 1])
    assert_bit_equal(out[:, 0, second], clean[:, 0, second])
    want, _ = ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], 0.3, a["state"])
    assert (np.isfinite(out) == np.isfinite(want)).all() or name != "q"
    assert not np.isfinite(out[at, 0, first]).all()


def test_gradients_of_values_that_are_not_finite_stay_before_their_position(hip):
    a = inputs(10, 100, 1, 1, 16, 16)
    clean = backward(hip, a, False)
    a["dout"][50, 0, 3] = np.nan
    got = backward(hip, a, False)
    assert_bit_equal(got[0][:50], clean[0][:50])                         # dq looks back
    for n in (1, 2):                                                     # dk and dv look ahead
        assert_bit_equal(got[n][51:], clean[n][51:])
        assert not np.isfinite(got[n][50]).all()


@pytest.mark.parametrize("batch,heads,dk,dv", [(1, 8, 64, 64), (3, 2, 17, 5), (300, 4, 128, 128), (70, 5, 128, 100),
                                               (2, 1, 1, 1)])
def test_steps_are_the_sequence(hip, batch, heads, dk, dv):
    a = inputs(11, 6, batch, heads, dk, dv)
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    out = hip.ones(a["v"].shape)
    for t in range(6):
        hip.linear_attention_step(up["q"][t], up["k"][t], up["v"][t], up["decay"], up["state"], out[t], scale=0.3)
    want, want_new = ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], 0.3, a["state"])
    size, size_new = ops.linear_attention(*[np.abs(a[n]) for n in ("q", "k", "v", "decay")], 0.3, np.abs(a["state"]))
    close(out.get(), want, size, roundings(6, dk), "out")
    close(up["state"].get(), want_new, size_new, roundings(6, dk), "state")


def test_a_sequence_in_pieces_is_the_sequence(hip):
    a = inputs(12, 150, 2, 3, 24, 20)
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    out = hip.ones(a["v"].shape)
    for first, last in ((0, 64), (64, 67), (67, 68), (68, 150)):
        hip.linear_attention_forward(up["q"][first:last], up["k"][first:last], up["v"][first:last], up["decay"],
                                     out[first:last], scale=0.3, state=up["state"], new_state=up["state"])
    want, want_new = ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], 0.3, a["state"])
    size, size_new = ops.linear_attention(*[np.abs(a[n]) for n in ("q", "k", "v", "decay")], 0.3, np.abs(a["state"]))
    close(out.get(), want, size, roundings(150, 24), "out")
    close(up["state"].get(), want_new, size_new, roundings(150, 24), "state")


def test_gradient_of_the_state_in_place(hip):
    a = inputs(13, 40, 2, 2, 10, 12)
    want = backward(hip, a, True)[4]
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    dq, dk, dv = hip.empty(a["q"].shape), hip.empty(a["k"].shape), hip.empty(a["v"].shape)
    hip.linear_attention_backward(up["q"], up["k"], up["v"], up["decay"], up["dout"], dq, dk, dv, scale=0.3,
                                  state=up["state"], dnew_state=up["dnew"], dstate=up["dnew"])
    assert_bit_equal(up["dnew"].get(), want)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_arrays_that_start_anywhere(hip, shift):
    a = inputs(14, 70, 2, 2, 20, 28)
    want, want_new = forward(hip, a, True)
    want_back = backward(hip, a, True)

    whole = []

    def up(x):
        flat = hip.zeros((x.size + 8,))
        hip.fill(flat, 3.0)
        view = flat[shift:shift + x.size].reshape(x.shape)
        hip.set_from_numpy(view, x)
        whole.append((flat, x.size))
        return view

    q, k, v, decay, state, dout, dnew = (up(a[n]) for n in ("q", "k", "v", "decay", "state", "dout", "dnew"))
    out, new, dq, dk, dv, ddecay, dstate = (up(np.ones_like(x)) for x in (a["v"], a["state"], a["q"], a["k"], a["v"],
                                                                         a["decay"], a["state"]))
    hip.linear_attention_forward(q, k, v, decay, out, 0.3, state, new)
    hip.linear_attention_backward(q, k, v, decay, dout, dq, dk, dv, ddecay, 0.3, state, dnew, dstate)
    assert_bit_equal(out.get(), want)
    assert_bit_equal(new.get(), want_new)
    for x, w in zip((dq, dk, dv, ddecay, dstate), want_back):
        assert_bit_equal(x.get(), w)
    for flat, size in whole:                                       # nothing around the arrays was written
        around = flat.get()
        assert (around[:shift] == 3).all() and (around[shift + size:] == 3).all()


def test_the_same_bits_every_time_and_in_a_recording(hip):
    a = inputs(15, 300, 2, 2, 40, 24, ragged=True)
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    out, new = hip.ones(a["v"].shape), hip.ones(a["state"].shape)
    grads = [hip.ones(a[n].shape) for n in ("q", "k", "v", "decay", "state")]

    def run():
        hip.linear_attention_forward(up["q"], up["k"], up["v"], up["decay"], out, 0.3, up["state"], new, up["lengths"])
        hip.linear_attention_backward(up["q"], up["k"], up["v"], up["decay"], up["dout"], *grads[:4], 0.3, up["state"],
                                      up["dnew"], grads[4], up["lengths"])

    run()
    want = [x.get() for x in [out, new] + grads]
    first, second = hip.record(run), hip.record(run)
    for step in (first, second, first, first, second):
        for x in [out, new] + grads:
            hip.fill(x, 7.0)
        step.replay()
        for x, w in zip([out, new] + grads, want):
            assert_bit_equal(x.get(), w)
        run()
        for x, w in zip([out, new] + grads, want):
            assert_bit_equal(x.get(), w)
    first.release()
    second.release()


def test_threads_share_the_library(hip):
    a = [inputs(16 + n, 130, 2, 2, 16 + 4 * n, 20) for n in range(3)]
    want = [(forward(hip, x, True), backward(hip, x, True)) for x in a]
    wrong = []

    def work(n):
        for _ in range(5):
            got = (forward(hip, a[n], True), backward(hip, a[n], True))
            for x, w in zip(got[0] + tuple(got[1]), want[n][0] + tuple(want[n][1])):
                if not np.array_equal(x, w):
                    wrong.append(n)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_row_pitched_views(hip):
    from brainstorm_amd import HipHandler
    pitched = HipHandler(seed=3, pitched_views=True)
    a = inputs(20, 40, 2, 2, 8, 8)
    hub = pitched.create_from_numpy(np.concatenate([a["q"], a["k"], a["v"]], 2))
    wide = pitched.zeros((40, 2, 40))
    state = pitched.create_from_numpy(a["state"])
    pitched.linear_attention_forward(hub[:, :, :16], hub[:, :, 16:32], hub[:, :, 32:], pitched.create_from_numpy(a["decay"]),
                                     wide[:, :, 3:19], 0.3, state, state)
    want, want_new = forward(hip, a, True)
    got = wide.get()
    assert_bit_equal(got[:, :, 3:19], want)
    assert not got[:, :, :3].any() and not got[:, :, 19:].any()
    assert_bit_equal(state.get(), want_new)
    hip.set_fusing(True)


# Short sequences without states, where all scores are formed: every width of the kernels, both lengths of the gradients',
# and sizes on both sides of the rules that choose them.
SHORT = [(5, 3, 2, 4, 4), (16, 2, 3, 30, 32), (17, 2, 2, 24, 60), (33, 2, 2, 31, 100), (48, 2, 2, 64, 20), (64, 3, 1, 50, 64),
         (64, 2, 2, 36, 125), (63, 2, 2, 128, 31), (65, 2, 2, 100, 33), (90, 2, 2, 33, 60), (96, 2, 2, 64, 64),
         (97, 2, 2, 60, 64), (100, 2, 2, 24, 20), (112, 2, 1, 127, 126), (128, 2, 2, 128, 128), (128, 3, 2, 40, 7),
         (129, 2, 1, 128, 128)]


@pytest.mark.parametrize("shape", SHORT)
@pytest.mark.parametrize("ragged", [False, True])
def test_short_sequences_without_states(hip, shape, ragged):
    a = inputs(sum(shape) + 30, *shape, ragged=ragged)
    check_forward(hip, a, False)
    check_backward(hip, a, False)


def test_many_short_sequences(hip):
    a = inputs(31, 9, 700, 3, 12, 16, ragged=True)
    check_forward(hip, a, False)
    check_backward(hip, a, False)


@pytest.mark.parametrize("decay", [[0.0, 1.0], [-0.5, 1.01], [1e-20, 0.999]])
def test_decays_at_the_ends_without_states(hip, decay):
    a = inputs(32, 70, 2, 2, 40, 48, ragged=True)
    a["decay"] = np.array(decay, F32)
    check_forward(hip, a, False)
    check_backward(hip, a, False)


@pytest.mark.parametrize("time,at", [(40, 5), (100, 20), (128, 99)])
@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_values_that_are_not_finite_without_states(hip, time, at, name):
    a = inputs(33, time, 2, 2, 120, 124)
    clean, _ = forward(hip, a, False)
    a[name][at, 0, 3] = np.nan
    a[name][at + 1, 0, 5] = np.inf
    out, _ = forward(hip, a, False)
    first, second = (slice(0, 124), slice(124, 248))
    assert_bit_equal(out[:at], clean[:at])
    assert_bit_equal(out[:, 1], clean[:, 1])
    assert_bit_equal(out[:, 0, second], clean[:, 0, second])
    assert not np.isfinite(out[at, 0, first]).all()
    if name == "q":                                                      # a query is its own position's alone
        assert_bit_equal(out[at + 2:], clean[at + 2:])
    if name == "v":                                                      # and a value its own column's
        rest = np.ones(248, bool)
        rest[[3, 5]] = False
        assert_bit_equal(out[:, :, rest], clean[:, :, rest])
        assert np.isnan(out[at:, 0, 3]).all() and not np.isfinite(out[at + 1:, 0, 5]).any()


@pytest.mark.parametrize("time,at,d", [(40, 5, 16), (64, 33, 60), (100, 50, 128), (128, 99, 40)])
@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
def test_gradients_that_are_not_finite_without_states(hip, time, at, d, name):
    a = inputs(34, time, 1, 2, d, d)
    clean = backward(hip, a, False)
    a[name][at, 0, 3] = np.nan
    got = backward(hip, a, False)
    for n in range(3):                                                   # the other head
        assert_bit_equal(got[n][:, :, d:], clean[n][:, :, d:])
    if name in ("q", "dout"):                                            # seen by itself and the keys up to it
        assert_bit_equal(got[0][:at], clean[0][:at])
        assert_bit_equal(got[0][at + 1:], clean[0][at + 1:])
        for n in (1, 2):
            assert_bit_equal(got[n][at + 1:], clean[n][at + 1:])
        assert not np.isfinite(got[1][at]).all() and not np.isfinite(got[2][at]).all()
    else:                                                                # by itself and the queries from it on
        assert_bit_equal(got[0][:at], clean[0][:at])
        assert not np.isfinite(got[0][at]).all()
        for n in (1, 2):
            assert_bit_equal(got[n][:at], clean[n][:at])
            assert_bit_equal(got[n][at + 1:], clean[n][at + 1:])


@pytest.mark.parametrize("time", [20, 100])
def test_padding_without_states(hip, time):
    a = inputs(35, time, 4, 2, 36, 40)
    a["lengths"] = np.array([time, 0, time // 2 + 0.9, np.nan], F32)
    lengths = ops.sequence_lengths(a["lengths"], time, 4)
    clean_out, _ = forward(hip, a, False)
    clean = backward(hip, a, False)
    for b, n in enumerate(lengths):
        for name in ("q", "k", "v", "dout"):
            a[name][n:, b] = np.nan if b % 2 else np.inf
    assert_bit_equal(forward(hip, a, False)[0], clean_out)
    for x, y in zip(backward(hip, a, False)[:4], clean):
        assert_bit_equal(x, y)
    for b, n in enumerate(lengths):
        for x in (clean_out, clean[0], clean[1], clean[2]):
            assert not x[n:, b].any()


@pytest.mark.parametrize("shape", [(30, 2, 2, 21, 23), (100, 2, 2, 125, 125)])
def test_short_sequences_anywhere_and_recorded(hip, shape):
    a = inputs(36, *shape)
    want_out, _ = forward(hip, a, False)
    want = [want_out] + backward(hip, a, False)[:4]
    whole = []

    def up(x, shift):
        flat = hip.zeros((x.size + 8,))
        hip.fill(flat, 3.0)
        hip.set_from_numpy(flat[shift:shift + x.size].reshape(x.shape), x)
        whole.append((flat, shift, x.size))
        return flat[shift:shift + x.size].reshape(x.shape)

    q, k, v, dout, decay = (up(a[n], 1 + i % 3) for i, n in enumerate(("q", "k", "v", "dout", "decay")))
    results = [up(np.ones_like(w), 3 - i % 3) for i, w in enumerate(want)]

    def run():
        hip.linear_attention_forward(q, k, v, decay, results[0], 0.3)
        hip.linear_attention_backward(q, k, v, decay, dout, *results[1:], scale=0.3)

    run()
    first, second = hip.record(run), hip.record(run)
    for step in (None, first, second, first):
        if step is not None:
            for x in results:
                hip.fill(x, 7.0)
            step.replay()
        for x, w in zip(results, want):
            assert_bit_equal(x.get(), w)
        run()
        for flat, shift, size in whole:
            around = flat.get()
            assert (around[:shift] == 3).all() and (around[shift + size:] == 3).all()
    first.release()
    second.release()


def test_more_features_than_a_pass_reaches(hip):
    # 2^25 + 1024 features in a step: refused for 4 steps, computed position by position for 3
    batch = 2 ** 15 + 1
    x, out = hip.zeros((4, batch, 1024)), hip.ones((4, batch, 1024))
    decay = hip.ones((8,))
    with pytest.raises(_lib.BshipError, match="features in a time step"):
        hip.linear_attention_forward(x, x, x, decay, out)
    assert (out[3][batch - 1].get() == 1).all()
    hip.fill(x, 1.0)
    hip.linear_attention_forward(x[:3], x[:3], x[:3], decay, out[:3])
    for t in range(3):
        for b in (0, batch - 1):
            assert_bit_equal(out[t][b].get(), np.full(1024, 128.0 * (t + 1), F32))


# Longer sequences by their number: columns in two parts (half of the compute units' number of sequences, or too few positions
# to cut), segments, neither.
@pytest.mark.parametrize("shape", [(200, 16, 8, 16, 80), (150, 33, 4, 20, 128), (300, 2, 2, 128, 100), (140, 40, 8, 8, 16),
                                   (700, 9, 8, 24, 72), (160, 64, 4, 12, 70)])
@pytest.mark.parametrize("ragged", [False, True])
def test_numbers_of_sequences(hip, shape, ragged):
    a = inputs(sum(shape) + 40, *shape, ragged=ragged)
    check_forward(hip, a, True)
    check_backward(hip, a, True)


@pytest.mark.parametrize("shape", [(100, 3, 2, 20, 24), (150, 10, 8, 64, 64), (300, 9, 8, 16, 128), (700, 2, 2, 33, 70)])
def test_a_state_replaced_by_several_segments(hip, shape):
    # 2 to 11 segments; every one of them starts from the state that the last one replaces
    a = inputs(sum(shape) + 50, *shape)
    up = {n: (None if x is None else hip.create_from_numpy(x)) for n, x in a.items()}
    out, grads = hip.ones(a["v"].shape), [hip.ones(a[n].shape) for n in ("q", "k", "v")]
    hip.linear_attention_backward(up["q"], up["k"], up["v"], up["decay"], up["dout"], *grads, scale=0.3, state=up["state"],
                                  dnew_state=up["dnew"], dstate=up["dnew"])
    hip.linear_attention_forward(up["q"], up["k"], up["v"], up["decay"], out, 0.3, up["state"], up["state"])
    time, dk, dv = shape[0], shape[3], shape[4]
    m = {n: np.abs(a[n]) for n in ("q", "k", "v", "decay", "dout", "state", "dnew")}
    want, size = (ops.linear_attention(x["q"], x["k"], x["v"], x["decay"], 0.3, x["state"]) for x in (a, m))
    for x, w, s, name in zip((out, up["state"]), want, size, ("out", "new_state")):
        close(x.get(), w, s, roundings(time, dk), name)
    want, size = (ops.linear_attention_gradients(x["q"], x["k"], x["v"], x["decay"], x["dout"], 0.3, x["state"], x["dnew"])
                  for x in (a, m))
    for n, (x, name) in enumerate(zip(grads + [up["dnew"]], ("dq", "dk", "dv", "dstate"))):
        n = 4 if name == "dstate" else n
        close(x.get(), want[n], size[n], roundings(time, max(dk, dv)), name)


@pytest.mark.parametrize("time", [2, 40, 300])
def test_an_empty_sequence_adds_nothing_to_the_gradient_of_the_decay(hip, time):
    # its new state is its state, whatever the decay: also where the gradient from behind is not finite
    a = inputs(63, time, 3, 2, 12, 16)
    a["lengths"] = np.array([time, 0, time // 2], F32)
    clean = backward(hip, a, True)
    a["dnew"][1, 0, 3, 4], a["dnew"][1, 1, 5, 6] = np.inf, np.nan
    got = backward(hip, a, True)
    for n in range(4):
        assert_bit_equal(got[n], clean[n])
    assert_bit_equal(got[4], np.stack([clean[4][0], a["dnew"][1], clean[4][2]]))


def kinds(x):
    """0 for finite elements, 1, -1 and 2 for infinities and NaN."""
    return np.where(np.isnan(x), 2, np.where(np.isfinite(x), 0, np.sign(x)))


@pytest.mark.parametrize("time,lengths", [(3, None), (20, None), (33, None), (64, (64, 40)), (100, (0, 100)), (300, (299, 65)),
                                          (700, None), (700, (64, 130))])
@pytest.mark.parametrize("decay", [[0.9, 1.0], [-0.5, 0.3], [0.07, -0.9], [1e-3, -1e-20]])
def test_infinite_states_stay_infinite(hip, time, lengths, decay):
    # infinities on their own in their rows and columns: sums with them are infinities of one sign, and so is what the
    # recurrence makes of them; one sequence has a NaN as well
    a = inputs(60, time, 2, 2, 20, 24)
    a["decay"] = np.array(decay, F32)
    a["lengths"] = None if lengths is None else np.array(lengths, F32)
    for name in ("state", "dnew"):
        a[name][0, 0, 3, 5], a[name][0, 1, 4, 6], a[name][1, 1, 7, 8] = np.inf, -np.inf, np.inf
        a[name][1, 1, 9, 2] = np.nan
    with np.errstate(invalid="ignore"):
        want = list(ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], 0.3, a["state"], a["lengths"]))
        back = ops.linear_attention_gradients(a["q"], a["k"], a["v"], a["decay"], a["dout"], 0.3, a["state"], a["dnew"],
                                              a["lengths"])
    got = list(forward(hip, a, True)) + backward(hip, a, True)
    want += list(back)
    for x, w, name in zip(got, want, ("out", "new_state", "dq", "dk", "dv", "ddecay", "dstate")):
        if name == "ddecay":                          # infinities of both signs meet in its sum
            assert (np.isfinite(x) == np.isfinite(w)).all()
        else:
            assert (kinds(x) == kinds(w)).all(), "%s: %d elements" % (name, (kinds(x) != kinds(w)).sum())


def test_infinite_states_behind_decays_that_have_vanished(hip):
    # 0.5 to the power of a segment's steps is 0 in float32 and, over all segments, in float64; 0.01 to that of a chunk's
    for time, decay in ((300, 0.5), (1200, 0.5), (8000, 0.5), (70, 0.01), (700, -0.01)):
        a = inputs(61, time, 1, 1, 16, 64)
        a["decay"][:] = decay
        a["state"][0, 0, 3, 5] = np.inf
        want, want_new = ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], 0.3, a["state"])
        out, new = forward(hip, a, True)
        assert (kinds(out) == kinds(want)).all() and (kinds(new) == kinds(want_new)).all()
        assert np.isinf(new[0, 0, 3, 5])


@pytest.mark.parametrize("time,at", [(3, 1), (40, 5), (40, 20), (128, 99), (200, 77), (600, 300)])
@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("carry", [False, True])
def test_exactly_the_positions_that_see_a_value_are_not_finite(hip, time, at, name, carry):
    a = inputs(62, time, 2, 2, 20, 24)
    a[name][at, 0, 3] = np.nan
    a[name][at + 1, 0, 5] = np.inf
    with np.errstate(invalid="ignore"):
        want, want_new = ops.linear_attention(a["q"], a["k"], a["v"], a["decay"], 0.3, a["state"] if carry else None)
    out, new = forward(hip, a, carry)
    assert (np.isfinite(out) == np.isfinite(want)).all() and not np.isfinite(out).all()
    if carry:
        assert (np.isfinite(new) == np.isfinite(want_new)).all()


def test_a_long_memory_loses_no_more_than_one_rounding_a_chunk(hip):
    # A state that remembers 4096 positions, formed in one piece. Every 32 positions it is multiplied and added to with one
    # rounding of its own size; what is added is a sum of 32 products with random signs, whose additions round against partial
    # sums of half its square in the mean, and two roundings of each product. A rounding's square is at most u^2 / 3 in the mean, what
    # is added makes up the state's square, and an old error fades with the state: the relative square of the error is at most
    # u^2 / 3 (sum over chunks of g^(2 32 c) + 32 / 2 + 2 + 2), the last 2 for the decay's powers.
    time, batch, heads, d = 4096, 40, 8, 16
    rng = np.random.RandomState(70)
    q, k, v = (rng.standard_normal((time, batch, heads * d)).astype(F32) for _ in range(3))
    decay = np.full(heads, 1 - 2.0 ** -12, F32)
    up = [hip.create_from_numpy(x) for x in (q, k, v, decay)]
    new = hip.ones((batch, heads, d, d))
    hip.linear_attention_forward(*up, hip.empty(v.shape), new_state=new)
    want = np.zeros((batch, heads, d, d))
    kf, vf = (x.reshape(time, batch, heads, d).astype(np.float64) for x in (k, v))
    for t in range(time):
        want = float(decay[0]) * want + kf[t, :, :, :, None] * vf[t, :, :, None, :]
    passed = (float(decay[0]) ** (64.0 * np.arange(time // 32))).sum()
    off = np.linalg.norm(new.get() - want) / np.linalg.norm(want)
    assert off <= U * np.sqrt((passed + 20) / 3)


@pytest.mark.parametrize("shape,decay", [((100, 2, 2, 20, 24), [1.9, -1.5]), ((100, 2, 2, 100, 60), [-1.9, 1.2]),
                                         ((40, 2, 2, 8, 8), [3.0, -6.0]), ((300, 2, 2, 20, 72), [1.25, -1.2]),
                                         ((3, 2, 2, 8, 8), [1e6, -1e12])])
@pytest.mark.parametrize("carry", [False, True])
def test_decays_that_grow(hip, shape, decay, carry):
    # as far as float32 holds the number of steps times the power of the decay
    a = inputs(sum(shape) + 80, *shape)
    a["decay"] = np.array(decay, F32)
    check_forward(hip, a, carry)
    check_backward(hip, a, carry)
