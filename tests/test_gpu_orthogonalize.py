"""GPU: Newton-Schulz orthogonalisation and the momentum update built on it, against 64 bits.

Tolerance, in the Frobenius norm relative to the result's. A product's entry is a sum over k of products whose
relative errors are at most 3 2^-23 (two factors kept to 23 bits, lo lo left out) with independent signs, and of
float32 additions: its error is of size 2^-22 sqrt(sum p_ik^2 x_kj^2), so |error of pX| is about 2^-22 |p|_F |X|_2 <=
2^-22 3.45 1.21 sqrt(m), and the errors of A and p add about 2^-22 (1.45 4.78 + 2.1 2.03 2) 1.21 sqrt(m): together below
24 2^-22 sqrt(m) for one step, against |X|_F >= 0.68 sqrt(m) after the last. A step multiplies what earlier steps left
by the polynomial's slope, at most 1.63 on [0.55, 1.13] where the large singular values are from the second step
on and 3.45 below, where an error grows no faster than the value that has it. Summed: 24 2^-22 (1 + 1.63 + ... +
1.63^4) / 0.68 = 1.4e-4 for five steps. What is not computed as described is off by far more: bfloat16-sized
factors by 4e-3, a lost low plane by 5e-4.
"""
import numpy as np
import pytest

from oracle import sequence_ops as ops
from util import assert_bit_equal

pytestmark = pytest.mark.gpu
F32 = np.float32
REL = 1.4e-4

SHAPES = [(1, 1), (1, 7), (9, 1), (3, 5), (16, 16), (10, 1200), (64, 64), (65, 63), (128, 128), (129, 300), (300, 129),
          (205, 1000), (784, 1200), (513, 512), (1000, 1000)]


def matrix(seed, *shape):
    rng = np.random.RandomState(seed)
    return (1e-3 * rng.standard_normal(shape)).astype(F32)


def off(got, want):
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize(hip, rows, cols):
    m = matrix(rows * 7 + cols, rows, cols)
    out = hip.ones((rows, cols))
    hip.orthogonalize(hip.create_from_numpy(m), out)
    assert off(out.get(), ops.orthogonalize(m)) <= REL


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_other_numbers_of_steps(hip, steps):
    m = matrix(3, 40, 70)
    out = hip.ones(m.shape)
    hip.orthogonalize(hip.create_from_numpy(m), out, steps=steps)
    assert off(out.get(), ops.orthogonalize(m, steps)) <= REL * max(1.0, 1.63 ** (steps - 5))


@pytest.mark.parametrize("shape", [(4, 30, 50), (3, 140, 60), (2, 256, 384), (0, 4, 5), (2, 0, 5), (2, 5, 0)])
def test_stacks(hip, shape):
    m = matrix(4, *shape)
    out = hip.ones(shape)
    hip.orthogonalize(hip.create_from_numpy(m), out)
    got = out.get()
    for one, x in zip(got, m):
        if x.size:
            assert off(one, ops.orthogonalize(x)) <= REL
            alone = hip.ones(x.shape)
            hip.orthogonalize(hip.create_from_numpy(x), alone)
            assert off(alone.get(), one.astype(np.float64)) <= REL


@pytest.mark.parametrize("scale", [1e-30, 1e-38, 1e20, 1e37])
def test_any_magnitude(hip, scale):
    m = (matrix(5, 33, 47) * 1e3 * scale).astype(F32)
    out = hip.ones(m.shape)
    hip.orthogonalize(hip.create_from_numpy(m), out)
    assert off(out.get(), ops.orthogonalize(m)) <= REL


def test_low_rank_and_uneven_matrices(hip):
    rng = np.random.RandomState(6)
    low = (rng.standard_normal((200, 3)) @ rng.standard_normal((3, 150))).astype(F32)
    one = np.zeros((130, 70), F32)
    one[100, 5] = -3.0
    spiked = matrix(7, 100, 260)
    spiked[3] *= 1e4
    for m in (low, one, spiked):
        out = hip.ones(m.shape)
        hip.orthogonalize(hip.create_from_numpy(m), out)
        want = ops.orthogonalize(m)
        # singular values that are zero but for the input's rounding grow by up to 3.45 a step, and so does
        # what the float32 input's own rounding puts there
        assert off(out.get(), want) <= REL


def test_zeros_and_values_that_are_not_finite(hip):
    m = matrix(8, 3, 40, 50)
    m[0] = 0
    m[1, 3, 4] = np.nan
    out = hip.ones(m.shape)
    hip.orthogonalize(hip.create_from_numpy(m), out)
    got = out.get()
    assert not got[0].any()
    assert np.isnan(got[1]).all()
    assert off(got[2], ops.orthogonalize(m[2])) <= REL
    m[1, 3, 4] = np.inf
    hip.orthogonalize(hip.create_from_numpy(m), out)
    assert np.isnan(out.get()[1]).all()


def test_in_place(hip):
    m = matrix(9, 70, 40)
    a, out = hip.create_from_numpy(m), hip.ones(m.shape)
    hip.orthogonalize(a, out)
    hip.orthogonalize(a, a)
    assert_bit_equal(a.get(), out.get())


@pytest.mark.parametrize("shape", [(12, 20), (200, 30), (3, 64, 65), (1000, 205), (1, 7, 300)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update(hip, shape, nesterov):
    rng = np.random.RandomState(10)
    g, v, p = matrix(11, *shape), matrix(12, *shape), rng.standard_normal(shape).astype(F32)
    dg, dv, dp = (hip.create_from_numpy(x) for x in (g, v, p))
    hip.orthogonal_update(0.9, -0.5, dg, dv, dp, nesterov=nesterov)
    want_v, want_p = ops.orthogonal_update(F32(0.9), -0.5, g, v, p, nesterov=nesterov)
    # the velocity as the handler's own operations form it: two roundings
    assert_bit_equal(dv.get(), (F32(0.9) * v) + g)
    moved = np.linalg.norm(want_p - p)
    assert np.linalg.norm(dp.get() - want_p) <= REL * moved + 2.0 ** -23 * np.linalg.norm(np.abs(p) + np.abs(want_p))
    assert_bit_equal(dg.get(), g)


def test_views_that_start_anywhere_keep_what_is_around_them(hip):
    m = matrix(13, 33, 41)
    flat = hip.zeros((m.size + 8,))
    view = flat[3:3 + m.size].reshape(m.shape)
    hip.set_from_numpy(view, m)
    out, around = hip.ones(m.shape), hip.zeros((m.size + 8,))
    hip.orthogonalize(hip.create_from_numpy(m), out)
    hip.orthogonalize(view, around[1:1 + m.size].reshape(m.shape))
    got = around.get()
    assert_bit_equal(got[1:1 + m.size].reshape(m.shape), out.get())
    assert not got[0] and not got[1 + m.size:].any()


def test_the_same_bits_every_time_and_in_a_recording(hip):
    m = matrix(14, 2, 150, 130)
    a, out = hip.create_from_numpy(m), hip.ones(m.shape)
    v, p = hip.zeros(m.shape), hip.zeros(m.shape)

    def run():
        hip.orthogonalize(a, out)
        hip.fill(v, 0.25)
        hip.fill(p, 1.0)
        hip.orthogonal_update(0.9, -0.1, a, v, p)

    run()
    want = [x.get() for x in (out, v, p)]
    first, second = hip.record(run), hip.record(run)
    for step in (first, second, first):
        for x in (out, v, p):
            hip.fill(x, 3.0)
        step.replay()
        for x, w in zip((out, v, p), want):
            assert_bit_equal(x.get(), w)
        run()
        for x, w in zip((out, v, p), want):
            assert_bit_equal(x.get(), w)
    first.release()
    second.release()


def test_steps_out_of_range_are_refused(hip):
    m = hip.ones((4, 4))
    for steps in (0, -1, 101):
        with pytest.raises(RuntimeError, match="steps"):
            hip.orthogonalize(m, m, steps=steps)


@pytest.mark.parametrize("shape", [(300, 20, 30), (70, 120, 130), (40, 129, 140), (257, 1, 9)])
def test_many_matrices(hip, shape):
    # more tiles than compute units, on both sides of the sides that take the finer sums
    m = matrix(12, *shape)
    out = hip.ones(shape)
    hip.orthogonalize(hip.create_from_numpy(m), out)
    got = out.get()
    for n in {0, 1, shape[0] // 2, shape[0] - 1}:
        assert off(got[n], ops.orthogonalize(m[n])) <= REL


def test_small_matrices_lose_no_more_than_float32(hip):
    # Planes round to 2^-24 like float32, and a sum rounds once for 32 entries instead of once for each: the error is not
    # larger than that of the same steps in NumPy's float32, but the two differ at random: a fifth for the mean of 40.
    def plain(m):
        x = m / np.sqrt((m * m).sum(dtype=F32))
        x = x.T if x.shape[0] > x.shape[1] else x
        for _ in range(5):
            gram = x @ x.T
            x = F32(3.4445) * x + (F32(-4.7750) * gram + F32(2.0315) * (gram @ gram)) @ x
        return x.T if m.shape[0] > m.shape[1] else x

    rng = np.random.RandomState(13)
    here, there = [], []
    for n in range(40):
        m = rng.standard_normal((rng.randint(8, 60), rng.randint(8, 200))).astype(F32)
        out = hip.ones(m.shape)
        hip.orthogonalize(hip.create_from_numpy(m), out)
        want = ops.orthogonalize(m)
        here.append(off(out.get(), want))
        there.append(off(plain(m), want))
    assert np.mean(here) <= 1.2 * np.mean(there), (np.mean(here), np.mean(there))


# How near the same steps in float32 the kernels have to be. Both lose bits where a matrix is stored and where products are added
# up, and the steps treat both alike. Stored: float32 rounds to 2^-24 of the binade, evenly spread, a mean square of 2^-48 / 3; two
# float16 planes round to half a unit of the low one, whose values spread evenly over its binades: 2^-46 / 3 (1/2 + 1/8 + ...) =
# (8/3) 2^-48 / 3. The product of two low planes that is left out: the square of a mean square of 2^-22 / 3, 2^-44 / 9, against the
# 2 2^-48 / 3 of two rounded factors another 8/3. Together 16/3, the root of which is 2.3; added up are 32 products at a time, where
# float32 rounds after each. 3 bounds the ratio then. Matrices of a few entries can be lucky in float32: a step's own error is
# about 30 2^-23 at most (A to 4.4 2^-23, p to 4.8 times that and 3.5 2^-23, the product to 1.2 times that), a quarter of it with signs
# at random, 2^-20.
def float32_steps(m, steps=5):
    if m.ndim == 3:
        return np.stack([float32_steps(x, steps) for x in m])
    x = (m.astype(np.float64) / np.linalg.norm(m.astype(np.float64))).astype(F32)
    x = x.T if x.shape[0] > x.shape[1] else x
    for _ in range(steps):
        gram = x @ x.T
        x = F32(3.4445) * x + (F32(-4.7750) * gram + F32(2.0315) * (gram @ gram)) @ x
    return x.T if m.shape[0] > m.shape[1] else x


def near_float32(hip, m, steps=5):
    out = hip.ones(m.shape)
    hip.orthogonalize(hip.create_from_numpy(m), out, steps=steps)
    want = ops.orthogonalize(m, steps)
    here, there = off(out.get(), want), off(float32_steps(m, steps), want)
    assert here <= 3 * there + 2.0 ** -20, (here, there)


@pytest.mark.parametrize("rows,cols", SHAPES + [(8, 2400), (2400, 64), (127, 131), (192, 192), (257, 1025)])
def test_as_near_as_float32(hip, rows, cols):
    near_float32(hip, matrix(rows * 7 + cols, rows, cols))


@pytest.mark.parametrize("steps", [1, 2, 3, 8, 12])
@pytest.mark.parametrize("shape", [(40, 70), (200, 150)])
def test_other_numbers_of_steps_as_near_as_float32(hip, steps, shape):
    near_float32(hip, matrix(3, *shape), steps)


@pytest.mark.parametrize("shape", [(4, 30, 50), (3, 140, 60), (2, 256, 384), (4, 300, 300)])
def test_stacks_as_near_as_float32(hip, shape):
    near_float32(hip, matrix(4, *shape))


def test_low_rank_and_uneven_matrices_as_near_as_float32(hip):
    rng = np.random.RandomState(6)
    one = np.zeros((130, 70), F32)
    one[100, 5] = -3.0
    spiked = matrix(7, 100, 260)
    spiked[3] *= 1e4
    for m in ((rng.standard_normal((200, 3)) @ rng.standard_normal((3, 150))).astype(F32), one, spiked):
        near_float32(hip, m)


@pytest.mark.parametrize("shape", [(12, 20), (200, 30), (3, 64, 65), (1000, 205)])
def test_update_as_near_as_float32(hip, shape):
    g, v, p = matrix(11, *shape), matrix(12, *shape), np.zeros(shape, F32)
    dg, dv, dp = (hip.create_from_numpy(x) for x in (g, v, p))
    hip.orthogonal_update(0.9, -0.5, dg, dv, dp)
    v = F32(0.9) * v + g                             # two roundings each, as the handler's own operations
    u = g + F32(0.9) * v
    factor = -0.5 * np.sqrt(max(1.0, shape[-2] / shape[-1]))
    want = factor * ops.orthogonalize(u)
    here, there = off(dp.get(), want), off(float32_steps(u), ops.orthogonalize(u))
    assert here <= 3 * there + 2.0 ** -20 + 2.0 ** -23, (here, there)      # the factor and the sum round too
