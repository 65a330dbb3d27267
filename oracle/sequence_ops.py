"""Linear attention with a decay, the gated residual with its norms, and Newton-Schulz orthogonalisation in
plain NumPy, float64 throughout, written from the definitions: what the tests of the kernels compare with. TEST
INFRASTRUCTURE, like the rest of this package; ``SequenceRefHandler`` gives the oracle handler these operators, so
that networks with them run on it."""
import numpy as np

from .numpy_ref_handler import NumpyRefHandler

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def sequence_lengths(lengths, time, batch):
    """Steps of every batch element from float labels: truncated, into [0, time], NaN counts as 0."""
    if lengths is None:
        return np.full(batch, time, dtype=int)
    x = np.nan_to_num(np.asarray(lengths, dtype=np.float64).ravel(), nan=0.0, posinf=time, neginf=0.0)
    return np.clip(np.trunc(x), 0, time).astype(int)


def _split(a, heads):
    return np.asarray(a, dtype=np.float64).reshape(a.shape[0], a.shape[1], heads, -1)


def linear_attention(q, k, v, decay, scale=1.0, state=None, lengths=None):
    """(out, new_state) of S_t = decay S_(t-1) + k_t^T v_t, out_t = scale q_t S_t, step by step."""
    heads = np.size(decay)
    q, k, v = (_split(a, heads) for a in (q, k, v))
    g = np.asarray(decay, dtype=np.float64).reshape(heads)[None, :, None, None]
    time, batch = q.shape[:2]
    n = sequence_lengths(lengths, time, batch)
    s = np.zeros((batch, heads, q.shape[3], v.shape[3]))
    if state is not None:
        s = s + np.asarray(state, dtype=np.float64).reshape(s.shape)
    out = np.zeros(v.shape)
    for t in range(time):
        live = t < n
        s[live] = g * s[live] + k[t, live, :, :, None] * v[t, live, :, None, :]
        out[t, live] = scale * np.einsum("bhi,bhij->bhj", q[t, live], s[live])
    return out.reshape(time, batch, -1), s


def linear_attention_gradients(q, k, v, decay, dout, scale=1.0, state=None, dnew_state=None, lengths=None):
    """(dq, dk, dv, ddecay, dstate), by the recurrence backwards through the states of every step."""
    heads = np.size(decay)
    q, k, v, do = (_split(a, heads) for a in (q, k, v, dout))
    g = np.asarray(decay, dtype=np.float64).reshape(heads)[None, :, None, None]
    time, batch = q.shape[:2]
    n = sequence_lengths(lengths, time, batch)
    s = np.zeros((batch, heads, q.shape[3], v.shape[3]))
    if state is not None:
        s = s + np.asarray(state, dtype=np.float64).reshape(s.shape)
    states = [s.copy()]                              # before each step
    for t in range(time):
        live = t < n
        s[live] = g * s[live] + k[t, live, :, :, None] * v[t, live, :, None, :]
        states.append(s.copy())
    r = np.zeros(s.shape)
    if dnew_state is not None:
        r = r + np.asarray(dnew_state, dtype=np.float64).reshape(s.shape)
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    ddecay = np.zeros(heads)
    for t in range(time - 1, -1, -1):
        live = t < n
        dq[t, live] = scale * np.einsum("bhj,bhij->bhi", do[t, live], states[t + 1][live])
        r[live] += scale * q[t, live, :, :, None] * do[t, live, :, None, :]
        dk[t, live] = np.einsum("bhij,bhj->bhi", r[live], v[t, live])
        dv[t, live] = np.einsum("bhij,bhi->bhj", r[live], k[t, live])
        ddecay += (r[live] * states[t][live]).sum((0, 2, 3))
        r[live] = g * r[live]
    return (dq.reshape(time, batch, -1), dk.reshape(time, batch, -1), dv.reshape(time, batch, -1), ddecay, r)


def gate_value(activation, z):
    z = np.asarray(z, dtype=np.float64)
    if activation == "sigmoid":
        return 1 / (1 + np.exp(-z))
    if activation == "tanh":
        return np.tanh(z)
    if activation == "rel":
        return np.maximum(z, 0)
    if activation == "el":
        return np.where(z > 0, z, np.expm1(np.minimum(z, 0)))
    if activation == "swish":
        return z / (1 + np.exp(-z))
    return z


def gate_slope(activation, z):
    z = np.asarray(z, dtype=np.float64)
    s = 1 / (1 + np.exp(-z))
    return {"sigmoid": s * (1 - s), "tanh": 1 - np.tanh(z) ** 2, "rel": (z > 0).astype(float),
            "el": np.where(z > 0, 1.0, np.exp(np.minimum(z, 0))), "swish": s + z * s * (1 - s),
            "linear": np.ones(z.shape)}[activation]


def inverse_rms(x, epsilon):
    x = np.asarray(x, dtype=np.float64)
    return 1 / np.sqrt((x * x).mean(1, keepdims=True) + epsilon)


def gated_residual(activation, block, gate, x, post, pre, residual_scale=1.0, epsilon=1e-6):
    """(y, h); block None: (x, norm of x); gate None: no gate; pre None: (y, None)."""
    x = np.asarray(x, dtype=np.float64)
    if block is None:
        y = x
    else:
        block = np.asarray(block, dtype=np.float64)
        value = 1.0 if gate is None else gate_value(activation, gate)
        y = residual_scale * x + value * np.asarray(post, dtype=np.float64) * block * inverse_rms(block, epsilon)
    return y, None if pre is None else np.asarray(pre, dtype=np.float64) * y * inverse_rms(y, epsilon)


def _norm_gradient(x, r, d):
    return r * (d - x * r * r * (d * x).mean(1, keepdims=True))


def gated_residual_gradients(activation, block, gate, post, pre, y, dy, dh, residual_scale=1.0, epsilon=1e-6):
    """dict of dx, and where they exist dblock, dgate, dpost, dpre, for a given y."""
    f64 = lambda a: None if a is None else np.asarray(a, dtype=np.float64)
    block, gate, post, pre, y, dy, dh = (f64(a) for a in (block, gate, post, pre, y, dy, dh))
    result = {}
    total = np.zeros((dh if dy is None else dy).shape) if dy is None else dy
    if pre is not None:
        r = inverse_rms(y, epsilon)
        total = total + _norm_gradient(y, r, dh * pre)
        result["dpre"] = (dh * y * r).sum(0)
    result["dx"] = residual_scale * total
    if block is not None:
        r = inverse_rms(block, epsilon)
        n, value = block * r, 1.0 if gate is None else gate_value(activation, gate)
        result["dpost"] = (total * value * n).sum(0)
        result["dblock"] = _norm_gradient(block, r, total * value * post)
        if gate is not None:
            result["dgate"] = total * post * n * gate_slope(activation, gate)
    return result


def orthogonalize(m, steps=5):
    """One matrix or a stack."""
    m = np.asarray(m, dtype=np.float64)
    if m.ndim == 3:
        return np.stack([orthogonalize(one, steps) for one in m]) if len(m) else m
    norm = np.sqrt((m * m).sum())
    x = m / norm if norm != 0 else m
    a, b, c = NS_COEFFICIENTS
    if x.shape[0] > x.shape[1]:
        x = x.T
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.T if m.shape[0] > m.shape[1] else x


def orthogonal_update(momentum, neg_learning_rate, gradients, velocity, parameters, steps=5, nesterov=True):
    """(velocity, parameters) after the update."""
    g, v, p = (np.asarray(a, dtype=np.float64) for a in (gradients, velocity, parameters))
    v = momentum * v + g
    u = g + momentum * v if nesterov else v
    rows, cols = p.shape[-2:]
    return v, p + neg_learning_rate * np.sqrt(max(1.0, rows / cols)) * orthogonalize(u, steps)


class SequenceRefHandler(NumpyRefHandler):
    """The oracle handler with HipHandler's sequence, norm and update operators (same signatures), in 64 bits and
    rounded once."""

    def linear_attention_forward(self, q, k, v, decay, out, scale=1.0, state=None, new_state=None, lengths=None):
        o, s = linear_attention(q, k, v, decay, scale, state, lengths)
        out[:] = o.reshape(out.shape)
        if new_state is not None:
            new_state[:] = s.reshape(new_state.shape)

    def linear_attention_step(self, q, k, v, decay, state, out, scale=1.0):
        o, s = linear_attention(q[None], k[None], v[None], decay, scale, state)
        out[:] = o.reshape(out.shape)
        state[:] = s.reshape(state.shape)

    def linear_attention_backward(self, q, k, v, decay, dout, dq, dk, dv, ddecay=None, scale=1.0, state=None,
                                  dnew_state=None, dstate=None, lengths=None):
        results = linear_attention_gradients(q, k, v, decay, dout, scale, state, dnew_state, lengths)
        for to, x in zip((dq, dk, dv, ddecay, dstate), results):
            if to is not None:
                to[:] = x.reshape(to.shape)

    def gated_residual_forward(self, activation, block, gate, x, post_weight, pre_weight, y, h, residual_scale=1.0,
                               epsilon=1e-6):
        y64, h64 = gated_residual(activation, block, gate, x, post_weight, pre_weight, residual_scale, epsilon)
        y[:] = y64
        if pre_weight is not None:
            h[:] = h64

    def gated_residual_backward(self, activation, block, gate, post_weight, pre_weight, y, dy, dh, dblock, dgate, dx,
                                dpost_weight, dpre_weight, residual_scale=1.0, epsilon=1e-6, accumulate=True):
        results = gated_residual_gradients(activation, block, gate, post_weight, pre_weight, y, dy,
                                           dh if pre_weight is not None else None, residual_scale, epsilon)
        for to, name in ((dblock, "dblock"), (dgate, "dgate"), (dx, "dx")):
            if to is not None:
                to[:] = results[name] + (to if accumulate else 0)
        for to, name in ((dpost_weight, "dpost"), (dpre_weight, "dpre")):
            if to is not None:
                to[:] = results[name].reshape(to.shape)

    def rms_norm_forward(self, x, weight, out, epsilon=1e-6):
        out[:] = gated_residual("linear", None, None, x, None, weight, epsilon=epsilon)[1]

    def rms_norm_backward(self, x, weight, dout, dx, dweight, epsilon=1e-6, accumulate=True):
        results = gated_residual_gradients("linear", None, None, None, weight, x, None, dout, epsilon=epsilon)
        dx[:] = results["dx"] + (dx if accumulate else 0)
        dweight[:] = results["dpre"].reshape(dweight.shape)

    def orthogonalize(self, m, out, steps=5):
        out[:] = orthogonalize(m, steps)

    def orthogonal_update(self, momentum, neg_learning_rate, gradients, velocity, parameters, steps=5, nesterov=True):
        velocity[:], parameters[:] = orthogonal_update(momentum, neg_learning_rate, gradients, velocity, parameters,
                                                       steps, nesterov)

    def momentum_update(self, momentum, neg_learning_rate, gradients, velocity, parameters):
        self.mult_st(momentum, velocity, out=velocity)
        self.mult_add_st(neg_learning_rate, gradients, out=velocity)
        self.add_tt(velocity, parameters, out=parameters)
