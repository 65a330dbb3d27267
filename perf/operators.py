"""What is measured of the sequence, norm and update operators, case by case.

Three operators, as a recurrent network built of them uses them: linear attention with a decay for each head
(a whole sequence, its training pass, one step), the norm behind a block with its gate, residual scale and
the norm before the next block (forward, training pass), and a momentum update whose matrices are
orthogonalised by Newton-Schulz products. ``run`` computes a case in plain torch operations, or, with ``own``
set, through brainstorm_amd's handler; ``exact`` gives the same outputs from the definitions in 64 bits.

Arrays are (time, batch, features) with the heads side by side in the features, as the handler's layers
have them, everything float32.
"""
import math

import torch

own = False

# quintic Newton-Schulz step x -> a x + b x^3 + c x^5
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
EPSILON = 1e-6
CHUNK = 64          # time steps of one chunk in the plain form of linear attention

_HANDLER = None


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token for one user: 8 heads, a launch's latency is what counts
        {"name": "step_one_sequence", "op": "step", "batch": 1, "heads": 8, "dk": 64, "dv": 64},
        # one token for each of 256 users at once: half a gigabyte of states read and written
        {"name": "step_many_sequences", "op": "step", "batch": 256, "heads": 16, "dk": 128, "dv": 128},
        # a long prompt of one user, its state kept: parallel work only along the time axis
        {"name": "prompt_long", "op": "attend", "time": 8192, "batch": 1, "heads": 16, "dk": 64, "dv": 64,
         "carry": True, "ragged": False},
        # training on the character sequences of the LSTM workload: 1000 units as 8 heads of 125 (odd rows)
        {"name": "train_char_sequences", "op": "attend_train", "time": 100, "batch": 100, "heads": 8, "dk": 125,
         "dv": 125, "carry": False, "ragged": False},
        # training on longer sequences with full-size heads
        {"name": "train_wide_heads", "op": "attend_train", "time": 1024, "batch": 8, "heads": 16, "dk": 128,
         "dv": 128, "carry": False, "ragged": False},
        # a padded batch cut out of longer sequences: lengths, a state from before and a gradient from behind
        {"name": "train_ragged_carry", "op": "attend_train", "time": 777, "batch": 5, "heads": 3, "dk": 40, "dv": 72,
         "carry": True, "ragged": True},
        # one token between two blocks of 1000 units
        {"name": "gate_one_row", "op": "gate", "rows": 1, "width": 1000, "activation": "swish"},
        # a batch between two blocks of the highway workload's width
        {"name": "gate_wide", "op": "gate", "rows": 2048, "width": 4096, "activation": "swish"},
        # training on the character sequences: 100 time steps of 100 sequences
        {"name": "gate_train_char", "op": "gate_train", "rows": 10000, "width": 1000, "activation": "sigmoid"},
        # a gradient of the first weight matrix of the image workload's perceptron, orthogonalised by itself
        {"name": "orthogonalize_perceptron", "op": "orthogonalize", "count": 1, "rows": 1200, "cols": 784},
        # the four recurrent matrices of the LSTM workload, back to back in the parameter vector
        {"name": "update_recurrent", "op": "update", "count": 4, "rows": 1000, "cols": 1000},
        # one weight matrix of the highway workload
        {"name": "update_highway", "op": "update", "count": 1, "rows": 4096, "cols": 4096},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "attend", "attend_train", "gate", "gate_train", "update", "orthogonalize"])
    if op in ("step", "attend", "attend_train"):
        case = {"op": op, "batch": _log_int(rng, 1, 256 if op == "step" else 64), "heads": _log_int(rng, 1, 16),
                "dk": _log_int(rng, 8, 128), "dv": _log_int(rng, 8, 128)}
        if op != "step":
            most = (1 << 23) // (case["batch"] * case["heads"] * max(case["dk"], case["dv"]))
            case.update(time=_log_int(rng, 1, max(1, min(8192, most))), carry=rng.random() < 0.5,
                        ragged=rng.random() < 0.5)
        return case
    if op in ("gate", "gate_train"):
        width = _log_int(rng, 16, 8192)
        return {"op": op, "rows": _log_int(rng, 1, min(20000, (1 << 23) // width)), "width": width,
                "activation": rng.choice(["linear", "sigmoid", "tanh", "swish"])}
    return {"op": op, "count": _log_int(rng, 1, 4), "rows": _log_int(rng, 8, 2400), "cols": _log_int(rng, 8, 2400)}


def work(case):
    op = case["op"]
    if op in ("step", "attend", "attend_train"):
        sequences, dk, dv = case["batch"] * case["heads"], case["dk"], case["dv"]
        tokens = sequences * case.get("time", 1)
        state = 4 * sequences * dk * dv
        if op == "step":
            return {"bytes": 4 * tokens * 2 * (dk + dv) + 2 * state, "flops": 4 * tokens * dk * dv}
        carried = 2 * state if case["carry"] else 0
        if op == "attend":
            return {"bytes": 4 * tokens * 2 * (dk + dv) + carried, "flops": 4 * tokens * dk * dv}
        # forward: k v^T into the state and q times it; backward: the state again, the state of the gradients,
        # and a product with one of the two for each of dq, dk, dv
        return {"bytes": 4 * tokens * 4 * (dk + dv) + 2 * carried, "flops": 14 * tokens * dk * dv}
    if op in ("gate", "gate_train"):
        n = case["rows"] * case["width"]
        if op == "gate":
            return {"bytes": 4 * n * 5, "flops": 12 * n}
        return {"bytes": 4 * n * 10, "flops": 40 * n}
    small, large = sorted((case["rows"], case["cols"]))
    # the two symmetric products of a step need one half each
    flops = 5 * (small * small * large + small ** 3 + 2 * small * small * large)
    arrays = 5 if op == "update" else 2
    return {"bytes": 4 * arrays * case["count"] * small * large, "flops": case["count"] * flops}


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std)

    def space(like):
        return torch.empty_like(like)

    op = case["op"]
    s = {"case": case, "op": op}
    if op in ("step", "attend", "attend_train"):
        heads, dk, dv, batch = case["heads"], case["dk"], case["dv"], case["batch"]
        lead = (batch,) if op == "step" else (case["time"], batch)
        s["scale"] = dk ** -0.5
        # one minus a power of two, from a memory of 32 steps to one of 512
        s["decay"] = 1 - torch.exp2(-torch.linspace(5, 9, heads, device="cuda"))
        s["q"], s["k"], s["v"] = normal(*lead, heads * dk), normal(*lead, heads * dk), normal(*lead, heads * dv)
        s["out"] = space(s["v"])
        if op == "step":
            s["state"] = normal(batch, heads, dk, dv, std=3.0)
            return s
        if case["ragged"]:
            s["lengths"] = torch.randint(0, case["time"] + 1, (batch,), generator=g, device="cuda").float()
        if case["carry"]:
            s["state"] = normal(batch, heads, dk, dv, std=3.0)
            s["new_state"] = space(s["state"])
        if op == "attend_train":
            s["dout"] = normal(*lead, heads * dv, std=0.01)
            s["dq"], s["dk"], s["dv"], s["ddecay"] = space(s["q"]), space(s["k"]), space(s["v"]), space(s["decay"])
            if case["carry"]:
                s["dnew_state"] = normal(batch, heads, dk, dv, std=0.01)
                s["dstate"] = space(s["state"])
    elif op in ("gate", "gate_train"):
        shape = (case["rows"], case["width"])
        s["block"], s["gate"], s["x"] = normal(*shape, std=0.7), normal(*shape), normal(*shape, std=2.0)
        s["post"] = 1 + normal(shape[1], std=0.1)
        s["pre"] = 1 + normal(shape[1], std=0.1)
        s["residual_scale"] = 0.9
        s["y"], s["h"] = space(s["x"]), space(s["x"])
        if op == "gate_train":
            s["dy"], s["dh"] = normal(*shape, std=0.01), normal(*shape, std=0.01)
            for name in ("dblock", "dgate", "dx"):
                s[name] = space(s["x"])
            s["dpost"], s["dpre"] = space(s["post"]), space(s["pre"])
    else:
        shape = (case["count"], case["rows"], case["cols"])
        rank = max(1, min(shape[1:]) // 16)
        # a gradient: a few strong directions and noise
        strong = torch.matmul(normal(shape[0], shape[1], rank), normal(shape[0], rank, shape[2]))
        s["gradients"] = (strong / math.sqrt(rank) + normal(*shape)) * 1e-3
        if op == "orthogonalize":
            s["out"] = space(s["gradients"])
            return s
        s["velocity"] = normal(*shape, std=1e-2)
        s["parameters"] = normal(*shape, std=shape[2] ** -0.5)
        s["momentum"], s["neg_learning_rate"] = 0.95, -0.02
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    op = s["op"]
    if op == "step":
        return _plain_step(s)
    if op == "attend":
        return _plain_attend(s)
    if op == "attend_train":
        return {**_plain_attend(s), **_plain_attend_backward(s)}
    if op == "gate":
        return _plain_gate(s)
    if op == "gate_train":
        return _plain_gate_train(s)
    if op == "orthogonalize":
        return {"out": _plain_orthogonal(s["gradients"])}
    return _plain_update(s)


def _own(s):
    views = s.get("views")
    if views is None:
        views = s["views"] = _handler_views(s)
    h = _HANDLER
    op = s["op"]
    if op == "step":
        h.linear_attention_step(views["q"], views["k"], views["v"], views["decay"], views["state"], views["out"],
                                scale=s["scale"])
        return {"out": s["out"], "state": s["state"]}
    if op in ("attend", "attend_train"):
        carried = s["case"]["carry"]
        h.linear_attention_forward(views["q"], views["k"], views["v"], views["decay"], views["out"], scale=s["scale"],
                                   state=views.get("state"), new_state=views.get("new_state"),
                                   lengths=views.get("lengths"))
        result = {"out": s["out"]}
        if carried:
            result["new_state"] = s["new_state"]
        if op == "attend_train":
            h.linear_attention_backward(views["q"], views["k"], views["v"], views["decay"], views["dout"],
                                        views["dq"], views["dk"], views["dv"], views["ddecay"], scale=s["scale"],
                                        state=views.get("state"), dnew_state=views.get("dnew_state"),
                                        dstate=views.get("dstate"), lengths=views.get("lengths"))
            result.update(dq=s["dq"], dk=s["dk"], dv=s["dv"], ddecay=s["ddecay"])
            if carried:
                result["dstate"] = s["dstate"]
        return result
    if op in ("gate", "gate_train"):
        h.gated_residual_forward(s["case"]["activation"], views["block"], views["gate"], views["x"], views["post"],
                                 views["pre"], views["y"], views["h"], residual_scale=s["residual_scale"],
                                 epsilon=EPSILON)
        result = {"y": s["y"], "h": s["h"]}
        if op == "gate_train":
            h.gated_residual_backward(s["case"]["activation"], views["block"], views["gate"], views["post"],
                                      views["pre"], views["y"], views["dy"], views["dh"], views["dblock"],
                                      views["dgate"], views["dx"], views["dpost"], views["dpre"],
                                      residual_scale=s["residual_scale"], epsilon=EPSILON, accumulate=False)
            result.update((name, s[name]) for name in ("dblock", "dgate", "dx", "dpost", "dpre"))
        return result
    if op == "orthogonalize":
        h.orthogonalize(views["gradients"], views["out"])
        return {"out": s["out"]}
    h.orthogonal_update(s["momentum"], s["neg_learning_rate"], views["gradients"], views["velocity"],
                        views["parameters"])
    return {"parameters": s["parameters"], "velocity": s["velocity"]}


def _handler_views(s):
    """The handler's arrays over a state's memory, made at the first pass and kept as a program keeps its own."""
    global _HANDLER
    from brainstorm_amd import DeviceArray, HipHandler
    if _HANDLER is None:
        _HANDLER = HipHandler(seed=0)
    return {name: DeviceArray(t.data_ptr(), tuple(t.shape), t, _HANDLER)
            for name, t in s.items() if isinstance(t, torch.Tensor)}


# ------------------------------------------------------------------ linear attention, plain
# o_t = scale q_t S_t,  S_t = decay S_{t-1} + k_t^T v_t, in chunks of CHUNK steps: products inside a chunk,
# the chunks' states U joined by a matrix of powers of the decay.
def _powers(decay, exponents):
    """decay^exponents for every head, from 64 bits; exponents below zero give 0."""
    e = exponents.double()
    return torch.where(e < 0, 0.0, decay.double().reshape(-1, *[1] * e.dim()) ** e.clamp(min=0)).float()


def _power_slopes(decay, exponents):
    """d/d decay of _powers."""
    e = exponents.double()
    d = decay.double().reshape(-1, *[1] * e.dim())
    return torch.where(e < 1, 0.0, e * d ** (e - 1).clamp(min=0)).float()


def _lengths(s):
    time, batch = s["q"].shape[:2]
    if "lengths" in s:
        return s["lengths"].long().clamp(0, time)
    return torch.full((batch,), time, device="cuda", dtype=torch.long)


def _chunked(s, name):
    """(batch, heads, chunks, CHUNK, d) of an array (time, batch, heads * d), rows behind the end zero."""
    t = s[name]
    time, batch, heads = t.shape[0], t.shape[1], s["decay"].numel()
    if "lengths" in s:
        rows = torch.arange(time, device="cuda")[:, None] < _lengths(s)
        t = torch.where(rows[:, :, None], t, 0.0)
    t = t.reshape(time, batch, heads, -1).permute(1, 2, 0, 3)
    chunks = -(-time // CHUNK)
    t = torch.nn.functional.pad(t, (0, 0, 0, chunks * CHUNK - time))
    return t.reshape(batch, heads, chunks, CHUNK, -1)


def _unchunked(s, t):
    time, batch = s["q"].shape[:2]
    t = t.flatten(2, 3)[:, :, :time].permute(2, 0, 1, 3).reshape(time, batch, -1)
    if "lengths" in s:
        rows = torch.arange(time, device="cuda")[:, None] < _lengths(s)
        t = torch.where(rows[:, :, None], t, 0.0)
    return t.contiguous()


def _chunk_tables(s):
    chunks = -(-s["q"].shape[0] // CHUNK)
    i, c = torch.arange(CHUNK, device="cuda"), torch.arange(chunks, device="cuda")
    inside, across = i[:, None] - i[None, :], CHUNK * (c[:, None] - 1 - c[None, :])
    return i, c, inside, across


def _into_end(s, chunks):
    """Exponents of the decay that a step's k^T v has in the final state: length - 1 - t (below zero: behind it)."""
    t = torch.arange(chunks * CHUNK, device="cuda").reshape(chunks, CHUNK)
    return _lengths(s)[:, None, None] - 1 - t


def _chunk_states(s, k, v):
    """The state at every chunk's beginning, and each chunk's own contribution to its end."""
    decay, (i, c, _, across) = s["decay"], _chunk_tables(s)
    u = torch.matmul((k * _powers(decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2), v)
    start = torch.matmul(_powers(decay, across), u.flatten(3)).reshape(u.shape)
    if "state" in s:
        start = start + _powers(decay, CHUNK * c)[:, :, None, None] * s["state"][:, :, None]
    return start, u


def _plain_attend(s):
    q, k, v = (_chunked(s, name) for name in ("q", "k", "v"))
    decay, (i, _, inside, _) = s["decay"], _chunk_tables(s)
    start, _ = _chunk_states(s, k, v)
    a = torch.matmul(q, k.transpose(-1, -2)) * _powers(decay, inside)[:, None]
    o = torch.matmul(a, v) + _powers(decay, i + 1)[:, None, :, None] * torch.matmul(q, start)
    result = {"out": _unchunked(s, s["scale"] * o)}
    if "state" in s:
        w = _powers(decay, _into_end(s, k.shape[2])).transpose(0, 1)[..., None]
        own_part = torch.matmul((k * w).flatten(2, 3).transpose(-1, -2), v.flatten(2, 3))
        result["new_state"] = own_part + _powers(decay, _lengths(s)).t()[..., None, None] * s["state"]
    return result


def _plain_attend_backward(s):
    q, k, v, do = (_chunked(s, name) for name in ("q", "k", "v", "dout"))
    decay, scale, (i, c, inside, across) = s["decay"], s["scale"], _chunk_tables(s)
    start, u = _chunk_states(s, k, v)
    d_inside, mix = _powers(decay, inside)[:, None], _powers(decay, across)
    w_in, w_out = _powers(decay, i + 1)[:, None, :, None], _powers(decay, CHUNK - 1 - i)[:, None, :, None]
    scores, dscores = torch.matmul(q, k.transpose(-1, -2)), torch.matmul(do, v.transpose(-1, -2))
    a, p = scores * d_inside, dscores * d_inside
    gs = scale * torch.matmul((q * w_in).transpose(-1, -2), do)                      # of a chunk's first state
    gu = torch.matmul(mix.transpose(-1, -2), gs.flatten(3)).reshape(gs.shape)        # of a chunk's contribution
    dq = scale * (torch.matmul(p, k) + w_in * torch.matmul(do, start.transpose(-1, -2)))
    dk = scale * torch.matmul(p.transpose(-1, -2), q) + w_out * torch.matmul(v, gu.transpose(-1, -2))
    dv = scale * torch.matmul(a.transpose(-1, -2), do) + w_out * torch.matmul(k, gu)
    # of the decay: inside the chunks, into a chunk, between chunks, out of a chunk
    slope = (scale * scores * dscores * _power_slopes(decay, inside)[:, None]).sum((0, 2, 3, 4))
    s_in = _power_slopes(decay, i + 1)[:, None, :, None]
    slope = slope + (scale * s_in * torch.matmul(q, start) * do).sum((0, 2, 3, 4))
    pairs = torch.matmul(gs.flatten(3), u.flatten(3).transpose(-1, -2))
    slope = slope + (pairs * _power_slopes(decay, across)).sum((0, 2, 3))
    s_out = _power_slopes(decay, CHUNK - 1 - i)[:, None, :, None]
    slope = slope + (s_out * torch.matmul(k, gu) * v).sum((0, 2, 3, 4))
    result = {}
    if "state" in s:
        first, last, length = s["state"], s["dnew_state"], _lengths(s)
        slope = slope + ((gs * first[:, :, None]).sum((3, 4)) * _power_slopes(decay, CHUNK * c)).sum((0, 2))
        end = _into_end(s, k.shape[2])
        w = _powers(decay, end).transpose(0, 1)[..., None]
        k_last = torch.matmul(k, last[:, :, None])
        dk = dk + w * torch.matmul(v, last[:, :, None].transpose(-1, -2))
        dv = dv + w * k_last
        slope = slope + (_power_slopes(decay, end).transpose(0, 1)[..., None] * k_last * v).sum((0, 2, 3, 4))
        slope = slope + ((first * last).sum((2, 3)) * _power_slopes(decay, length).t()).sum(0)
        result["dstate"] = ((gs * _powers(decay, CHUNK * c)[:, :, None, None]).sum(2)
                            + _powers(decay, length).t()[..., None, None] * last)
    result.update(dq=_unchunked(s, dq), dk=_unchunked(s, dk), dv=_unchunked(s, dv), ddecay=slope)
    return result


def _plain_step(s):
    batch, heads = s["q"].shape[0], s["decay"].numel()
    q, k, v = (s[name].reshape(batch, heads, -1) for name in ("q", "k", "v"))
    s["state"].mul_(s["decay"][:, None, None]).add_(k[..., None] * v[..., None, :])
    o = s["scale"] * torch.matmul(q[:, :, None], s["state"])
    return {"out": o.reshape(s["v"].shape), "state": s["state"]}


# ------------------------------------------------------------------ the norms and the gate, plain
def _gate_value(activation, z):
    if activation == "linear":
        return z
    if activation == "sigmoid":
        return torch.sigmoid(z)
    if activation == "tanh":
        return torch.tanh(z)
    return z * torch.sigmoid(z)


def _gate_slope(activation, z):
    if activation == "linear":
        return torch.ones_like(z)
    if activation == "sigmoid":
        return torch.sigmoid(z) * (1 - torch.sigmoid(z))
    if activation == "tanh":
        return 1 - torch.tanh(z) ** 2
    sig = torch.sigmoid(z)
    return sig * (1 + z * (1 - sig))


def _inverse_rms(x):
    return torch.rsqrt((x * x).mean(1, keepdim=True) + EPSILON)


def _plain_gate(s):
    block, x = s["block"], s["x"]
    gate = _gate_value(s["case"]["activation"], s["gate"])
    y = s["residual_scale"] * x + gate * (s["post"] * (block * _inverse_rms(block)))
    return {"y": y, "h": s["pre"] * (y * _inverse_rms(y))}


def _norm_gradient(x, r, d):
    """Gradient of x for n = x r(x), given d = that of n."""
    return r * (d - x * (r * r) * (d * x).mean(1, keepdim=True))


def _plain_gate_train(s):
    result = _plain_gate(s)
    block, y, activation = s["block"], result["y"], s["case"]["activation"]
    ry, rb = _inverse_rms(y), _inverse_rms(block)
    total = s["dy"] + _norm_gradient(y, ry, s["dh"] * s["pre"])
    gate, normed = _gate_value(activation, s["gate"]), block * rb
    result["dpre"] = (s["dh"] * (y * ry)).sum(0)
    result["dpost"] = (total * gate * normed).sum(0)
    result["dx"] = s["residual_scale"] * total
    result["dgate"] = total * (s["post"] * normed) * _gate_slope(activation, s["gate"])
    result["dblock"] = _norm_gradient(block, rb, total * gate * s["post"])
    return result


# ------------------------------------------------------------------ the orthogonalised update, plain
def _plain_orthogonal(u):
    norm = u.double().square().sum((1, 2), keepdim=True).sqrt()
    x = torch.where(norm == 0, 0.0, u / norm).float()
    rows, cols = x.shape[1:]
    if rows > cols:
        x = x.transpose(1, 2).contiguous()
    for _ in range(5):
        a = torch.matmul(x, x.transpose(1, 2))
        b = NS_B * a + NS_C * torch.matmul(a, a)
        x = NS_A * x + torch.matmul(b, x)
    return x.transpose(1, 2).contiguous() if rows > cols else x


def _plain_update(s):
    v = s["velocity"]
    v.mul_(s["momentum"]).add_(s["gradients"])
    x = _plain_orthogonal(s["gradients"] + s["momentum"] * v)
    rows, cols = x.shape[1:]
    s["parameters"].add_(x, alpha=s["neg_learning_rate"] * max(1.0, rows / cols) ** 0.5)
    return {"parameters": s["parameters"], "velocity": v}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {name: t.double() for name, t in s.items() if isinstance(t, torch.Tensor) and t.numel()}
    if op == "step":
        batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
        state = d["decay"].reshape(1, heads, 1, 1) * d["state"] + torch.einsum(
            "bhi,bhj->bhij", d["k"].reshape(batch, heads, dk), d["v"].reshape(batch, heads, dv))
        out = (d["q"].reshape(batch, heads, dk, 1) * state).sum(2) * s["scale"]
        return {"out": out.reshape(batch, heads * dv), "state": state}
    if op in ("attend", "attend_train"):
        return _exact_attention(case, s, d)
    if op in ("gate", "gate_train"):
        return _exact_gate(case, s, d)
    if op == "orthogonalize":
        return {"out": torch.stack([_exact_orthogonal(one) for one in d["gradients"]])}
    return _exact_update(case, s, d)


def _exact_attention(case, s, d):
    """Every head of every sequence from the full matrix of decay^(t - s), sequence by sequence."""
    time, batch, heads, dk, dv = case["time"], case["batch"], case["heads"], case["dk"], case["dv"]
    if batch * heads * time * time > 5e9:
        return None
    train, carry, scale = case["op"] == "attend_train", case["carry"], s["scale"]
    f64 = {"dtype": torch.float64, "device": "cuda"}
    result = {"out": torch.zeros(time, batch, heads * dv, **f64)}
    if carry:
        result["new_state"] = torch.zeros(batch, heads, dk, dv, **f64)
    if train:
        result.update(dq=torch.zeros(time, batch, heads * dk, **f64), dk=torch.zeros(time, batch, heads * dk, **f64),
                      dv=torch.zeros(time, batch, heads * dv, **f64), ddecay=torch.zeros(heads, **f64))
        if carry:
            result["dstate"] = torch.zeros(batch, heads, dk, dv, **f64)
    lengths = [int(x) for x in s["lengths"]] if "lengths" in s else [time] * batch
    decays = [float(x) for x in s["decay"]]
    for b, n in enumerate(lengths):
        t = torch.arange(n, **f64)
        gap = t[:, None] - t[None, :]
        for h, decay in enumerate(decays):
            ks, vs = slice(h * dk, h * dk + dk), slice(h * dv, h * dv + dv)
            q, k, v = d["q"][:n, b, ks], d["k"][:n, b, ks], d["v"][:n, b, vs]
            weight = torch.tril(decay ** gap.clamp(min=0))
            scores = q @ k.T
            o = (weight * scores) @ v
            if carry:
                first = d["state"][b, h]
                o = o + decay ** (t + 1)[:, None] * (q @ first)
                to_end = decay ** (n - 1 - t)[:, None]
                result["new_state"][b, h] = (k * to_end).T @ v + decay ** n * first
            result["out"][:n, b, vs] = scale * o
            if not train:
                continue
            do = scale * d["dout"][:n, b, vs]
            grads = do @ v.T
            dq, dks, dvs = (weight * grads) @ k, (weight * grads).T @ q, (weight * scores).T @ do
            slope = (torch.tril(gap) * decay ** (gap - 1).clamp(min=0) * scores * grads).sum()
            if carry:
                last = d["dnew_state"][b, h]
                dq = dq + decay ** (t + 1)[:, None] * (do @ first.T)
                dks = dks + to_end * (v @ last.T)
                dvs = dvs + to_end * (k @ last)
                result["dstate"][b, h] = (q * decay ** (t + 1)[:, None]).T @ do + decay ** n * last
                slope = slope + ((t + 1) * decay ** t * ((q @ first) * do).sum(1)).sum()
                slope = slope + ((n - 1 - t) * decay ** (n - 2 - t).clamp(min=0) * ((k @ last) * v).sum(1)).sum()
                slope = slope + n * decay ** max(0, n - 1) * (first * last).sum()
            result["dq"][:n, b, ks], result["dk"][:n, b, ks], result["dv"][:n, b, vs] = dq, dks, dvs
            result["ddecay"][h] += slope
    return result


def _exact_gate(case, s, d):
    """The forward pass written out, its gradients by automatic differentiation."""
    train = case["op"] == "gate_train"
    leaves = {n: d[n].requires_grad_(train) for n in ("block", "gate", "x", "post", "pre")}
    z = leaves["gate"]
    value = {"linear": lambda: z, "sigmoid": lambda: 1 / (1 + torch.exp(-z)), "tanh": lambda: torch.tanh(z),
             "swish": lambda: z / (1 + torch.exp(-z))}[case["activation"]]()
    block = leaves["block"]
    normed = block / torch.sqrt(block.pow(2).mean(1, keepdim=True) + EPSILON) * leaves["post"]
    y = s["residual_scale"] * leaves["x"] + value * normed
    h = y / torch.sqrt(y.pow(2).mean(1, keepdim=True) + EPSILON) * leaves["pre"]
    result = {"y": y.detach(), "h": h.detach()}
    if train:
        torch.autograd.backward((y, h), (d["dy"], d["dh"]))
        result.update(("d" + n, leaf.grad) for n, leaf in leaves.items())
    return result


def _exact_orthogonal(u):
    rows, cols = u.shape
    x = u / max(float(torch.linalg.vector_norm(u)), 1e-300)
    for _ in range(5):
        a = x @ x.T if rows <= cols else x.T @ x
        poly = NS_B * a + NS_C * (a @ a)
        x = NS_A * x + (poly @ x if rows <= cols else x @ poly)
    return x


def _exact_update(case, s, d):
    v = s["momentum"] * d["velocity"] + d["gradients"]
    u = d["gradients"] + s["momentum"] * v
    x = torch.stack([_exact_orthogonal(one) for one in u])
    factor = s["neg_learning_rate"] * math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return {"parameters": d["parameters"] + factor * x, "velocity": v}
