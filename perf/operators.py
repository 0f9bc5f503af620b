"""The operators of voxel-sequence networks: what they compute, in plain tensor operations, and the calls a program makes.

A voxel-sequence block takes the active voxels of a sparse tensor in some order (rows of `[rows, channels]` features, the
sequences of a batch behind one another) and mixes them along that order instead of through a kernel neighbourhood:
layer norm, a projection in 8-bit integers, a gated linear recurrence over the sequences, a projection back.  Here stand

* layer norm over the channels, with the residual sum in front of it (`op = "norm"`), with its backward pass
  (`"norm_train"`), and writing 8-bit rows for the product behind it (`"norm_linear"`),
* the product of 8-bit rows and 8-bit weights with a scale per row and per output channel (`"linear"`), also behind the
  quantisation of floating-point rows (`"quantize_linear"`),
* the gated linear recurrence h[t] = f[t] h[t-1] + (1 - f[t]) x[t], f = sigmoid(gate), over sequences of any length
  (`"scan"`, either direction), with its backward pass (`"scan_train"`), and for one token a sequence (`"step"`).

`listed()` names twelve cases, `draw()` gives more over the same ranges.  The plain form works in 32 bits (sums over all
rows in 64) and rounds once, at the end.
"""
import math

import torch

own = False  # False: the plain form; True: the package's operators

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # smallest: the tokens of one box head, launch and host path decide; odd number of rows
        dict(name="norm_257x96_fp32", op="norm", rows=257, channels=96, dtype="fp32", residual=False),
        # residual sum and norm in front of a block, 120 k voxels
        dict(name="norm_sum_120k_128_bf16", op="norm", rows=120000, channels=128, dtype="bf16", residual=True),
        # fine-tuning: norm and its backward pass at the second level of a detector, many rows of few channels
        dict(name="norm_train_238k_64_bf16", op="norm_train", rows=238000, channels=64, dtype="bf16"),
        # the same for few wide rows, in fp32
        dict(name="norm_train_4099x4096_fp32", op="norm_train", rows=4099, channels=4096, dtype="fp32"),
        # the front of a block in deployment: residual sum, norm and the 8-bit projection to features and gates
        dict(name="norm_linear_66k_256_512_bf16", op="norm_linear", rows=66001, inputs=256, outputs=512, dtype="bf16",
             residual=True),
        # one row through a large layer: every weight is read for it
        dict(name="linear_1_4096_4096_bf16", op="linear", rows=1, inputs=4096, outputs=4096, dtype="bf16"),
        # a thin projection over all voxels of a fine level: bytes
        dict(name="linear_238k_64_192_fp16", op="linear", rows=238000, inputs=64, outputs=192, dtype="fp16"),
        # the largest: a wide layer over many rows, products
        dict(name="linear_8192_4096_8192_bf16", op="linear", rows=8192, inputs=4096, outputs=8192, dtype="bf16"),
        # floating-point rows of odd widths (points with appended statistics) quantised and projected
        dict(name="quantize_linear_18501_131_387", op="quantize_linear", rows=18501, inputs=131, outputs=387, dtype="bf16"),
        # streaming: one new token for each of 512 tracks
        dict(name="step_512x1024_bf16", op="step", rows=512, channels=1024, dtype="bf16"),
        # a whole scan as one sequence per batch entry, walked backwards
        dict(name="scan_463k_64_bf16", op="scan", rows=463001, channels=64, seqs=2, dtype="bf16", reverse=True),
        # fine-tuning over groups of a few hundred voxels, empty and single ones among them
        dict(name="scan_train_120k_128_fp16", op="scan_train", rows=120000, channels=128, seqs=400, dtype="fp16",
             reverse=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A number of channels: mostly multiples of 16, one in three any number."""
    w = _log_int(rng, low, high)
    return w if rng.random() < 0.34 else max(16, w // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "norm_train", "norm_linear", "linear", "linear", "quantize_linear", "step", "scan", "scan_train"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if op in ("norm", "norm_train"):
        channels = _width(rng, 16, 8192)
        c = dict(op=op, rows=_log_int(rng, 1, min(463001, (1 << 25) // channels)), channels=channels, dtype=dtype)
        return dict(c, residual=rng.random() < 0.5) if op == "norm" else c
    if op in ("norm_linear", "linear", "quantize_linear"):
        inputs, outputs = _width(rng, 16, 4096), _width(rng, 16, 8192)
        most = min(463001, (1 << 26) // max(inputs, outputs), (1 << 37) // (inputs * outputs))
        c = dict(op=op, rows=_log_int(rng, 1, most), inputs=inputs, outputs=outputs, dtype=dtype)
        if op != "norm_linear":
            return c
        # a norm in 32 bits leaves a value next to the border of two 8-bit steps on either side of it, which shows in
        # results of 32 bits: half-precision features, which is what is deployed in 8 bits
        return dict(c, dtype=dtype if dtype != "fp32" else "fp16", residual=rng.random() < 0.5)
    if op == "step":
        channels = _width(rng, 16, 4096)
        return dict(op=op, rows=_log_int(rng, 1, min(65536, (1 << 24) // channels)), channels=channels, dtype=dtype)
    channels = _width(rng, 16, 1024)
    rows = _log_int(rng, 1, min(463001, (1 << 24) // channels))
    return dict(op=op, rows=rows, channels=channels, seqs=_log_int(rng, 1, min(rows, 4096)), dtype=dtype,
                reverse=rng.random() < 0.5)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    def features(rows, channels):
        """Rows of different scale, channels of different mean."""
        scale = torch.exp(0.5 * normal(rows, 1))
        return (normal(rows, channels) * scale + 0.3 * normal(1, channels)).to(dtype)

    def norm_parameters(channels):
        return 1.0 + 0.2 * normal(channels), 0.1 * normal(channels)

    def layer(inputs, outputs):
        """8-bit weights, a scale per output channel, bias."""
        w = normal(outputs, inputs)
        scale = w.abs().amax(1) / 127
        q = torch.round(w / scale[:, None]).to(torch.int8)
        return q, scale / math.sqrt(inputs), 0.1 * normal(outputs)

    s = dict(op=op, dtype=dtype)
    if op in ("norm", "norm_train"):
        s["x"] = features(case["rows"], case["channels"])
        s["weight"], s["bias"] = norm_parameters(case["channels"])
        if op == "norm_train":
            s["grad"] = normal(case["rows"], case["channels"]).to(dtype)
        s["residual"] = features(case["rows"], case["channels"]) if case.get("residual") else None
    elif op in ("norm_linear", "quantize_linear"):
        s["x"] = features(case["rows"], case["inputs"])
        s["residual"] = features(case["rows"], case["inputs"]) if case.get("residual") else None
        if op == "norm_linear":
            s["weight"], s["bias"] = norm_parameters(case["inputs"])
        s["q_weight"], s["q_scale"], s["q_bias"] = layer(case["inputs"], case["outputs"])
    elif op == "linear":  # rows as a quantiser leaves them: the largest magnitude of each is 127
        x = normal(case["rows"], case["inputs"])
        scale = x.abs().amax(1) / 127
        s["x"], s["x_scale"] = torch.round(x / scale[:, None]).to(torch.int8), scale
        s["q_weight"], s["q_scale"], s["q_bias"] = layer(case["inputs"], case["outputs"])
    else:
        rows, channels = case["rows"], case["channels"]
        s["x"] = features(rows, channels)
        # channels from short memory to long: mean gate 0 (half of the state is kept) to 6 (99.75 %)
        s["gate"] = (normal(rows, channels) + torch.linspace(0, 6, channels, device=DEV)).to(dtype)
        if op == "step":
            s["initial"] = normal(rows, channels)
        else:
            seqs = case["seqs"]
            cuts = torch.randint(0, rows + 1, (seqs - 1,), generator=gen, device=DEV).sort().values
            ends = torch.tensor([0, rows], device=DEV)
            s["offsets"] = torch.cat([ends[:1], cuts, ends[1:]]).int()
            s["initial"] = normal(seqs, channels)
            s["reverse"] = case["reverse"]
            if op == "scan_train":
                s["grad"] = normal(rows, channels).to(dtype)
                s["grad_final"] = normal(seqs, channels)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _norm(x, weight, bias):
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    hat = centred * rstd
    return hat * weight + bias, hat, rstd


def _quantize(x):
    """Rows in steps of the 127th part of their largest magnitude; the quotient in 64 bits, so that a value next to the
    border of two steps goes to the right one."""
    scale = x.abs().amax(1) / 127
    return torch.round(x.double() / scale.double()[:, None]).nan_to_num().float(), scale


def _linear(q, scale, s):
    acc = q @ s["q_weight"].float().T
    return (acc * scale[:, None] * s["q_scale"] + s["q_bias"]).to(s["dtype"])


def _starts(offsets, rows, reverse):
    """For rows in the order they are walked in: whether a sequence starts, and which one the row belongs to."""
    order = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(offsets[1:].contiguous(), order.int(), right=True)
    if reverse:
        seq = seq.flip(0)
    first = torch.ones(rows, dtype=torch.bool, device=DEV)
    first[1:] = seq[1:] != seq[:-1]
    return first, seq


def _walk(a, b):
    """h[t] = a[t] h[t-1] + b[t], h[-1] = 0, by doubling: after the pass of distance d every row holds its last 2 d terms."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _scan(s):
    """Plain recurrence, forward and, where there are gradients, backward."""
    rows = s["x"].shape[0]
    turn = (lambda t: t.flip(0)) if s["reverse"] else (lambda t: t)
    x, gate = turn(s["x"].float()), turn(s["gate"].float())
    keep, add = torch.sigmoid(gate), torch.sigmoid(-gate)
    first, seq = _starts(s["offsets"], rows, s["reverse"])
    first, initial = first[:, None], s["initial"]
    zero = torch.zeros((), device=DEV)
    h = _walk(torch.where(first, zero, keep), add * x + torch.where(first, keep * initial[seq], zero))
    last = torch.ones_like(first)
    last[:-1] = first[1:]
    final = initial.clone()  # a sequence without rows ends where it starts
    at = last[:, 0].nonzero()[:, 0]
    final[seq[at]] = h[at]
    outs = (turn(h).to(s["dtype"]), final)
    if "grad" not in s:
        return outs
    # delta[t] = grad[t] + f[t+1] delta[t+1], walked from the last row of each sequence to the first
    back = lambda t: t.flip(0)
    ahead = torch.cat([keep[1:], keep[:1]])
    grad = turn(s["grad"].float()) + torch.where(last, s["grad_final"][seq], zero)
    delta = back(_walk(back(torch.where(last, zero, ahead)), back(grad)))
    before = torch.where(first, initial[seq], torch.cat([h[:1], h[:-1]]))
    grad_x = turn(delta * add).to(s["dtype"])
    grad_gate = turn(delta * (before - x) * keep * add).to(s["dtype"])
    grad_initial = s["grad_final"].clone()
    at = first[:, 0].nonzero()[:, 0]
    grad_initial[seq[at]] = (keep * delta)[at]
    return outs + (grad_x, grad_gate, grad_initial)


def _plain(s):
    op, dtype = s["op"], s["dtype"]
    if op == "norm":
        if s["residual"] is None:
            return _norm(s["x"].float(), s["weight"], s["bias"])[0].to(dtype)
        total = (s["x"].float() + s["residual"].float()).to(dtype)
        return _norm(total.float(), s["weight"], s["bias"])[0].to(dtype), total
    if op == "norm_train":
        y, hat, rstd = _norm(s["x"].float(), s["weight"], s["bias"])
        grad = s["grad"].float()
        g = grad * s["weight"]
        dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        return (y.to(dtype), dx.to(dtype), (grad * hat).sum(0, dtype=torch.float64).float(),
                grad.sum(0, dtype=torch.float64).float())
    if op == "norm_linear":
        total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(dtype)
        y = _linear(*_quantize(_norm(total.float(), s["weight"], s["bias"])[0]), s)
        return y if s["residual"] is None else (y, total)
    if op == "quantize_linear":
        return _linear(*_quantize(s["x"].float()), s)
    if op == "linear":
        return _linear(s["x"].float(), s["x_scale"], s)
    if op == "step":
        gate = s["gate"].float()
        h = torch.sigmoid(gate) * s["initial"] + torch.sigmoid(-gate) * s["x"].float()
        return h.to(dtype), h
    return _scan(s)


# ---- the package's operators ----------------------------------------------------------------------------------------
def _own(s):
    from deploy3d_b200 import ops
    op, dtype = s["op"], s["dtype"]
    if op == "norm":
        return ops.layer_norm(s["x"], s["weight"], s["bias"], EPS, residual=s["residual"])
    if op == "norm_train":
        y, mean, rstd = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS, with_stats=True)
        return (y,) + ops.layer_norm_backward(s["grad"], s["x"], s["weight"], mean, rstd)
    if op == "norm_linear":
        q = ops.layer_norm_int8(s["x"], s["weight"], s["bias"], EPS, residual=s["residual"])
        y = ops.int8_linear(q[0], q[1], s["q_weight"], s["q_scale"], s["q_bias"], dtype=dtype)
        return y if s["residual"] is None else (y, q[2])
    if op == "quantize_linear":
        q, scale = ops.quantize_rows(s["x"])
        return ops.int8_linear(q, scale, s["q_weight"], s["q_scale"], s["q_bias"], dtype=dtype)
    if op == "linear":
        return ops.int8_linear(s["x"], s["x_scale"], s["q_weight"], s["q_scale"], s["q_bias"], dtype=dtype)
    if op == "step":
        return ops.gated_recurrence_step(s["x"], s["gate"], s["initial"])
    if op == "scan":
        return ops.gated_recurrence(s["x"], s["gate"], s["offsets"], s["initial"], reverse=s["reverse"])
    out, final, states = ops.gated_recurrence(s["x"], s["gate"], s["offsets"], s["initial"], reverse=s["reverse"],
                                              with_states=True)
    return (out, final) + ops.gated_recurrence_backward(s["grad"], s["x"], s["gate"], s["offsets"], states, s["initial"],
                                                        grad_final=s["grad_final"], reverse=s["reverse"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    """Every input read once, every output written once; a multiply-add is two operations."""
    e, op = ESIZE[case["dtype"]], case["op"]
    if op == "norm":
        n = case["rows"] * case["channels"]
        return {"bytes": n * e * (4 if case["residual"] else 2) + 8 * case["channels"], "flops": 8 * n}
    if op == "norm_train":
        n = case["rows"] * case["channels"]
        return {"bytes": n * e * 4 + 16 * case["channels"], "flops": 22 * n}
    if op in ("norm_linear", "quantize_linear", "linear"):
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        read = m * k + 4 * m if op == "linear" else m * k * e * (3 if case.get("residual") else 1)
        return {"bytes": read + n * k + 8 * n + m * n * e, "flops": 2 * m * n * k}
    n = case["rows"] * case["channels"]
    if op == "step":
        return {"bytes": n * (3 * e + 8), "flops": 10 * n}
    ends = 4 * case["seqs"] * case["channels"]
    return {"bytes": n * e * (3 if op == "scan" else 6) + ends * (2 if op == "scan" else 4),
            "flops": (10 if op == "scan" else 30) * n}


def exact(case, seed):
    """The definition in 64 bits, from the same inputs."""
    s = prepare(case, seed)
    op, f64 = s["op"], torch.float64
    v = {k: t.to(f64) for k, t in s.items() if torch.is_tensor(t) and k != "offsets"}

    def norm(x):
        mean = x.sum(1, keepdim=True) / x.shape[1]
        var = (x - mean).square().sum(1, keepdim=True) / x.shape[1]
        return mean, (var + EPS).rsqrt()

    def product(q, scale):
        return torch.addmm(v["q_bias"], q * scale, (v["q_weight"] * v["q_scale"][:, None]).T)

    def steps(x):
        scale = (x.abs().amax(1, keepdim=True).float() / 127).to(f64)  # the scale itself is held in 32 bits
        return (x / scale).round().nan_to_num(), scale

    def summed():
        return s["x"].to(f64) if s["residual"] is None else (v["x"] + v["residual"]).to(s["dtype"]).to(f64)

    if op in ("norm", "norm_linear"):
        x = summed()
        mean, rstd = norm(x)
        y = (x - mean) * rstd * v["weight"] + v["bias"]
        if op == "norm_linear":
            y = product(*steps(y))
        return y if s["residual"] is None else (y, x)
    if op == "norm_train":
        x, n = v["x"], case["channels"]
        mean, rstd = norm(x)
        dy = v["grad"] * v["weight"]
        # dx = J dy with J = rstd (1 - 1/n - (x - mean)(x - mean)^T rstd^2 / n)
        along = ((x - mean) * dy).sum(1, keepdim=True)
        dx = rstd * dy - rstd * dy.sum(1, keepdim=True) / n - rstd ** 3 * along * (x - mean) / n
        return ((x - mean) * rstd * v["weight"] + v["bias"], dx, (v["grad"] * (x - mean) * rstd).sum(0), v["grad"].sum(0))
    if op == "quantize_linear":
        return product(*steps(v["x"]))
    if op == "linear":
        return product(v["x"], v["x_scale"][:, None])
    if op == "step":
        f = 1 / (1 + (-v["gate"]).exp())
        h = f * v["initial"] + (1 - f) * v["x"]
        return h, h

    # the recurrence: blocks of rows walked side by side one row at a time, then their ends, then the ends brought in
    rows, channels, seqs = case["rows"], case["channels"], case["seqs"]
    offsets = s["offsets"].tolist()
    begins = [offsets[i] for i in range(seqs) if offsets[i + 1] > offsets[i]]
    ends = [offsets[i + 1] - 1 for i in range(seqs) if offsets[i + 1] > offsets[i]]
    filled = [i for i in range(seqs) if offsets[i + 1] > offsets[i]]
    if s["reverse"]:
        begins, ends = ends, begins
    begins, ends, filled = (torch.tensor(t, device=DEV) for t in (begins, ends, filled))
    f = 1 / (1 + (-v["gate"]).exp())

    def walk(a, b, backwards):
        if backwards:
            a, b = a.flip(0), b.flip(0)
        block = max(1, int(math.sqrt(rows)))
        many = (rows + block - 1) // block
        pad = (0, 0, 0, many * block - rows)
        a = torch.nn.functional.pad(a, pad).view(many, block, channels).clone()
        b = torch.nn.functional.pad(b, pad).view(many, block, channels).clone()
        for t in range(1, block):
            b[:, t] += a[:, t] * b[:, t - 1]
            a[:, t] *= a[:, t - 1]
        carry = torch.zeros((many, channels), dtype=f64, device=DEV)
        for t in range(1, many):
            carry[t] = a[t - 1, -1] * carry[t - 1] + b[t - 1, -1]
        h = (b + a * carry[:, None]).view(-1, channels)[:rows]
        return h.flip(0) if backwards else h

    a, b = f.clone(), (1 - f) * v["x"]
    b[begins] += f[begins] * v["initial"][filled]
    a[begins] = 0
    h = walk(a, b, s["reverse"])
    final = v["initial"].clone()
    final[filled] = h[ends]
    if op == "scan":
        return h, final
    before = torch.empty_like(h)
    before[1:], before[:1] = h[:-1], h[:1]
    after = torch.empty_like(f)
    after[:-1], after[-1:] = f[1:], f[-1:]
    if s["reverse"]:
        before[:-1], before[-1:] = h[1:], h[-1:]
        after[1:], after[:1] = f[:-1], f[:1]
    before[begins] = v["initial"][filled]
    after[ends] = 0
    g = v["grad"].clone()
    g[ends] += v["grad_final"][filled]
    delta = walk(after, g, not s["reverse"])
    grad_initial = v["grad_final"].clone()
    grad_initial[filled] = f[begins] * delta[begins]
    return h, final, delta * (1 - f), delta * (before - v["x"]) * f * (1 - f), grad_initial
