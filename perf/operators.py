"""Performance cases of the recurrence, 4-bit projection and optimiser operators.

Three operators around a mixer's projections are measured here, each as a user calls it:

* ``gated_scan`` / ``gated_step``: the elementwise gated linear recurrence, whole sequences (forward,
  and forward with all gradients) and one decoded token;
* ``linear_w4``: a projection of a few rows with 4-bit weights and group scales;
* ``orthogonalize``: the Newton-Schulz orthogonalisation of an optimiser update.

``run`` computes each either in its plain form (elementary torch operations in 32 bits, rounded once
at the end) or, with ``own`` set, through the package's kernels. ``exact`` is the operator's
definition in 64 bits. Sizes are those of ``Mamba3`` models with d_model 256, 768, 1024 and 2560:
recurrence widths 2 * d_model, in_proj weights [10768, 2560] (d_model 2560) and [1336, 256]
(d_model 256), out_proj weights [d_model, 2 * d_model], decode batches 1, 4, 64 and 256.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

#: a, b, c of x' = a x + b (x x^T) x + c (x x^T)^2 x
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_STEPS = 5


def listed():
    return [
        # one decoded token of one sequence, d_model 2560: all latency
        dict(name="step, 1 sequence", op="step", batch=1, channels=5120, dtype="bf16", gate=True),
        # the largest decode batch: the state is read and written once
        dict(name="step, 256 sequences", op="step", batch=256, channels=5120, dtype="bf16", gate=True),
        # a ragged evaluation batch in full precision: odd length and width, document boundaries, no gate
        dict(name="scan, odd sizes", op="scan", batch=3, length=777, channels=1001, dtype="fp32", gate=False, reset=True),
        # prefill of 8 sequences, d_model 1024, columns of one projection
        dict(name="scan, prefill", op="scan", batch=8, length=8192, channels=2048, dtype="bf16", gate=True, reset=False),
        # prefill of one long sequence, d_model 768: parallel over time or not at all
        dict(name="scan, one long sequence", op="scan", batch=1, length=65536, channels=1536, dtype="bf16", gate=True,
             reset=False),
        # a training step of packed documents, d_model 1024: outputs and every gradient
        dict(name="scan, training", op="train", batch=4, length=2048, channels=2048, dtype="bf16", gate=True, reset=True),
        # in_proj of one decoded token, d_model 2560: a stream of weights
        dict(name="w4, in_proj, 1 row", op="w4", rows=1, out_dim=10768, in_dim=2560, group=128, zeros=False, dtype="bf16"),
        # out_proj of four decoded sequences, zero points
        dict(name="w4, out_proj, 4 rows", op="w4", rows=4, out_dim=2560, in_dim=5120, group=64, zeros=True, dtype="fp16"),
        # in_proj at decode batch 64: the same weights, 64 times the products
        dict(name="w4, in_proj, 64 rows", op="w4", rows=64, out_dim=10768, in_dim=2560, group=128, zeros=False,
             dtype="bf16"),
        # a small model with sizes that divide by nothing
        dict(name="w4, odd sizes", op="w4", rows=3, out_dim=1337, in_dim=517, group=32, zeros=True, dtype="fp16"),
        # in_proj updates of a four-layer model, d_model 256, as one stack
        dict(name="orthogonalize, 4 small", op="orth", count=4, rows=1336, cols=256, dtype="fp32"),
        # the in_proj update of one layer, d_model 2560
        dict(name="orthogonalize, large", op="orth", count=1, rows=10768, cols=2560, dtype="bf16"),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], evenly spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "train", "w4", "w4", "orth"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "step":
        return dict(op="step", batch=_between(rng, 1, 256), channels=_between(rng, 64, 5120), dtype=dtype,
                    gate=rng.random() < 0.7)
    if kind in ("scan", "train"):
        most = 8 * 8192 * 2048 if kind == "scan" else 4 * 4096 * 2048  # values of one input
        channels = _between(rng, 64, 5120)
        if rng.random() < 0.6:
            channels = (channels + 63) // 64 * 64
        length = min(_between(rng, 1, 65536 if kind == "scan" else 16384), most // channels)
        batch = min(_between(rng, 1, 16), max(1, most // (channels * length)))
        return dict(op=kind, batch=batch, length=length, channels=channels, dtype=dtype, gate=rng.random() < 0.7,
                    reset=rng.random() < 0.4)
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        in_dim, out_dim = _between(rng, 128, 8192), _between(rng, 128, 10768)
        if rng.random() < 0.75:
            in_dim = (in_dim + group - 1) // group * group
        return dict(op="w4", rows=_between(rng, 1, 64), out_dim=out_dim, in_dim=in_dim, group=group,
                    zeros=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))
    rows, cols = _between(rng, 64, 10768), _between(rng, 64, 2560)
    if rng.random() < 0.5:
        rows, cols = cols, rows
    count = min(_between(rng, 1, 16), max(1, 10768 * 2560 // (rows * cols)))
    return dict(op="orth", count=count, rows=rows, cols=cols, dtype=dtype)


# ---- inputs ------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"case": case, "op": case["op"]}
    dtype = _TYPES[case["dtype"]]
    if case["op"] in ("step", "scan", "train"):
        batch, channels = case["batch"], case["channels"]
        lead = (batch,) if case["op"] == "step" else (batch, case["length"])
        parts = 3 if case["gate"] else 2
        # columns of one projection, as a mixer has them
        projected = normal(*lead, parts * channels).to(dtype)
        # forget logits around +3, some channels short and some very long: decays of 0.3 to 0.9995
        shift = torch.empty(channels, device="cuda").uniform_(-1.0, 6.0, generator=g)
        projected[..., channels:2 * channels] += shift.to(dtype)
        s["value"], s["forget"] = projected[..., :channels], projected[..., channels:2 * channels]
        s["gate"] = projected[..., 2 * channels:] if case["gate"] else None
        s["state"] = normal(batch, channels)
        if case["op"] != "step":
            # documents of 500 tokens on average
            s["reset"] = (torch.rand(*lead, device="cuda", generator=g) < 0.002) if case["reset"] else None
        if case["op"] == "train":
            s["dy"] = (normal(*lead, channels) * 0.1).to(dtype)
            s["dstate"] = normal(batch, channels) * 0.1
    elif case["op"] == "w4":
        out_dim, in_dim, group = case["out_dim"], case["in_dim"], case["group"]
        groups = -(-in_dim // group)
        s["x"] = normal(case["rows"], in_dim).to(dtype)
        s["codes"] = torch.randint(0, 256, (out_dim, (in_dim + 1) // 2), device="cuda", generator=g, dtype=torch.uint8)
        if in_dim % 2:
            s["codes"][:, -1] &= 15  # the high half of a row's last byte stands for nothing
        s["scales"] = ((0.5 + torch.rand(out_dim, groups, device="cuda", generator=g)) * (0.4 / in_dim ** 0.5)).to(dtype)
        s["zeros"] = None
        if case["zeros"]:
            s["zeros"] = torch.randint(5, 11, (out_dim, groups), device="cuda", generator=g).to(dtype)
    else:
        count, rows, cols = case["count"], case["rows"], case["cols"]
        # momentum of a matrix in training: a few strong directions over noise
        rank = max(1, min(rows, cols) // 64)
        strong = normal(count, rows, rank) * torch.logspace(0.0, -1.0, rank, device="cuda")
        s["update"] = (1e-3 * (normal(count, rows, cols) + 2.0 * strong @ normal(count, rank, cols))).to(dtype)
    return s


# ---- plain forms -------------------------------------------------------------------------------


def _scan(decay, inputs):
    """h_t = decay_t h_{t-1} + inputs_t along dimension 1 from h = 0, and the products of the decays
    up to t: neighbours at distances 1, 2, 4, ... joined."""
    length, distance = decay.shape[1], 1
    while distance < length:
        inputs = torch.cat((inputs[:, :distance], inputs[:, distance:] + decay[:, distance:] * inputs[:, :-distance]), 1)
        decay = torch.cat((decay[:, :distance], decay[:, distance:] * decay[:, :-distance]), 1)
        distance *= 2
    return inputs, decay


def _plain_forward(s):
    value, keep = s["value"].float(), torch.sigmoid(s["forget"].float())
    carry = keep
    if s["reset"] is not None:
        carry = keep * (~s["reset"])[..., None].float()
    local, reach = _scan(carry, torch.sigmoid(-s["forget"].float()) * value)
    h = local + reach * s["state"][:, None]
    y = h
    if s["gate"] is not None:
        gate = s["gate"].float()
        y = h * (gate * torch.sigmoid(gate))
    return h, y, keep, carry


def _plain_scan(s):
    h, y, _, _ = _plain_forward(s)
    return {"y": y.to(s["value"].dtype), "state": h[:, -1]}


def _plain_train(s):
    h, y, keep, carry = _plain_forward(s)
    dtype, value = s["value"].dtype, s["value"].float()
    dy = s["dy"].float()
    out = {"y": y.to(dtype), "state": h[:, -1]}
    dh = dy
    if s["gate"] is not None:
        gate = s["gate"].float()
        sig = torch.sigmoid(gate)
        out["dgate"] = (dy * h * (sig * (1.0 + gate * (1.0 - sig)))).to(dtype)
        dh = dy * (gate * sig)
    dh = torch.cat((dh[:, :-1], dh[:, -1:] + s["dstate"][:, None]), 1)
    # the total gradient of h_t: the same recurrence from the back, with the decay of the token after
    after = torch.cat((carry[:, 1:], torch.zeros_like(carry[:, :1])), 1)
    total = _scan(after.flip(1), dh.flip(1))[0].flip(1)
    before = torch.cat((s["state"][:, None], h[:, :-1]), 1)
    if s["reset"] is not None:
        before = before * (~s["reset"])[..., None].float()
    lose = torch.sigmoid(-s["forget"].float())
    out["dvalue"] = (total * lose).to(dtype)
    out["dforget"] = (total * (before - value) * (keep * lose)).to(dtype)
    out["dstate"] = carry[:, 0] * total[:, 0]
    return out


def _plain_step(s):
    forget = s["forget"].float()
    h = torch.sigmoid(forget) * s["state"] + torch.sigmoid(-forget) * s["value"].float()
    y = h
    if s["gate"] is not None:
        gate = s["gate"].float()
        y = h * (gate * torch.sigmoid(gate))
    return {"y": y.to(s["value"].dtype), "state": h}


def _plain_w4(s):
    in_dim, group = s["case"]["in_dim"], s["case"]["group"]
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(1)[:, :in_dim].float()
    scales = s["scales"].float().repeat_interleave(group, 1)[:, :in_dim]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, 1)[:, :in_dim]
    return (s["x"].float() @ ((codes - zeros) * scales).t()).to(s["x"].dtype)


def _newton_schulz(x):
    a, b, c = _COEFFICIENTS
    gram = x @ x.mT
    return a * x + (b * gram + c * (gram @ gram)) @ x


def _plain_orthogonalize(s):
    x = s["update"].float()
    wide = x.shape[-1] >= x.shape[-2]
    x = x if wide else x.mT
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(1e-20)
    for _ in range(_STEPS):
        x = _newton_schulz(x)
    return (x if wide else x.mT).contiguous().to(torch.bfloat16)


def run(s):
    op = s["op"]
    if own:
        from mamba3_b200 import gated_scan, gated_step, linear_w4, orthogonalize

        if op == "step":
            y, state = gated_step(s["value"], s["forget"], s["state"], s["gate"])
            return {"y": y, "state": state}
        if op == "scan":
            y, state = gated_scan(s["value"], s["forget"], s["gate"], initial_state=s["state"], reset=s["reset"])
            return {"y": y, "state": state}
        if op == "train":
            names = ["value", "forget", "state"] + ([] if s["gate"] is None else ["gate"])
            leaves = {name: s[name].detach().requires_grad_() for name in names}
            y, state = gated_scan(leaves["value"], leaves["forget"], leaves.get("gate"), initial_state=leaves["state"],
                                  reset=s["reset"])
            grads = torch.autograd.grad((y, state), list(leaves.values()), (s["dy"], s["dstate"]))
            return {"y": y, "state": state, **{"d" + name: grad for name, grad in zip(names, grads)}}
        if op == "w4":
            return linear_w4(s["x"], s["codes"], s["scales"], s["zeros"], group_size=s["case"]["group"])
        return orthogonalize(s["update"], steps=_STEPS, coefficients=_COEFFICIENTS)
    return {"step": _plain_step, "scan": _plain_scan, "train": _plain_train, "w4": _plain_w4,
            "orth": _plain_orthogonalize}[op](s)


def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "step":
        n = case["batch"] * case["channels"]
        tensors = 4 if case["gate"] else 3
        return {"bytes": n * (tensors * size + 8), "flops": n * (18 if case["gate"] else 10)}
    if op in ("scan", "train"):
        rows, tensors = case["batch"] * case["length"], 4 if case["gate"] else 3
        n, ends = rows * case["channels"], 8 * case["batch"] * case["channels"]
        if op == "train":  # dy read, a gradient for each input written
            tensors += tensors
            ends *= 2
        flops = n * (18 if case["gate"] else 10) * (3 if op == "train" else 1)
        return {"bytes": n * tensors * size + ends + (rows if case["reset"] else 0), "flops": flops}
    if op == "w4":
        rows, o, i = case["rows"], case["out_dim"], case["in_dim"]
        groups = -(-i // case["group"]) * (2 if case["zeros"] else 1)
        return {"bytes": o * ((i + 1) // 2) + o * groups * size + rows * (o + i) * size, "flops": 2 * rows * o * i}
    count, m, n = case["count"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # each step: the two symmetric products (half of each) and the full one
    flops = _STEPS * (m * m * n + m * m * m + 2 * m * m * n)
    return {"bytes": count * m * n * (size + 2), "flops": count * flops}


# ---- definitions in 64 bits --------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "w4":
        codes = s["codes"].to(torch.int64)
        index = torch.arange(case["in_dim"], device="cuda")
        q = torch.where(index % 2 == 0, codes[:, index // 2] % 16, codes[:, index // 2] // 16).double()
        column = index // case["group"]
        zero = s["zeros"].double()[:, column] if s["zeros"] is not None else 8.0
        weight = s["scales"].double()[:, column] * (q - zero)
        return torch.einsum("ri,oi->ro", s["x"].double(), weight)
    if op == "orth":
        a, b, c = _COEFFICIENTS
        x = s["update"].double()
        x = x / torch.linalg.matrix_norm(x)[:, None, None]
        for _ in range(_STEPS):
            if case["rows"] >= case["cols"]:  # Horner's form on the narrow side
                gram = torch.einsum("bij,bik->bjk", x, x)
                x = a * x + torch.bmm(b * x + c * torch.bmm(x, gram), gram)
            else:
                gram = torch.einsum("bij,bkj->bik", x, x)
                x = a * x + torch.bmm(gram, b * x + c * torch.bmm(gram, x))
        return x

    def logistic(t):
        return 1.0 / (1.0 + torch.exp(-t))

    if op == "step":
        keep = logistic(s["forget"].double())
        h = s["state"].double() + (1.0 - keep) * (s["value"].double() - s["state"].double())
        y = h if s["gate"] is None else h * s["gate"].double() * logistic(s["gate"].double())
        return {"y": y, "state": h}
    if case["batch"] * case["length"] * case["channels"] > 8 * 8192 * 2048:
        return None
    length = case["length"]
    keep, gate, reset = logistic(s["forget"].double()), s["gate"], s["reset"]
    h, states, starts = s["state"].double(), [], []
    for t in range(length):  # one token after another
        if reset is not None:
            h = torch.where(reset[:, t, None], torch.zeros_like(h), h)
        if op == "train":
            starts.append(h)
        h = keep[:, t] * h + (1.0 - keep[:, t]) * s["value"][:, t]
        states.append(h)
    states = torch.stack(states, 1)
    out = {"y": states, "state": h}
    if gate is not None:
        gate = gate.double()
        out["y"] = states * gate * logistic(gate)
    if op == "train":
        dy = s["dy"].double()
        if gate is not None:
            slope = logistic(gate) + gate * logistic(gate) * logistic(-gate)
            out["dgate"], dy = dy * states * slope, dy * gate * logistic(gate)
        total, dvalue, dforget = s["dstate"].double(), [None] * length, [None] * length
        for t in reversed(range(length)):
            total = total + dy[:, t]
            dvalue[t] = total * (1.0 - keep[:, t])
            dforget[t] = total * (starts[t] - s["value"][:, t].double()) * keep[:, t] * (1.0 - keep[:, t])
            total = total * keep[:, t]
            if reset is not None:
                total = torch.where(reset[:, t, None], torch.zeros_like(total), total)
        out["dvalue"], out["dforget"], out["dstate"] = torch.stack(dvalue, 1), torch.stack(dforget, 1), total
    return out
