"""Cases of the training operators: the AdamW step over many tensors (ictc_o3.optim) and the
norms before and after a block with its gate and residual scale (ictc_o3.ops.block_norm).

``own`` selects the framework's calls; otherwise the same mathematics in elementary torch
operations.
"""
import math
import os
import random
import sys

import torch

own = False

# The package root is a folder whose name is no module name: as the README says, on the path.
sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ictc-o3-hp-ascend_b200"))

DEVICE = "cuda"
BLOCK = 256                       # values that share one scale of an 8-bit state
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
AVERAGE = 0.99                    # decay of the weight average
STEP = 137                        # steps behind the state that a pass starts from
NORM_EPS = 1e-6


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One step over the weights of a C8/lmax-2 potential (42 small tensors): launch latency.
        {"name": "adamw32 C8/L2 weights", "op": "adamw", "bits": 32, "channels": 8, "lmax": 2, "clip": False,
         "average": False},
        # C64/lmax-2 potential with clipping and the weight average, as a trainer runs it.
        {"name": "adamw32 C64/L2 clip+avg", "op": "adamw", "bits": 32, "channels": 64, "lmax": 2, "clip": True,
         "average": True},
        # The C128/lmax-3 potential of the force-loss training step, with clipping.
        {"name": "adamw32 C128/L3 clip", "op": "adamw", "bits": 32, "channels": 128, "lmax": 3, "clip": True,
         "average": False},
        # Many odd-sized tensors, far above the cache: bandwidth.
        {"name": "adamw32 160M values", "op": "adamw", "bits": 32, "total": 160_000_000, "tensors": 230,
         "shapes": 11, "clip": True, "average": True},
        # The same potential with states in 8 bits.
        {"name": "adamw8 C128/L3", "op": "adamw", "bits": 8, "channels": 128, "lmax": 3, "clip": False,
         "average": False},
        # 8-bit states where they matter: large totals.
        {"name": "adamw8 160M values", "op": "adamw", "bits": 8, "total": 160_000_000, "tensors": 230, "shapes": 12,
         "clip": True, "average": False},
        # End of a block for one small cell (40 atoms): latency.
        {"name": "block fwd 40 C32/L2", "op": "block", "run": "forward", "rows": 40, "channels": 32, "lmax": 2,
         "layout": "mul_ir", "gate": True, "pre": True},
        # Molecular dynamics of 262,144 atoms at C64/lmax 2: inference, no gradients.
        {"name": "block fwd 262144 C64/L2", "op": "block", "run": "forward", "rows": 262144, "channels": 64,
         "lmax": 2, "layout": "mul_ir", "gate": True, "pre": True},
        # First norm of a stack, with its gradients, 16,384 atoms at C64/lmax 2.
        {"name": "norm train 16384 C64/L2", "op": "norm", "run": "train", "rows": 16384, "channels": 64, "lmax": 2,
         "layout": "mul_ir", "gate": False, "pre": True},
        # Forces of the training batch (4 x 2,048 atoms, C128/lmax 3): forward and first gradients.
        {"name": "block train 8192 C128/L3", "op": "block", "run": "train", "rows": 8192, "channels": 128, "lmax": 3,
         "layout": "mul_ir", "gate": True, "pre": True},
        # The force loss of the same batch differentiates those gradients.
        {"name": "block force 8192 C128/L3", "op": "block", "run": "force", "rows": 8192, "channels": 128, "lmax": 3,
         "layout": "mul_ir", "gate": True, "pre": True},
        # Odd channels and rows, the operators' other layout, no gate.
        {"name": "block force 10007 C50/L1", "op": "block", "run": "force", "rows": 10007, "channels": 50, "lmax": 1,
         "layout": "ir_mul", "gate": False, "pre": True},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        case = {"op": "adamw", "bits": rng.choice((8, 32)), "clip": rng.random() < 0.5,
                "average": rng.random() < 0.3}
        if rng.random() < 0.3:
            case |= {"channels": _between(rng, 5, 160), "lmax": rng.randint(1, 3)}
        else:
            tensors = _between(rng, 1, 300)
            case |= {"total": max(tensors, _between(rng, 1000, 80_000_000)), "tensors": tensors,
                     "shapes": rng.randrange(1 << 20)}
        return case
    lmax = rng.randint(0, 3)
    channels = rng.choice((_between(rng, 3, 260), 4 * _between(rng, 1, 65)))
    values = _between(rng, 2000, 16_000_000)
    op = "norm" if rng.random() < 0.2 else "block"
    return {"op": op, "run": rng.choice(("forward", "train", "force")),
            "rows": max(1, values // (channels * (lmax + 1) ** 2)), "channels": channels, "lmax": lmax,
            "layout": rng.choice(("mul_ir", "ir_mul")), "gate": op == "block" and rng.random() < 0.6,
            "pre": op == "norm" or rng.random() < 0.8}


def _shapes(case):
    """Weight shapes of a two-layer potential of the given channels and lmax, or `tensors`
    odd sizes that add up to `total`."""
    if "total" in case:
        rng, k = random.Random(case["shapes"]), case["tensors"]
        weights = [math.exp(rng.uniform(0.0, 5.0)) for _ in range(k)]
        spare = case["total"] - k
        return [(1 + int(spare * w / sum(weights)),) for w in weights]
    c, lmax = case["channels"], case["lmax"]
    degrees = range(lmax + 1)
    paths = [(i, j, k) for i in degrees for j in degrees for k in degrees
             if abs(i - j) <= k <= i + j and (i + j + k) % 2 == 0]
    shapes = [(c, 3)]
    for layer in range(2):
        used = [p for p in paths if layer or p[0] == 0]
        shapes += [(c, c) for _ in (degrees if layer else (0,))]
        shapes += [(64, 8), (64, 64), (64, 64), (len(used) * c, 64)]
        shapes += [(c, c * sum(p[2] == l for p in used)) for l in degrees]
        shapes += [(3, 1, c, c)]
        for l in degrees if layer == 0 else (0,):
            shapes += [(3, 14 * (l + 1), c), (3, 3 + l, c), (3, 1, c)]
        shapes += [(c, c) for _ in (degrees if layer == 0 else (0,))]
    return shapes + [(1, c), (16, c), (1, 16)]


def _spans(case):
    """(start, size, shape) of every tensor in one buffer; starts are multiples of BLOCK."""
    spans, start = [], 0
    for shape in _shapes(case):
        spans.append((start, math.prod(shape), shape))
        start += -(-math.prod(shape) // BLOCK) * BLOCK
    return spans, start


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        # weights, gradients and both moments in, weights and moments out; the 8-bit moments are one
        # byte each way and come back as two-byte values; the average is read and written
        per = (28 if case["bits"] == 32 else 16 + 4) + (8 if case["average"] else 0)
        return {"bytes": per * n, "flops": 20 * n}
    row = 4 * case["channels"] * (case["lmax"] + 1) ** 2
    gate = 4 * case["channels"] * (case["lmax"] + 1) if case["gate"] else 0
    pre = int(case["pre"])
    if case["op"] == "norm":      # in: x, (q), (cotangent of dx); out: u, (dx), (its adjoints)
        rows = {"forward": 2, "train": 4, "force": 7}[case["run"]]
        gates = 0
    else:
        rows = {"forward": 3 + pre, "train": 6 + 2 * pre, "force": 11 + 3 * pre}[case["run"]]
        gates = {"forward": 1, "train": 2, "force": 4}[case["run"]]
    return {"bytes": case["rows"] * (rows * row + gates * gate), "flops": case["rows"] * rows * row}


# ---------------------------------------------------------------------------
# 8-bit states
# ---------------------------------------------------------------------------

def _decode(codes, exponents, signed):
    """Values of 8-bit codes [n]: a float whose top bits are the code, times the block's 2^(byte-127)."""
    low = (codes & 127) if signed else codes
    bits = (low.int() + (896 if signed else 768)) << 20
    value = torch.where(low == 0, 0.0, bits.view(torch.float32))
    if signed:
        value = torch.where(codes > 127, -value, value)
    scale = (exponents.int() << 23).view(torch.float32)
    return (value.view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)


def _encode(value, rand, signed):
    """(codes, exponents) of values [n] with 16-bit random numbers [n] for the rounding."""
    size = value.abs().view(-1, BLOCK)
    exponents = ((size.amax(1).view(torch.int32) >> 23) + 1).clamp(1, 253)
    size = (size * ((254 - exponents) << 23).view(torch.float32).unsqueeze(1)).view(-1)
    base, top = (896, 127) if signed else (768, 255)
    least = 1.125 * 2.0 ** (base // 8 - 127)
    code = (((size.view(torch.int32) + (rand << 4)) >> 20) - base).clamp(max=top)
    # below the least value: its share of it decides (first moment), or it stays the least (second)
    small = (rand.float() < size * (65536.0 / least)) if signed else size > 0
    code = torch.where(size < least, small.int(), code)
    if signed:
        code = code + 128 * ((value < 0) & (code > 0)).int()
    return code.to(torch.uint8), exponents.to(torch.uint8)


def _philox(quads, step, seed):
    """Philox4x32-7: [quads * 4] random 32-bit words (in int64) of counters (quad, step) and the key `seed`."""
    mask = 0xFFFFFFFF
    q = torch.arange(quads, device=DEVICE, dtype=torch.int64)
    c0, c1 = q & mask, q >> 32
    c2, c3 = torch.full_like(q, step & mask), torch.full_like(q, step >> 32)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), 1).view(-1)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _adamw_inputs(case, seed):
    """Flat buffers; every tensor's gradients have a scale of their own, the moments fit them."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    spans, size = _spans(case)
    scales = torch.exp(-8.0 * torch.rand(len(spans), device=DEVICE, generator=gen))
    lengths = torch.tensor([-(-n // BLOCK) * BLOCK for _, n, _ in spans], device=DEVICE)
    used = torch.tensor([n for _, n, _ in spans], device=DEVICE)
    starts = torch.tensor([s for s, _, _ in spans], device=DEVICE)
    scale = torch.repeat_interleave(scales, lengths)
    end = torch.repeat_interleave(starts + used, lengths)
    scale = torch.where(torch.arange(size, device=DEVICE) < end, scale, 0.0)    # nothing between the tensors
    normal = lambda: torch.randn(size, device=DEVICE, generator=gen)  # noqa: E731
    data = {"weights": 0.09 * normal() * (scale > 0), "grads": normal() * scale, "m": 0.3 * normal() * scale,
            "v": (0.2 + torch.rand(size, device=DEVICE, generator=gen)) * scale * scale}
    if case["average"]:
        data["average"] = data["weights"] * 1.01
    if case["bits"] == 8:
        for name in ("m", "v"):
            rand = torch.randint(0, 65536, (size,), device=DEVICE, generator=gen, dtype=torch.int32)
            data[name], data[name + "_exponents"] = _encode(data[name], rand, name == "m")
    # half of the gradients' norm: clipping acts
    data["max_norm"] = 0.5 * float(data["grads"].double().square().sum().sqrt()) if case["clip"] else None
    data["seed"] = 0x9E3779B97F4A7 ^ seed
    return data, spans


def _block_inputs(case, seed, dtype=torch.float32):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    n, c, lmax = case["rows"], case["channels"], case["lmax"]
    width = c * (lmax + 1) ** 2
    normal = lambda *shape: torch.randn(*shape, device=DEVICE, generator=gen)  # noqa: E731
    data = {"x": normal(n, width)}
    if case["op"] == "block":
        data["y"] = 0.3 * normal(n, width) * torch.exp(0.5 * normal(n, 1))
        data["post"] = 1.0 + 0.1 * normal(lmax + 1, c)
        data["scale"] = 0.5 + 0.1 * normal(lmax + 1, c)
    if case["gate"]:
        data["gate"] = normal(n, (lmax + 1) * c)
    if case["pre"]:
        data["pre"] = 1.0 + 0.1 * normal(lmax + 1, c)
    names = list(data)
    if case["run"] != "forward":
        data["p"] = normal(n, width) if case["op"] == "block" else None
        data["q"] = normal(n, width) if case["pre"] else None
    if case["run"] == "force":
        data |= {"d" + k: normal(*data[k].shape) for k in ("x", "y", "gate") if k in names}
    return {k: v.to(dtype) for k, v in data.items() if v is not None}


def prepare(case, seed):
    if case["op"] == "adamw":
        state, spans = _adamw_inputs(case, seed)
        state |= {"case": case, "step": STEP}
        if own:
            from ictc_o3.optim import AdamW
            weights = [torch.nn.Parameter(state["weights"][s:s + n].view(shape)) for s, n, shape in spans]
            for w, (s, n, shape) in zip(weights, spans):
                w.grad = state["grads"][s:s + n].view(shape)
            opt = AdamW(weights, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                        max_norm=state["max_norm"], ema_decay=AVERAGE if case["average"] else None,
                        seed=state["seed"])
            saved = opt.state_dict()
            for i, (s, n, shape) in enumerate(spans):
                entry = {"step": STEP}
                if case["bits"] == 32:
                    entry |= {"exp_avg": state["m"][s:s + n].view(shape), "exp_avg_sq": state["v"][s:s + n].view(shape)}
                else:
                    first, last = s // BLOCK, -(-(s + n) // BLOCK)
                    entry |= {"exp_avg": state["m"][s:s + n].view(shape), "exp_avg_sq": state["v"][s:s + n].view(shape),
                              "exp_avg_exponent": state["m_exponents"][first:last],
                              "exp_avg_sq_exponent": state["v_exponents"][first:last]}
                if case["average"]:
                    entry["ema"] = state["average"][s:s + n].view(shape)
                saved["state"][i] = entry
            opt.load_state_dict(saved)
            state = {"case": case, "opt": opt, "weights": state["weights"]}
        return state
    state = _block_inputs(case, seed)
    for name in ("x", "y", "gate", "post", "scale", "pre", "p", "q"):
        if name in state and case["run"] != "forward":
            state[name].requires_grad_(True)
    return state | {"case": case}


# ---------------------------------------------------------------------------
# Passes
# ---------------------------------------------------------------------------

def _adamw_plain(state):
    case, t = state["case"], state["step"] + 1
    w, g = state["weights"], state["grads"]
    out = []
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        out.append(norm)
    m, v = state["m"], state["v"]
    if case["bits"] == 8:
        m = _decode(m, state["m_exponents"], True)
        v = _decode(v, state["v_exponents"], False)
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    denominator = v.sqrt() * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS
    w.copy_(w * (1.0 - LR * DECAY) - (LR / (1.0 - BETA1 ** t)) * (m / denominator))
    if case["average"]:
        state["average"] = state["average"] * AVERAGE + w * (1.0 - AVERAGE)
        out.append(state["average"])
    state["step"] = t
    if case["bits"] == 8:
        words = _philox(w.numel() // 4, t, state["seed"])
        state["m"], state["m_exponents"] = _encode(m, (words & 65535).int(), True)
        state["v"], state["v_exponents"] = _encode(v, (words >> 16).int(), False)
        # four significant bits times a power of two: exact in bf16
        m = _decode(state["m"], state["m_exponents"], True).bfloat16()
        v = _decode(state["v"], state["v_exponents"], False).bfloat16()
    else:
        state["m"], state["v"] = m, v
    return [w, m, v, *out]


def _adamw_own(state):
    opt = state["opt"]
    opt.step()
    out = [state["weights"], *opt.moments()]
    if state["case"]["clip"]:
        out.append(opt.grad_norm)
    if state["case"]["average"]:
        out.append(opt.averages())
    return out


def _degrees(case, x):
    """The degree blocks of rows as [N, channels, 2l+1]."""
    c = case["channels"]
    blocks = [x[:, c * l * l:c * (l + 1) ** 2] for l in range(case["lmax"] + 1)]
    if case["layout"] == "ir_mul":
        return [b.reshape(x.shape[0], -1, c).transpose(1, 2) for b in blocks]
    return [b.reshape(x.shape[0], c, -1) for b in blocks]


def _rows(case, blocks):
    if case["layout"] == "ir_mul":
        blocks = [b.transpose(1, 2) for b in blocks]
    return torch.cat([b.reshape(b.shape[0], -1) for b in blocks], 1)


def _normed(case, x, weight):
    """x / sqrt(mean over the degree of x^2 + eps) times weight [degree, channel]."""
    return [b / (b.square().mean((1, 2), keepdim=True) + NORM_EPS).sqrt() * weight[l].unsqueeze(-1)
            for l, b in enumerate(_degrees(case, x))]


def _block_plain(state):
    case, x = state["case"], state["x"]
    if case["op"] == "norm":
        return [_rows(case, _normed(case, x, state["pre"]))]
    branch = _normed(case, state["y"], state["post"] * state["scale"])
    if case["gate"]:
        gate = 1.0 / (1.0 + torch.exp(-state["gate"].view(x.shape[0], case["lmax"] + 1, -1)))
        branch = [b * gate[:, l].unsqueeze(-1) for l, b in enumerate(branch)]
    stream = x + _rows(case, branch)
    return [stream] + ([_rows(case, _normed(case, stream, state["pre"]))] if case["pre"] else [])


def _block_own(state):
    from ictc_o3.ops.block_norm import degree_norm, residual_block_norm
    case, s = state["case"], state
    form = {"channels": case["channels"], "lmax": case["lmax"], "layout": case["layout"], "eps": NORM_EPS}
    if case["op"] == "norm":
        return [degree_norm(s["x"], s["pre"], **form)]
    stream, normed = residual_block_norm(s["x"], s["y"], post_weight=s["post"], scale=s["scale"], gate=s.get("gate"),
                                         pre_weight=s.get("pre"), **form)
    return [stream] + ([normed] if case["pre"] else [])


def _leaves(state, names):
    return [state[k] for k in names if k in state]


def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        return _adamw_own(state) if own else _adamw_plain(state)
    block = _block_own if own else _block_plain
    if case["run"] == "forward":
        with torch.no_grad():
            return block(state)
    out = block(state)
    cotangents = _leaves(state, ("p", "q"))
    if case["run"] == "train":
        grads = torch.autograd.grad(out, _leaves(state, ("x", "y", "gate", "post", "scale", "pre")), cotangents)
        return [*(o.detach() for o in out), *grads]
    # forces: gradients of the rows, then the adjoint of those gradients
    first = torch.autograd.grad(out, _leaves(state, ("x", "y", "gate")), cotangents, create_graph=True)
    second = torch.autograd.grad(first, _leaves(state, ("x", "y", "gate", "post", "scale", "pre", "p", "q")),
                                 _leaves(state, ("dx", "dy", "dgate")), allow_unused=True, materialize_grads=True)
    return [*(o.detach() for o in (*out, *first)), *second]


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _nearest_states(value, rand, signed):
    """The value that an 8-bit state stands for after rounding with 16-bit random numbers."""
    size = value.abs().view(-1, BLOCK)
    largest = size.amax(1, keepdim=True)
    scale = torch.exp2((torch.floor(torch.log2(largest.clamp(min=2.0 ** -140))) + 1).clamp(-126, 126))
    size = (size / scale).view(-1)
    least = 1.125 * 2.0 ** (-15 if signed else -31)
    grain = torch.exp2(torch.floor(torch.log2(size.clamp(min=least))) - 3)       # three fraction bits
    up = torch.floor(size / grain + rand.double() / 65536.0) * grain
    low = (rand.double() < size / least * 65536.0).double() * least if signed else (size > 0).double() * least
    size = torch.where(size < least, low, up)
    return (size.view(-1, BLOCK) * scale).view(-1) * torch.sign(value)


def _adamw_exact(case, seed):
    data, _ = _adamw_inputs(case, seed)
    t = STEP + 1
    w, g = data["weights"].double(), data["grads"].double()
    out = []
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g = g * min(1.0, data["max_norm"] / (float(norm) + 1e-6))
        out.append(norm)
    if case["bits"] == 8:
        m = _decode(data["m"], data["m_exponents"], True).double()
        v = _decode(data["v"], data["v_exponents"], False).double()
    else:
        m, v = data["m"].double(), data["v"].double()
    m += (g - m) * (1.0 - BETA1)
    v += (g.square() - v) * (1.0 - BETA2)
    w = w - LR * DECAY * w - LR * (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)).sqrt() + EPS)
    if case["average"]:
        out.append(data["average"].double() + (1.0 - AVERAGE) * (w - data["average"].double()))
    if case["bits"] == 8:
        words = _philox(w.numel() // 4, t, data["seed"])
        m = _nearest_states(m, words & 65535, True)
        v = _nearest_states(v, words >> 16, False)
    return [w, m, v, *out]


def _block_exact(case, seed):
    """Gradients from the formulas (the plain form leaves them to autograd)."""
    s = _block_inputs(case, seed, torch.float64)
    c, degrees = case["channels"], range(case["lmax"] + 1)
    cut = lambda x: _degrees(case, x)  # noqa: E731
    join = lambda blocks: _rows(case, blocks)  # noqa: E731
    wide = lambda w: [w[l][None, :, None] for l in degrees]  # noqa: E731
    rate = lambda bs: [(b.square().mean((1, 2), keepdim=True) + NORM_EPS) ** -0.5 for b in bs]  # noqa: E731
    mean = lambda a, b: (a * b).mean((1, 2), keepdim=True)  # noqa: E731
    x, pre = cut(s["x"]), None
    block, gated = case["op"] == "block", case["gate"]
    if block:
        y = cut(s["y"])
        r1 = rate(y)
        post, scale = wide(s["post"]), wide(s["scale"])
        if gated:
            z = s["gate"].view(-1, case["lmax"] + 1, c, 1)
            sig = [torch.sigmoid(z[:, l]) for l in degrees]
        else:
            sig = [torch.ones((), device=DEVICE, dtype=torch.float64) for _ in degrees]
        weight = [post[l] * scale[l] for l in degrees]
        a = [weight[l] * sig[l] for l in degrees]
        h = [x[l] + a[l] * r1[l] * y[l] for l in degrees]
    else:
        h = x
    out = [join(h)] if block else []
    if case["pre"]:
        pre, r2 = wide(s["pre"]), rate(h)
        out.append(join([pre[l] * r2[l] * h[l] for l in degrees]))
    if case["run"] == "forward":
        return out
    p = cut(s["p"]) if block else [torch.zeros_like(b) for b in h]
    T = p
    if case["pre"]:
        q = cut(s["q"])
        t2 = [pre[l] * q[l] for l in degrees]
        T = [p[l] + r2[l] * t2[l] - r2[l] ** 3 * h[l] * mean(h[l], t2[l]) for l in degrees]
    first = [join(T)]
    if block:
        t1 = [a[l] * T[l] for l in degrees]
        first.append(join([r1[l] * t1[l] - r1[l] ** 3 * y[l] * mean(y[l], t1[l]) for l in degrees]))
        S = [(r1[l] * y[l] * T[l]).sum(2, keepdim=True) for l in degrees]        # per row and channel
        if gated:
            slope = [g * (1 - g) for g in sig]
            gates = lambda v: torch.cat([b.expand(-1, c, 1)[:, :, 0] for b in v], 1)  # noqa: E731
            first.append(gates([weight[l] * slope[l] * S[l] for l in degrees]))
    per = lambda v: torch.stack([b.sum((0, 2)) for b in v])  # noqa: E731
    if case["run"] == "train":
        last = []
        if block:
            total = per([sig[l] * S[l] for l in degrees])
            last += [total * s["scale"], total * s["post"]]
        if case["pre"]:
            last.append(per([r2[l] * h[l] * q[l] for l in degrees]))
        return [*out, *first, *last]
    tau = cut(s["dx"])
    if block:
        be = cut(s["dy"])
        inner = [r1[l] * be[l] - r1[l] ** 3 * y[l] * mean(y[l], be[l]) for l in degrees]
        gy = [-r1[l] ** 3 * (y[l] * mean(t1[l], be[l]) + t1[l] * mean(y[l], be[l]) + be[l] * mean(y[l], t1[l]))
              + 3 * r1[l] ** 5 * y[l] * mean(y[l], t1[l]) * mean(y[l], be[l]) for l in degrees]
        tau = [tau[l] + a[l] * inner[l] for l in degrees]
        ga = [(T[l] * inner[l]).sum(2, keepdim=True) for l in degrees]            # by sigma * weight
        gw = [sig[l] * ga[l] for l in degrees]
        if gated:
            de = s["dgate"].view(-1, case["lmax"] + 1, c, 1)
            de = [de[:, l] for l in degrees]
            zz = [de[l] * weight[l] * slope[l] for l in degrees]
            tau = [tau[l] + zz[l] * r1[l] * y[l] for l in degrees]
            gy = [gy[l] + r1[l] * zz[l] * T[l] - r1[l] ** 3 * y[l] * mean(y[l], zz[l] * T[l]) for l in degrees]
            gw = [gw[l] + de[l] * slope[l] * S[l] for l in degrees]
            gg = [weight[l] * slope[l] * (ga[l] + de[l] * (1 - 2 * sig[l]) * S[l]) for l in degrees]
    gp, gh = tau, [torch.zeros_like(b) for b in h]
    if case["pre"]:
        down = [r2[l] * tau[l] - r2[l] ** 3 * h[l] * mean(h[l], tau[l]) for l in degrees]
        gq = [pre[l] * down[l] for l in degrees]
        gpre = per([q[l] * down[l] for l in degrees])
        gh = [-r2[l] ** 3 * (h[l] * mean(t2[l], tau[l]) + t2[l] * mean(h[l], tau[l]) + tau[l] * mean(h[l], t2[l]))
              + 3 * r2[l] ** 5 * h[l] * mean(h[l], t2[l]) * mean(h[l], tau[l]) for l in degrees]
    second = [join(gh)]
    if block:
        # h' = x + a N(y): its gradient reaches y, the gate and the weights too
        t3 = [a[l] * gh[l] for l in degrees]
        gy = [gy[l] + r1[l] * t3[l] - r1[l] ** 3 * y[l] * mean(y[l], t3[l]) for l in degrees]
        S3 = [(r1[l] * y[l] * gh[l]).sum(2, keepdim=True) for l in degrees]
        gw = [gw[l] + sig[l] * S3[l] for l in degrees]
        second.append(join(gy))
        if gated:
            second.append(gates([gg[l] + weight[l] * slope[l] * S3[l] for l in degrees]))
        total = per(gw)
        second += [total * s["scale"], total * s["post"]]
    if case["pre"]:
        second.append(gpre)
    if block:
        second.append(join(gp))
    if case["pre"]:
        second.append(join(gq))
    return [*out, *first, *second]


def exact(case, seed):
    if case["op"] == "adamw":
        return _adamw_exact(case, seed)
    return _block_exact(case, seed)
