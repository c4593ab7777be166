"""The sequence and training operators of megacrn_amd as cases to time and to check: the gated linear recurrence (whole
sequences, their gradients, single steps) and the AdamW step over many tensors (32-bit or 8-bit moments).

`run` computes a case in its plain form, elementary torch operations in 32 bits, or - with `own` set - through the
package's entry points.  `exact` computes it from the definition in 64 bits.

Gated linear recurrence, per channel, over time steps t (masked steps keep the state):
    a_t = sigmoid(gate_t)      x_t = (1 - a_t) * act(cand_t)      h_t = a_t * h_{t-1} + x_t
AdamW, per element, with g already scaled and clipped by the norm over all tensors:
    m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g g
    p = (1 - lr wd) p - lr / (1 - b1^s) * m / (sqrt(v) / sqrt(1 - b2^s) + eps)
8-bit moments: blocks of 64 elements, a power-of-two scale each (one byte, biased by 127), m as a signed float of 4
exponent and 3 mantissa bits (bias 7), v as an unsigned one of 5 and 3 (bias 15), both rounded stochastically with
16 + 16 bits that are a function of (seed, tensor, step, element).
"""
import math

import torch

own = False

F32 = torch.float32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 64
BETAS, EPS, LR, SEED = (0.9, 0.999), 1e-8, 1e-3, 20


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _glr(name, kind, B, T, N, H, G, dtype, mask, act="tanh"):
    case = {"op": "glr", "kind": kind, "B": B, "T": T, "N": N, "H": H, "G": G, "dtype": dtype, "mask": mask, "act": act}
    return dict(case, name=name) if name else case


def _adamw(name, dtype, bits, clip, N=0, H=64, layers=0, done=100):
    case = {"op": "adamw", "dtype": dtype, "bits": bits, "clip": clip, "N": N, "H": H, "layers": layers, "done": done}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one new reading of every METR-LA sensor arrives at a server that keeps the states: latency is all
        _glr("step_one", "step", 1, 1, 207, 64, 64, "f32", False),
        # the same for a batch of rollouts over PEMS-BAY's sensors, with sensors that sent nothing
        _glr("step_batch", "step", 64, 1, 325, 64, 64, "bf16", True),
        # the encoder's window of a METR-LA training batch, missing readings masked
        _glr("train_window", "train", 64, 12, 207, 64, 64, "f32", True),
        # a week of 5-minute readings as one sequence, as training on long histories has it
        _glr("train_week", "train", 4, 2016, 207, 64, 64, "f32", False),
        # EXPY-TKY's links with one forget gate for each link, over a day of 10-minute readings
        _glr("train_node_gate", "train", 2, 144, 1843, 32, 1, "bf16", True),
        # a month of PEMS-BAY read once to build the state that a forecast starts from
        _glr("read_month", "read", 1, 8928, 325, 64, 64, "bf16", False),
        # one sensor's long record: hardly any channels, all the work lies along the time axis; odd in every size
        _glr("train_sensor", "train", 1, 20161, 1, 33, 33, "f32", True, "none"),
        # the optimizer step of the METR-LA model: 14 tensors, most of them tiny
        _adamw("adamw_metrla", "f32", 32, True, N=207),
        # the same for PEMS-BAY with 8-bit moments
        _adamw("adamw8_pemsbay", "f32", 8, True, N=325),
        # a deep stack of wide cells
        _adamw("adamw_stack", "f32", 32, True, H=1024, layers=4),
        # a stack of odd width whose moments are held in 8 bits, without clipping
        _adamw("adamw8_odd", "f32", 8, False, H=333, layers=12),
        # the wide stack in bf16 with fp32 master weights and 8-bit moments
        _adamw("adamw8_master", "bf16", 8, True, H=1024, layers=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if rng.random() < 0.6:
        kind = rng.choice(["step", "read", "train", "train"])
        H = rng.choice([rng.randint(1, 130), 32, 64, 128])
        G = rng.choice([H, H, 1, next(q for q in range(max(2, H // 4), H + 1) if H % q == 0) if H > 1 else 1])
        N = _log(rng, 1, 2000)
        B = _log(rng, 1, 64)
        most = 100_000_000 if kind == "train" else 180_000_000
        T = 1 if kind == "step" else min(_log(rng, 1, 20000), max(1, most // (B * N * H)))
        return _glr("", kind, B, T, N, H, G, dtype, rng.random() < 0.5, rng.choice(["tanh", "none"]))
    bits, clip, done = rng.choice([8, 32]), rng.random() < 0.6, _log(rng, 1, 100000)
    dtype = rng.choice(["f32", "f32", "bf16"])
    if rng.random() < 0.4:
        return _adamw("", dtype, bits, clip, N=_log(rng, 3, 8192), H=rng.randint(5, 128), done=done)
    H = _log(rng, 16, 700)
    return _adamw("", dtype, bits, clip, H=H, layers=rng.randint(1, 8), done=done)


def _shapes(case):
    """Shapes of the parameters: the model's (N > 0; 20 memory items of 64 values, 3 hops), or those of a stack of cells."""
    H, K = case["H"], 3

    def cell(din, h):
        return [(2 * K * (din + h), 2 * h), (2 * h,), (2 * K * (din + h), h), (h,)]

    if case["N"]:
        M, D = 20, 64
        return [(M, D), (H, D), (case["N"], M), (case["N"], M)] + cell(1, H) + cell(2, H + D) + [(1, H + D), (1,)]
    return [s for i in range(case["layers"]) for s in cell(1 if i == 0 else H, H)]


def _padded(case):
    return [(math.prod(s) + BLOCK - 1) // BLOCK * BLOCK for s in _shapes(case)]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    rng = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, std=1.0, mean=0.0, dtype=F32):
        return torch.randn(shape, generator=rng, device="cuda").mul_(std).add_(mean).to(dtype)

    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "glr":
        B, T, N, H, G = (case[k] for k in "BTNHG")
        lead = (B, N) if case["kind"] == "step" else (B, T, N)
        s["gate"] = normal((*lead, G), 1.5, 2.0, dt)
        s["cand"] = normal((*lead, H), 1.0, 0.0, dt)
        s["state"] = normal((B, N, H), 0.5)
        s["mask"] = torch.rand(lead, generator=rng, device="cuda") >= 0.08 if case["mask"] else None
        if case["kind"] == "train":
            s["dout"], s["dlast"] = normal((*lead, H), 1.0, 0.0, dt), normal((B, N, H))
            for k in ("gate", "cand", "state"):
                s[k].requires_grad_()
        return s
    shapes, n, total = _shapes(case), _padded(case), sum(_padded(case))
    s["params"] = [normal(q, 0.05, 0.0, dt) for q in shapes]
    spread = [10.0 ** (i % 5 - 4) for i in range(len(shapes))]     # tensors' gradients differ by orders of magnitude
    s["grads"] = [normal(q, k, 0.0, dt) for q, k in zip(shapes, spread)]
    real = torch.cat([torch.arange(k, device="cuda") < math.prod(q) for k, q in zip(n, shapes)])
    size = torch.cat([torch.full((k,), w, device="cuda") for k, w in zip(n, spread)]) * real
    s["m"] = normal(total, 0.3) * size
    s["v"] = (normal(total, 0.5, 1.0) * size).square()
    s["master"] = _flat(s["params"], case) if case["dtype"] == "bf16" else None
    s["steps"] = case["done"]
    if case["bits"] == 8:
        zero = torch.zeros(total, dtype=torch.int64, device="cuda")
        s["m"], s["v"] = _encode(s["m"], zero, 7, 7, True), _encode(s["v"], zero, 15, 15, False)
    if own:
        import megacrn_amd
        s["opt"] = megacrn_amd.AdamW(s["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=0.01, state_bits=case["bits"],
                                     max_grad_norm=1.0 if case["clip"] else 0.0, seed=SEED)
        held = {"m": s["m"], "v": s["v"]} if case["bits"] == 32 else {
            "m": s["m"][0], "m_scale": s["m"][1], "v": s["v"][0], "v_scale": s["v"][1]}
        if s["master"] is not None:
            held["master"] = s["master"]
        s["opt"].load_state_dict(dict(held, steps=[case["done"]] * len(shapes), state_bits=case["bits"]))
        s["m"] = s["v"] = s["master"] = None
    return s


def _flat(tensors, case):
    """The tensors behind one another in 32 bits, each filled up with zeros to whole blocks."""
    return torch.cat([torch.nn.functional.pad(t.reshape(-1).float(), (0, n - t.numel())) for t, n in zip(tensors, _padded(case))])


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "glr":
        return (_own_glr if own else _plain_glr)(s, case)
    return (_own_adamw if own else _plain_adamw)(s, case)


def _own_glr(s, case):
    import megacrn_amd
    if case["kind"] == "step":
        out = megacrn_amd.gated_linear_recurrence_step(s["gate"], s["cand"], s["state"], s["mask"], activation=case["act"])
        return {"out": out, "state": s["state"]}
    out, last = megacrn_amd.gated_linear_recurrence(s["gate"], s["cand"], s["state"], s["mask"], activation=case["act"])
    if case["kind"] == "read":
        return {"out": out, "last": last}
    grads = torch.autograd.grad((out, last), (s["gate"], s["cand"], s["state"]), (s["dout"], s["dlast"]))
    return {"out": out, "last": last, "dgate": grads[0], "dcand": grads[1], "dstate": grads[2]}


def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t from h = 0, along dim 1, by doubling the stride; a and x are overwritten."""
    d = 1
    while d < x.shape[1]:
        x[:, d:] += a[:, d:] * x[:, :-d]
        if 2 * d < x.shape[1]:
            a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return x


@torch.no_grad()
def _plain_glr(s, case):
    dt, H, G = DTYPES[case["dtype"]], case["H"], case["G"]
    step = case["kind"] == "step"
    gate, cand, h0 = s["gate"].float(), s["cand"].float(), s["state"]
    lead = gate.shape[:-1]
    grouped = (*lead, G, H // G)
    a, w = torch.sigmoid(gate).unsqueeze(-1).expand(grouped).reshape(cand.shape), torch.sigmoid(-gate).unsqueeze(-1).expand(grouped).reshape(cand.shape)
    c = torch.tanh(cand) if case["act"] == "tanh" else cand
    x = w * c
    if s["mask"] is not None:
        keep = s["mask"].unsqueeze(-1)
        a, x = torch.where(keep, a, 1.0), torch.where(keep, x, 0.0)
    if step:
        s["state"].copy_(a * h0 + x)
        return {"out": s["state"].to(dt), "state": s["state"]}
    x[:, 0] += a[:, 0] * h0
    h = _scan(a.clone(), x)
    last = h[:, -1].clone()
    if case["kind"] == "read":
        return {"out": h.to(dt), "last": last}
    # gradient: lam_t = dout_t + a_{t+1} lam_{t+1}, from the far end
    d = s["dout"].to(F32, copy=True)
    d[:, -1] += s["dlast"]
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    lam = _scan(nxt.flip(1), d.flip(1)).flip(1)
    prev = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    dc, dg = lam * w, lam * a * w * (prev - c)
    if case["act"] == "tanh":
        dc = dc * (1 - c * c)
    if s["mask"] is not None:
        dc, dg = torch.where(keep, dc, 0.0), torch.where(keep, dg, 0.0)
    return {"out": h.to(dt), "last": last, "dgate": dg.reshape(grouped).sum(-1).to(dt), "dcand": dc.to(dt), "dstate": a[:, 0] * lam[:, 0]}


def _own_adamw(s, case):
    opt = s["opt"]
    opt.step(grads=s["grads"])
    m, v = opt.moments()
    out = {"params": s["params"], "m": m, "v": v}
    if case["dtype"] == "bf16":
        out["master"] = opt.master
    if case["clip"]:
        out["norm"] = opt.total_norm
    return out


M32 = 0xFFFFFFFF


def _mix(x):
    """A mixing of 32 bits (xor-shifts and odd multipliers) on Python numbers or int64 tensors that hold 32 bits."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _random_bits(case, step):
    """32 bits for every element of the flat order: a function of the seed, the tensor, the step and the element's index."""
    keys = [_mix((SEED + 0x9E3779B9 * (i + 1) + _mix(step & M32)) & M32) for i in range(len(_shapes(case)))]
    index = torch.cat([torch.arange(n, device="cuda") for n in _padded(case)])
    key = torch.repeat_interleave(torch.tensor(keys, device="cuda"), torch.tensor(_padded(case), device="cuda"))
    return _mix(((index & M32) * 0x9E3779B9 + (index >> 32) * 0x85157AF5 + key) & M32)


def _encode(x, bits16, bias, top, signed):
    """Codes (uint8) and the blocks' scale bytes: the largest finite value of a block comes to [2^top, 2^(top+1)).
    bits16: the random bits that are added below the last kept one."""
    size = x.abs().reshape(-1, BLOCK)
    size_or_0 = torch.where(torch.isfinite(size), size, 0.0)
    scale = ((size_or_0.amax(1).view(torch.int32) >> 23) - top).clamp(min=1)
    # below 2^-126 the exponent field is 0 and the bits are those of a fixed point: the format's own subnormals
    t = (size * ((254 - scale) << 23).view(F32).unsqueeze(1)).reshape(-1) * 2.0 ** (bias - 127)
    code = (t.view(torch.int32) + (bits16.to(torch.int32) << 4)) >> 20
    if not signed:
        code = torch.where((x > 0) & (code < 1), 1, code)     # what is above nothing stays above nothing
    code = torch.where(torch.isfinite(x), code, 0x7F if signed else 0xFF)
    if signed:
        code = code | ((x.view(torch.int32) >> 24) & 0x80)
    return code.to(torch.uint8), scale.to(torch.uint8)


def _decode(held, bias, signed):
    code, scale = held[0].to(torch.int32), held[1].to(torch.int32)
    sign = 1.0 - 2.0 * (code >> 7).to(F32) if signed else 1.0
    code = code & 0x7F if signed else code
    value = (code << 20).view(F32) * 2.0 ** (127 - bias)
    value = torch.where(code == (0x7F if signed else 0xFF), torch.nan, value)
    return sign * (value.reshape(-1, BLOCK) * (scale << 23).view(F32).unsqueeze(1)).reshape(-1)


def _plain_adamw(s, case):
    (b1, b2), eight = BETAS, case["bits"] == 8
    s["steps"] += 1
    n = s["steps"]
    g = _flat(s["grads"], case)
    out = {"params": s["params"]}
    if case["clip"]:
        norm = g.double().square().sum().sqrt().to(F32)
        out["norm"] = norm
        g = g * (torch.ones_like(norm) / (norm + 1e-6)).clamp(max=1.0)
    m, v = (_decode(s["m"], 7, True), _decode(s["v"], 15, False)) if eight else (s["m"], s["v"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    p = s["master"] if s["master"] is not None else _flat(s["params"], case)
    p = p * (1 - LR * 0.01) - (m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** n)) + EPS)) * (LR / (1 - b1 ** n))
    pieces = [q[: w.numel()].view(w.shape) for q, w in zip(p.split(_padded(case)), s["params"])]
    torch._foreach_copy_(s["params"], pieces)
    if s["master"] is not None:
        out["master"] = s["master"] = p
    if eight:
        bits = _random_bits(case, n)
        s["m"], s["v"] = _encode(m, bits & 0xFFFF, 7, 7, True), _encode(v, bits >> 16, 15, 15, False)
        out["m"], out["v"] = _decode(s["m"], 7, True), _decode(s["v"], 15, False)
    else:
        out["m"], out["v"] = s["m"], s["v"] = m, v
    return out


# ---------------------------------------------------------------------------------------------------------------------
# work, and the outputs in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "glr":
        rows = case["B"] * case["T"] * case["N"]
        gate, cand, state = rows * case["G"] * size, rows * case["H"] * size, case["B"] * case["N"] * case["H"] * 4
        mask = rows if case["mask"] else 0
        one = gate + 2 * cand + 2 * state + mask             # gate, cand, state, mask in; out, last out
        if case["kind"] != "train":
            return {"bytes": one, "flops": 12 * rows * case["H"]}
        return {"bytes": one + 2 * cand + gate + 2 * state, "flops": 30 * rows * case["H"]}   # dout, dlast in; three gradients out
    n = sum(math.prod(q) for q in _shapes(case))
    held = 8 if case["bits"] == 32 else 2 + 2 / BLOCK        # both moments of an element
    each = 3 * size + 2 * held + (8 if case["dtype"] == "bf16" else 0)      # p, g in and p out; moments and masters both ways
    return {"bytes": int(n * (each + (8 if case["bits"] == 8 else 0))), "flops": 15 * n}      # 8-bit moments come back as values


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_glr if case["op"] == "glr" else _exact_adamw)(s, case)


@torch.no_grad()
def _exact_glr(s, case):
    H, G = case["H"], case["G"]
    step = case["kind"] == "step"
    gate, cand = (s[k].double().unsqueeze(1) if step else s[k].double() for k in ("gate", "cand"))
    a = 1 / (1 + torch.exp(-gate))
    w = 1 / (1 + torch.exp(gate))
    a, w = (q.repeat_interleave(H // G, dim=-1) for q in (a, w))
    c = torch.tanh(cand) if case["act"] == "tanh" else cand
    B, T, N = cand.shape[:3]
    keep = torch.ones((B, T, N, 1), dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"].reshape(B, T, N, 1)
    w = w.masked_fill(~keep, 0.0)
    a = a.masked_fill(~keep, 1.0)
    h, x = torch.empty_like(c), w * c
    now = s["state"].double()
    for t in range(T):
        now = torch.addcmul(x[:, t], a[:, t], now)
        h[:, t] = now
    if step:
        return {"out": h[:, 0], "state": h[:, 0]}
    if case["kind"] == "read":
        return {"out": h, "last": now}
    lam, back = torch.empty_like(c), s["dlast"].double()
    dout = s["dout"].double()
    for t in reversed(range(T)):
        torch.add(dout[:, t], back, out=lam[:, t])
        back = a[:, t] * lam[:, t]
    dc = lam * w * (1 - c * c if case["act"] == "tanh" else 1.0)
    h -= c
    dg = lam * w * a
    dg[:, 1:] *= h[:, :-1] + (c[:, :-1] - c[:, 1:])
    dg[:, 0] *= s["state"].double() - c[:, 0]
    h += c
    return {"out": h, "last": now, "dgate": dg.reshape(B, T, N, G, H // G).sum(-1), "dcand": dc, "dstate": back}


def _exact_adamw(s, case):
    (b1, b2), eight, n = BETAS, case["bits"] == 8, case["done"] + 1
    norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in s["grads"]))
    coef = min(1.0, 1.0 / (norm + 1e-6)) if case["clip"] else 1.0
    if eight:
        m0, v0 = _value64(s["m"], 7, True), _value64(s["v"], 15, False)
    else:
        m0, v0 = s["m"].double(), s["v"].double()
    at, out = 0, {"params": [], "m": [], "v": [], "master": []}
    for w, g, room in zip(s["params"], s["grads"], _padded(case)):
        k = w.numel()
        g, p = g.double().reshape(-1) * coef, w.double().reshape(-1)
        m = b1 * m0[at:at + k] + (1 - b1) * g
        v = b2 * v0[at:at + k] + (1 - b2) * g * g
        p = p * (1 - LR * 0.01) - LR / (1 - b1 ** n) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** n) + EPS)
        out["params"].append(p.view(w.shape))
        for key, val in (("m", m), ("v", v), ("master", p)):
            out[key] += [val, val.new_zeros(room - k)]
        at += room
    got = {"params": out["params"], "m": None if eight else torch.cat(out["m"]), "v": None if eight else torch.cat(out["v"])}
    if case["dtype"] == "bf16":
        got["master"] = torch.cat(out["master"])
    if case["clip"]:
        got["norm"] = torch.tensor(norm, dtype=torch.float64)
    return got


def _value64(held, bias, signed):
    """What the codes stand for, from a table of the format's values."""
    table = [(c * 2.0 ** (-2 - bias) if c < 8 else (8 + (c & 7)) / 8 * 2.0 ** ((c >> 3) - bias)) for c in range(128 if signed else 256)]
    table = torch.tensor(table + [-q for q in table] if signed else table, dtype=torch.float64, device="cuda")
    return table[held[0].long()] * torch.exp2(held[1].double() - 127).repeat_interleave(BLOCK)
