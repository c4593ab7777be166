"""Oracle of the gated linear recurrence and of the AdamW step: numpy in float64, one step after the other, straight from the
definitions; and error bounds of an fp32 evaluation that run along with them (u = 2^-24, half an fp32 step).
Test infrastructure only."""
import numpy as np

U = 2.0 ** -24

# Relative errors, in units of u, that the bounds grant an fp32 evaluation of the step's functions:
#   the smaller one of a = sigmoid(gate) and w = 1 - a <= 10: exponential 4, and half of it again through the sum, sum 1, reciprocal 2, product 1 (a gate
#   beyond 17: exponential up to 7, the others exact); the larger one enters as 1 - that, so what it multiplies is off by the smaller one's error
#   and a rounding of the result
#   tanh <= 12: exponential 4 (its weight is at most 1 where the quotient is used), difference 1, sum 3, reciprocal 2, product 1, one spare
#   a w <= 17: the smaller one's 10 times (1 - 2 n) / (1 - n) <= 1, product and sum 2, spare
# of inputs of any type: they are converted to fp32 first.
KW, KC, KP = 10, 12, 17


def _gates(gate, cand, mask, act):
    H, G = cand.shape[-1], gate.shape[-1]
    g = np.repeat(gate, H // G, axis=-1)
    with np.errstate(over="ignore"):
        w = 1.0 / (1.0 + np.exp(g))
        a = 1.0 / (1.0 + np.exp(-g))
    c = np.tanh(cand) if act == "tanh" else cand.copy()
    if mask is not None:
        off = ~np.broadcast_to(mask, cand.shape[:3])
        w[off], a[off], c[off] = 0.0, 1.0, 0.0          # whatever was there, NaN included
    return a, w, c


def _c_error(c, act):
    """Error granted to phi(cand), in units of u."""
    return KC * np.abs(c) if act == "tanh" else np.zeros_like(c)


def glr_fwd(gate, cand, state=None, mask=None, act="tanh", dt="f32"):
    """gate (B,T,N,G), cand (B,T,N,H), state (B,N,H), mask (B,T,N) -> out, last, bound of |error| of out in fp32, cache.
    dt: the inputs' type; the arithmetic is fp32 for all of them, so the bounds do not depend on it."""
    B, T, N, H = cand.shape
    a, w, c = _gates(gate, cand, mask, act)
    h = np.zeros((B, N, H)) if state is None else state.astype(np.float64)
    out, err, prev = np.zeros((B, T, N, H)), np.zeros((B, T, N, H)), np.zeros((B, T, N, H))
    size, e = np.abs(h), np.zeros((B, N, H))            # recursion on absolute values: no cancellation is counted on
    for t in range(T):
        prev[:, t] = h
        span = np.abs(c[:, t]) + size
        e = a[:, t] * e + U * ((KW + 2) * np.minimum(a[:, t], w[:, t]) * span + w[:, t] * _c_error(c[:, t], act))
        size = a[:, t] * size + w[:, t] * np.abs(c[:, t])
        e = e + U * size
        h = a[:, t] * h + w[:, t] * c[:, t]
        out[:, t], err[:, t] = h, e
    # a step's rounding enters twice where maps of segments are composed before the steps are run
    return out, h, 2 * err, (a, w, c, prev, 2 * err, act, gate.shape[-1])


def glr_bwd(cache, dout=None, dlast=None):
    """-> dgate, dcand, dstate and bounds of their errors in fp32 (the same order)."""
    a, w, c, prev, eh, act, G = cache
    B, T, N, H = a.shape
    mu = np.zeros((B, N, H)) if dlast is None else dlast.astype(np.float64)
    size, e = np.abs(mu), np.zeros((B, N, H))
    dg, dc, eg, ec = (np.zeros((B, T, N, H)) for _ in range(4))
    for t in reversed(range(T)):
        d = 0.0 if dout is None else dout[:, t]
        lam, big = mu + d, size + np.abs(d)
        el = e + U * big                                # error of lam
        slope = 1 - c[:, t] ** 2 if act == "tanh" else np.ones_like(lam)
        dc[:, t] = lam * w[:, t] * slope
        ec[:, t] = w[:, t] * (slope * (2 * el + U * (KW + 4) * np.abs(lam)) + U * (2 * np.abs(c[:, t]) * _c_error(c[:, t], act) + 2) * np.abs(lam) * (act == "tanh"))
        p, diff = a[:, t] * w[:, t], prev[:, t] - c[:, t]
        before = eh[:, t - 1] if t else 0.0
        dg[:, t] = lam * p * diff
        eg[:, t] = p * (2 * el * np.abs(diff) + np.abs(lam) * (before + U * (_c_error(c[:, t], act) + np.abs(prev[:, t]) + (KP + 3) * np.abs(diff))))
        mu = a[:, t] * lam
        size = a[:, t] * big
        e = a[:, t] * el + U * ((KW + 1) * np.minimum(a[:, t], w[:, t]) * big + size)
    D = H // G
    terms = np.abs(dg).reshape(B, T, N, G, D).sum(-1)
    dgate = dg.reshape(B, T, N, G, D).sum(-1)
    egate = eg.reshape(B, T, N, G, D).sum(-1) + (D - 1) * U * terms
    return dgate, dc, mu, egate, ec, 2 * e


def half_step(x, dtype):
    """Half the distance of two numbers of `dtype` at x: what one rounding to it can be off by."""
    half, tiny = {"f32": (2.0 ** -24, 2.0 ** -150), "bf16": (2.0 ** -8, 2.0 ** -134), "f16": (2.0 ** -11, 2.0 ** -25)}[dtype]
    return half * np.abs(x) + tiny


# ---------------------------------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------------------------------
def adamw_step(p, g, m, v, step, lr, wd, b1=0.9, b2=0.999, eps=1e-8, factor=1.0):
    """One element-wise step in float64 -> p, m, v and bounds of what an fp32 evaluation from the same inputs is off by."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    g = g * factor
    big_m, big_v = b1 * np.abs(m) + (1 - b1) * np.abs(g), b2 * v + (1 - b2) * g * g
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em, ev = 5 * U * big_m + 2.0 ** -148, 7 * U * big_v + 2.0 ** -148     # constant, factor (2), product, sum; g twice in v
    denom = np.sqrt(v) / np.sqrt(1 - b2 ** step) + eps
    size = lr / (1 - b1 ** step)
    upd = size * m / denom
    # sqrt halves v's relative error (or leaves sqrt(ev) where v is below what fp32 holds), four roundings in the denominator
    ed = np.where(v > 2.0 ** -120, 0.5 * ev / np.sqrt(np.maximum(v, 2.0 ** -120)), np.sqrt(ev)) / np.sqrt(1 - b2 ** step) + 4 * U * denom
    new = p * (1 - lr * wd) - upd
    ep = size / denom * em + np.abs(upd) * ed / denom + 4 * U * np.abs(upd) + 3 * U * np.abs(p)
    return new, m, v, ep, em, ev


F = np.float32


def mix(x):
    x = x & 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(seed, tensor, step, n):
    """32 bits for each of the n elements of a tensor."""
    key = mix(seed + 0x9E3779B9 * (tensor + 1) + mix(step))
    return np.array([mix(i * 0x9E3779B9 + key) for i in range(n)], dtype=np.uint64).astype(np.int64)


def table(second):
    """The numbers of the 8-bit formats, by their codes: the sign apart from m."""
    bias = 15 if second else 7
    return np.array([c * 2.0 ** (-2 - bias) if c < 8 else (1 + (c % 8) / 8) * 2.0 ** (c // 8 - bias) for c in range(256 if second else 128)])


def encode(x, bits16, second):
    """fp32 values -> codes and scale bytes, one value after the other: the chance of the upper neighbour is the distance from the
    lower one, decided by the 16 random bits against the value's own bits below the third of the mantissa."""
    n = len(x)
    codes, scales = np.zeros(n, np.uint8), []
    bias, top = (15, 15) if second else (7, 7)
    for b in range(0, n, 64):
        blk = x[b:b + 64]
        fin = [abs(float(q)) for q in blk if np.isfinite(q)]
        big = max(fin, default=0.0)
        field = int(np.array(big, F).view(np.int32)) >> 23
        s = max(field - top, 1)
        scales.append(s)
        for k, q in enumerate(blk):
            if not np.isfinite(q):
                codes[b + k] = 0xFF if second else 0x7F | (0x80 if np.signbit(q) else 0)
                continue
            units = abs(float(q)) * 2.0 ** (127 - s) * 2.0 ** (bias - 127)          # exact in float64
            u = int(np.array(F(units)).view(np.int32))
            c = (u + (int(bits16[b + k]) << 4)) >> 20
            if second:
                c = max(c, 1) if q > 0 else c
            elif np.signbit(q):
                c |= 0x80
            codes[b + k] = c
    return codes, np.array(scales, np.uint8)


def decode(codes, scales, second):
    t = table(second)
    c = codes.astype(int)
    val = t[c] if second else t[c & 0x7F] * np.where(c & 0x80, -1.0, 1.0)
    val = np.where(c == 0xFF if second else (c & 0x7F) == 0x7F, np.nan, val)
    return val * np.exp2(np.repeat(scales.astype(float), 64)[:len(codes)] - 127)


def moments_f32(g, m, v, factor, b1=0.9, b2=0.999):
    """The moments as single fp32 operations, in the order that the kernels have."""
    g = g.astype(F) * F(factor)
    m = F(b1) * m.astype(F) + F(1 - b1) * g
    return m, F(b2) * v.astype(F) + (F(1 - b2) * g) * g
