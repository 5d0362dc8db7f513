"""numpy restatement of the AdamW step in float64, with states in full precision or in 8 bits, and
of the gradient norm.

TEST INFRASTRUCTURE ONLY.  The full-precision step is pinned by ``torch.optim.AdamW`` in float64
(tests/test_adamw.py); the 8-bit states follow the definition in include/gi2d.h.

``u`` is half a step of float32.  Beside each result stands a bound for how far float32 arithmetic
may be from it, counted rounding by rounding."""
import numpy as np

u = 2.0 ** -24
BLOCK = 256


def step(p, g, m, v, t, lr, betas, eps, weight_decay, clip=1.0, more=0):
    """New (p, m, v) and the bounds of their float32 counterparts.  Inputs are the float32 (or
    half) values, exactly; ``clip`` the float32 coefficient, ``more`` the roundings by which it may
    itself be off.  The parameter with 8-bit states: the root 3.5 from v and 1, the denominator's
    factors 3 each (itself, the step size, their quotient), its sum 1, the hardware's reciprocal a
    unit in the last place (2), the difference 1: 11.5, below the 14 counted here."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    b1, b2 = betas
    g = g * clip                                     # 1 rounding of g
    m_new = b1 * m + (1 - b1) * g
    # each product: its coefficient, itself (and g's own), then the sum: 4 roundings of the larger
    tol_m = u * (4 * np.abs(b1 * m) + (4 + more) * np.abs((1 - b1) * g)) + 2.0 ** -149
    v_new = b2 * v + (1 - b2) * g * g
    # all terms positive: g twice, g*g, coefficient, product, sum (v itself may be a rounded
    # square: 1 more)
    tol_v = (7 + 2 * more) * u * v_new + 2.0 ** -148
    step_size = lr / (1 - b1 ** t)
    denom = np.sqrt(v_new / (1 - b2 ** t)) + eps
    with np.errstate(divide="ignore", invalid="ignore"):
        up = step_size * m_new / denom
        # denominator: half of v's 7, the root 1, the coefficient 1, the product 1, eps 1 and the
        # sum 1 = 8.5 (and `more`); the quotient 1, the step size 2, the product 1, the difference
        # 1: below 14
        tol_p = u * (3 * np.abs(p) + (14 + more) * np.abs(up)) + step_size * tol_m / denom
    return p * (1 - lr * weight_decay) - up, m_new, v_new, tol_p, tol_m, tol_v


def e4m3_values():
    """The 128 values of e4m3's codes without sign (the last one NaN)."""
    c = np.arange(128)
    e, f = c >> 3, c & 7
    x = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    x[127] = np.nan
    return x


def decode(codes, scales, n):
    """Values of ``n`` uint8 codes with a scale for each 256."""
    x = e4m3_values()[codes & 127]
    return np.where(codes & 128, -x, x) * np.repeat(np.asarray(scales, np.float64), BLOCK)[:n]


def _hash(x):
    x = np.asarray(x, np.uint64)
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        x = x ^ (x >> np.uint64(shift))
        x = (x * np.uint64(factor)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def words(seed, t, first_block, n):
    """The random word of each of ``n`` elements of a tensor whose first block has this number."""
    low = np.uint64(0xFFFFFFFF)
    stride = np.uint64(0x9E3779B9)
    key = _hash(_hash(seed) ^ ((np.uint64(t) * stride) & low))
    i = np.arange(n, dtype=np.uint64)
    block = (np.uint64(first_block) + i // np.uint64(BLOCK)) & low
    return _hash((_hash((key + block * stride) & low) + (i % np.uint64(BLOCK)) * stride) & low)


def encode(x, random16, nonzero):
    """uint8 codes and scales of ``x``; also, element by element, how much the value could move
    before the random number sent it to the other code."""
    n = x.size
    blocks = -(-n // BLOCK)
    a = np.zeros(blocks * BLOCK)
    finite = np.isfinite(x)
    a[:n] = np.where(finite, np.abs(x), 0.0)
    top = a.reshape(blocks, BLOCK).max(1)
    with np.errstate(divide="ignore"):
        k = np.ceil(np.log2(top / 448.0))
    for d in (-1, 0, 1):                             # (log2 may be off at a power of two)
        k0 = np.ceil(np.log2(np.maximum(top, 1e-300) / 448.0)) + d
        k = np.where((top <= 448.0 * 2.0 ** k0) & (top > 448.0 * 2.0 ** (k0 - 1)), k0, k)
    k = np.clip(k, -100, 119)
    scales = 2.0 ** k
    values = e4m3_values()[:127]
    y = (a / np.repeat(scales, BLOCK))[:n]
    lo = np.clip(np.searchsorted(values, y, side="right") - 1, 0, 126)
    hi = np.minimum(lo + 1, 126)
    gap = np.where(hi > lo, values[hi] - values[lo], 1.0)
    at = (y - values[lo]) / gap + (np.asarray(random16, np.float64) + 0.5) / 65536
    code = np.where(at >= 1, hi, lo)
    if nonzero:
        code = np.where((code == 0) & (x > 0), 1, code)
    code = np.where(finite, code, 127)
    margin = np.abs(at - 1) * gap * np.repeat(scales, BLOCK)[:n]
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8), scales, margin


def grad_norm(grads, max_norm):
    total = sum(float(np.sum(np.asarray(g, np.float64) ** 2)) for g in grads)
    norm = np.sqrt(total)
    return norm, min(1.0, max_norm / (norm + 1e-6))
