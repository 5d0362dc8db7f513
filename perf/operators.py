"""Optimizer operators over lists of tensors: the AdamW step with 32-bit and with 8-bit states, and
the norm of all gradients with the clip coefficient that belongs to it.

``own = False`` computes them from elementary torch operations, ``own = True`` through
``gaussianimage_amd.adamw``.  The tensors of a case are views into one buffer of each kind, every
tensor on a boundary of 256 elements as an allocator would place it; the gaps hold zeros, which the
operators neither read nor write and which the plain form maps to zeros.
"""
import math
import random

import torch

own = False

BLOCK = 256                      # elements behind one scale of an 8-bit state
DEVICE = "cuda:0"
BETAS, EPS, DECAY, LR, MAX_NORM = (0.9, 0.999), 1e-8, 1e-2, 1e-3, 1.0
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------- the cases

def listed():
    return [
        # one image of 5 000 Gaussians (positions, covariances, colours): a step of a small fit
        {"name": "step32_fit_5k", "op": "step32", "layout": "fit", "images": 1, "points": 5000,
         "param": "f32", "grad": "f32", "master": False, "clip": False, "step": 7},
        # 24 images of 30 000 Gaussians fitted together, gradients clipped
        {"name": "step32_fit_24x30k_clip", "op": "step32", "layout": "fit", "images": 24,
         "points": 30000, "param": "f32", "grad": "f32", "master": False, "clip": True, "step": 500},
        # mixed-precision training of stacked layers: bf16 weights and gradients, fp32 masters
        {"name": "step32_layers_bf16_master", "op": "step32", "layout": "layers", "width": 1024,
         "depth": 8, "param": "bf16", "grad": "bf16", "master": True, "clip": False, "step": 1000},
        # many small odd tensors, gradients accumulated in fp32
        {"name": "step32_ragged_bf16", "op": "step32", "layout": "ragged", "tensors": 257,
         "total": 3000017, "param": "bf16", "grad": "f32", "master": False, "clip": False, "step": 3},
        # one long flat tensor of odd length (a flattened shard)
        {"name": "step32_flat_f32", "op": "step32", "layout": "ragged", "tensors": 1,
         "total": 200000003, "param": "f32", "grad": "f32", "master": False, "clip": False,
         "step": 20000},
        # one image of 30 000 Gaussians, states in 8 bits
        {"name": "step8_fit_30k", "op": "step8", "layout": "fit", "images": 1, "points": 30000,
         "param": "f32", "grad": "f32", "master": False, "clip": False, "step": 40},
        # stacked layers in bf16 with 8-bit states, gradients clipped
        {"name": "step8_layers_bf16_clip", "op": "step8", "layout": "layers", "width": 1024,
         "depth": 8, "param": "bf16", "grad": "bf16", "master": False, "clip": True, "step": 1000},
        # many small odd tensors in fp16 with masters
        {"name": "step8_ragged_f16_master", "op": "step8", "layout": "ragged", "tensors": 131,
         "total": 5000011, "param": "f16", "grad": "f16", "master": True, "clip": False, "step": 9},
        # one long flat tensor of odd length
        {"name": "step8_flat_f32", "op": "step8", "layout": "ragged", "tensors": 1,
         "total": 120000007, "param": "f32", "grad": "f32", "master": False, "clip": False,
         "step": 300},
        # the norm alone: one image; stacked layers in bf16; a long flat tensor
        {"name": "norm_fit_30k", "op": "norm", "layout": "fit", "images": 1, "points": 30000,
         "grad": "f32"},
        {"name": "norm_layers_bf16", "op": "norm", "layout": "layers", "width": 1024, "depth": 8,
         "grad": "bf16"},
        {"name": "norm_flat_f32", "op": "norm", "layout": "ragged", "tensors": 1,
         "total": 200000003, "grad": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("step32", "step32", "step8", "step8", "norm"))
    layout = rng.choice(("fit", "layers", "ragged", "ragged"))
    case = {"op": op, "layout": layout}
    if layout == "fit":
        case["images"] = _log(rng, 1, 24)
        case["points"] = _log(rng, 1000, 200000)
    elif layout == "layers":
        case["width"] = 8 * _log(rng, 16, 128) + rng.choice((0, 0, 1, 4))
        case["depth"] = rng.randint(1, 8)
    else:
        case["tensors"] = _log(rng, 1, 300)
        case["total"] = case["tensors"] + _log(rng, 100, 100000000)
    if op == "norm":
        case["grad"] = rng.choice(("f32", "bf16", "f16"))
        return case
    case["param"] = rng.choice(("f32", "bf16", "f16"))
    case["grad"] = rng.choice((case["param"], case["param"], "f32"))
    case["master"] = case["param"] != "f32" and rng.random() < 0.5
    case["clip"] = rng.random() < 0.4
    case["step"] = _log(rng, 1, 50000)
    return case


def _shapes(case):
    """The tensors' shapes, from the case alone."""
    if case["layout"] == "fit":
        lead = (case["points"],) if case["images"] == 1 else (case["images"], case["points"])
        return [lead + (2,), lead + (3,), lead + (3,)]
    if case["layout"] == "layers":
        w = case["width"]
        one = [(w,), (3 * w, w), (w, w), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
        return [(8 * w, w)] + one * case["depth"] + [(w,)]
    r = random.Random(case["tensors"] * 1000003 + case["total"])
    share = [math.exp(r.uniform(0, 7)) for _ in range(case["tensors"])]
    total = sum(share)
    rest = case["total"] - case["tensors"]
    sizes = [1 + int(rest * s / total) for s in share]
    sizes[0] += case["total"] - sum(sizes)
    return [(s,) for s in sizes]


def work(case):
    n = sum(math.prod(s) for s in _shapes(case))
    per = SIZE[case["grad"]]
    if case["op"] == "norm":
        return {"bytes": per * n, "flops": 2 * n}
    if case["master"]:
        per += 8 + SIZE[case["param"]]          # master read and written, parameter written
    else:
        per += 2 * SIZE[case["param"]]
    per += 16 if case["op"] == "step32" else 4 + 16 / BLOCK
    return {"bytes": per * n, "flops": (16 if case["clip"] else 13) * n}


# ---------------------------------------------------------------------------- the inputs

def _views(flat, starts, shapes):
    return [flat[a:a + math.prod(s)].view(s) for a, s in zip(starts, shapes)]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    shapes = _shapes(case)
    starts, end = [], 0
    for s in shapes:
        starts.append(end)
        end += -(-math.prod(s) // BLOCK) * BLOCK
    inside = torch.zeros(end, dtype=torch.bool, device=DEVICE)
    for v in _views(inside, starts, shapes):
        v.fill_(True)

    def normal():
        return torch.randn(end, generator=gen, device=DEVICE) * inside

    # gradients, parameters and states differ in size from block to block of 256, as those of
    # different rows and tensors do
    size = torch.exp2(torch.randn(end // BLOCK, generator=gen, device=DEVICE) * 2 - 8)
    size = size.repeat_interleave(BLOCK)
    st = {"case": case, "grads": (normal() * size).to(DTYPE[case["grad"]])}
    names = ["grads"]
    if case["op"] != "norm":
        weights = normal() * 0.02
        st["params"] = weights.to(DTYPE[case["param"]])
        names.append("params")
        if case["master"]:
            st["masters"] = weights
            names.append("masters")
        mean, root = normal() * size * 0.3, normal().abs() * size + size * 0.05 * inside
        if case["op"] == "step32":
            st["exp_avgs"], st["exp_avg_sqs"] = mean, root * root
            names += ["exp_avgs", "exp_avg_sqs"]
        else:
            for name, x in (("exp_avgs", mean), ("exp_avg_rms", root)):
                rows = x.view(-1, BLOCK)
                top = rows.abs().amax(1).clamp(min=2.0 ** -90)
                scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
                st[name] = (rows / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
                st[name + "_scales"] = scale
                names.append(name)
            st["seed"] = seed % 65521
    del inside, size
    # what the program holds: lists of tensors over the buffers
    st["lists"] = {n: _views(st[n], starts, shapes) for n in names}
    if case["op"] == "step8":
        blocks = [(-(-math.prod(s) // BLOCK),) for s in shapes]
        for n in ("exp_avgs_scales", "exp_avg_rms_scales"):
            st["lists"][n] = _views(st[n], [a // BLOCK for a in starts], blocks)
    return st


# ---------------------------------------------------------------------------- one pass

def _outputs(st, norm=None, coef=None):
    out = {n: st[n] for n in ("params", "masters", "exp_avgs", "exp_avg_sqs", "exp_avg_rms",
                              "exp_avgs_scales", "exp_avg_rms_scales") if n in st}
    if norm is not None:
        out["norm"], out["coef"] = norm, coef
    return out


def _run_own(st):
    from gaussianimage_amd import adamw
    case, ls = st["case"], st["lists"]
    norm = coef = None
    if case["op"] == "norm" or case["clip"]:
        norm, coef = adamw.grad_norm(ls["grads"], max_norm=MAX_NORM)
    if case["op"] == "norm":
        return {"norm": norm, "coef": coef}
    kw = dict(step=case["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
              masters=ls.get("masters"), clip=coef)
    if case["op"] == "step32":
        adamw.adamw_step(ls["params"], ls["grads"], ls["exp_avgs"], ls["exp_avg_sqs"], **kw)
    else:
        adamw.adamw_step_8bit(ls["params"], ls["grads"], ls["exp_avgs"], ls["exp_avgs_scales"],
                              ls["exp_avg_rms"], ls["exp_avg_rms_scales"], seed=st["seed"], **kw)
    return _outputs(st, norm, coef)


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _plain_norm(grads):
    total = grads.float().square().sum(dtype=torch.float64)
    norm = total.sqrt().float()
    return norm, (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)


def _mix(x):
    """A 32-bit integer hash (two rounds of xor-shift and multiply), on int64 tensors or ints."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_words(seed, step, blocks):
    """One 32-bit word for each element: a hash of (seed, step), of the block, of the place in it."""
    key = _mix(_mix(seed) ^ (step * 0x9E3779B9 & 0xFFFFFFFF))
    block = torch.arange(blocks, device=DEVICE)
    block = _mix((key + block * 0x9E3779B9) & 0xFFFFFFFF)
    place = torch.arange(BLOCK, device=DEVICE) * 0x9E3779B9
    return _mix((block[:, None] + place) & 0xFFFFFFFF)


def _encode(x, word, floor):
    """e4m3 codes and the scale of each row of 256: the scale is the smallest power of two (2^-100
    to 2^119) with max|x| <= 448 * scale; |x| / scale goes to one of its two neighbours at random,
    by 16 random bits; ``floor``: what is not zero does not become zero."""
    a = x.abs()
    good = torch.isfinite(x)
    top = (a * good).nan_to_num(0.0).amax(1)
    k = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 135).clamp(-100, 119)
    scale = ((k + 127) << 23).view(torch.float32)
    y = a * ((127 - k) << 23).view(torch.float32)[:, None] * 2.0 ** -120
    code = ((y.view(torch.int32) + (word * 16 + 8).to(torch.int32)) >> 20).clamp(max=126)
    if floor:
        code = torch.where((code == 0) & (x > 0), 1, code)
    code = torch.where(good, code, 127)
    code = torch.where(x < 0, code + 128, code).to(torch.uint8)
    return code.view(torch.float8_e4m3fn), scale


def _run_plain(st):
    case = st["case"]
    norm = coef = None
    if case["op"] == "norm" or case["clip"]:
        norm, coef = _plain_norm(st["grads"])
    if case["op"] == "norm":
        return {"norm": norm, "coef": coef}
    b1, b2 = BETAS
    t = case["step"]
    g = st["grads"].float()
    if coef is not None:
        g = g * coef
    if case["op"] == "step32":
        m, v = st["exp_avgs"], st["exp_avg_sqs"]
    else:
        m = (st["exp_avgs"].float().view(-1, BLOCK) * st["exp_avgs_scales"][:, None]).view(-1)
        r = (st["exp_avg_rms"].float().view(-1, BLOCK) * st["exp_avg_rms_scales"][:, None]).view(-1)
        v = r * r
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    w = st["masters"] if case["master"] else st["params"].float()
    step = m / (root * (1 / math.sqrt(1 - b2 ** t)) + EPS)
    w = w * (1 - LR * DECAY) - step * (LR / (1 - b1 ** t))
    st["params"].copy_(w)
    if case["master"]:
        st["masters"].copy_(w)
    if case["op"] == "step32":
        st["exp_avgs"].copy_(m)
        st["exp_avg_sqs"].copy_(v)
        return _outputs(st, norm, coef)
    words = _random_words(st["seed"], t, m.numel() // BLOCK)
    code, scale = _encode(m.view(-1, BLOCK), words >> 16, False)
    st["exp_avgs"].copy_(code.view(-1))
    st["exp_avgs_scales"].copy_(scale)
    code, scale = _encode(root.view(-1, BLOCK), words & 0xFFFF, True)
    st["exp_avg_rms"].copy_(code.view(-1))
    st["exp_avg_rms_scales"].copy_(scale)
    return _outputs(st, norm, coef)


# ---------------------------------------------------------------------------- in 64 bits

def _exact_code(x, u, keep):
    """Values of e4m3 (before the scale) and scales, from the definition: the grid around |x|/scale
    has a spacing of 2^(e-3), e its exponent and at least -6."""
    rows = x.abs().view(-1, BLOCK)
    top = rows.amax(1)
    scale = torch.ones_like(top)
    some = top > 0
    mant, expo = torch.frexp(top[some])                     # top = mant * 2^expo, 1/2 <= mant < 1
    k = torch.where(mant <= 0.875, expo - 9, expo - 8).clamp(-100, 119).double()
    scale[some] = torch.exp2(k)
    scale[~some] = 2.0 ** -100
    a = rows / scale[:, None]
    _, e = torch.frexp(a)
    gap = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    q = torch.floor(a / gap + u.view_as(a)) * gap
    if keep:
        q = torch.where((q == 0) & (a > 0), 2.0 ** -9, q)
    q = q.clamp(max=448.0) * torch.sign(x).view_as(q)
    return q.view(-1), scale


def _exact_words(seed, t, n):
    import numpy as np
    mask = np.uint64(0xFFFFFFFF)

    def h(z):
        for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
            z = z ^ (z >> np.uint64(shift))
            z = (z * np.uint64(factor)) & mask
        return z ^ (z >> np.uint64(16))

    golden = np.uint64(0x9E3779B9)
    key = h(h(np.uint64(seed)) ^ ((np.uint64(t) * golden) & mask))
    index = np.arange(n, dtype=np.uint64)
    block = h((key + (index // np.uint64(BLOCK)) * golden) & mask)
    return h((block + (index % np.uint64(BLOCK)) * golden) & mask)


def exact(case, seed):
    st = prepare(case, seed)
    grad = st["grads"].double()
    out = {}
    c = 1.0
    if case["op"] == "norm" or case["clip"]:
        out["norm"] = torch.linalg.vector_norm(grad)
        out["coef"] = torch.minimum(torch.ones_like(out["norm"]), MAX_NORM / (out["norm"] + 1e-6))
        c = out["coef"]
    if case["op"] == "norm":
        return out
    b1, b2, t = BETAS[0], BETAS[1], case["step"]
    grad = grad * c
    if case["op"] == "step32":
        mean, square = st["exp_avgs"].double(), st["exp_avg_sqs"].double()
    else:
        mean = st["exp_avgs"].double() * st["exp_avgs_scales"].double().repeat_interleave(BLOCK)
        square = (st["exp_avg_rms"].double()
                  * st["exp_avg_rms_scales"].double().repeat_interleave(BLOCK)) ** 2
    mean = torch.lerp(grad, mean, b1)
    square = torch.lerp(grad ** 2, square, b2)
    w = st["masters" if case["master"] else "params"].double()
    w = w - LR * DECAY * w - LR * (mean / (1 - b1 ** t)) / (torch.sqrt(square / (1 - b2 ** t)) + EPS)
    out["params"] = w
    if case["master"]:
        out["masters"] = w
    if case["op"] == "step32":
        out["exp_avgs"], out["exp_avg_sqs"] = mean, square
        return out
    if mean.numel() > 30000000:                             # (the words come from the host)
        out["exp_avgs"] = out["exp_avg_rms"] = None
        out["exp_avgs_scales"] = out["exp_avg_rms_scales"] = None
        return out
    import numpy as np
    word = _exact_words(st["seed"], t, mean.numel())
    for name, x, bits, keep in (("exp_avgs", mean, word >> np.uint64(16), False),
                                ("exp_avg_rms", square.sqrt(), word & np.uint64(0xFFFF), True)):
        u = (torch.from_numpy(bits.astype(np.float64)).to(DEVICE) + 0.5) / 65536
        out[name], out[name + "_scales"] = _exact_code(x, u, keep)
    return out
