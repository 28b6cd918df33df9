"""Work of the optimizer operators over many tensors: the AdamW step with states in 32 or in 8 bits, the global gradient
norm that clips it, and the selection of state rows when the number of Gaussians changes.

Every operator has a plain form here (elementary torch operations in 32 bits, the norm's sum in 64) and the call that a
training program makes of the framework's kernels (``own``).

What 8-bit states are: the flattened tensor in blocks of 64 elements; per block one fp32 scale for the first moment
(its largest magnitude) and one for the square root u of the second moment (its largest value).  Relative to its scale the first
moment is a sign and 7 bits with 8 levels per octave, u is 8 bits with 16 levels per octave, the top level is 1 and
code 0 is 0.  A value between two levels goes up with a probability equal to its distance from the lower one, the
random number being a hash of (seed, tensor, step, element).
"""
import math

import torch

own = False

BLOCK = 64            # elements that share a scale
BETAS = (0.9, 0.999)
EPS = 1e-15           # what Gaussian training uses
WEIGHT_DECAY = 0.01
SEED = 7
STEP = 400            # updates that the states have behind them
M32 = 0xFFFFFFFF
ONE = 0x3F800000      # the bits of 1.0f

# the six parameter groups of a Gaussian model: name, shape of a row, learning rate
GROUPS = (("xyz", (3,), 1.6e-4), ("f_dc", (1, 3), 2.5e-3), ("f_rest", (15, 3), 1.25e-4), ("opacity", (1,), 0.05),
          ("scaling", (3,), 5e-3), ("rotation", (4,), 1e-3))


def listed():
    return [
        # the smallest model of the tests: what a step costs before its data does
        {"name": "step32 200", "op": "step", "bits": 32, "n": 200, "clip": False},
        # an object-scale scene with clipping; the colour gradients are column ranges of the rasterizer's (N,16,3) output
        {"name": "step32 300k clip", "op": "step", "bits": 32, "n": 300_000, "clip": True},
        # an outdoor scene: 177 M parameters
        {"name": "step32 3M", "op": "step", "bits": 32, "n": 3_000_000, "clip": False},
        # bf16 weights beside the Gaussians (fp32 value kept through a 16-bit remainder): matrices and odd vectors
        {"name": "step32 bf16 weights", "op": "weights", "bits": 32, "width": 2000, "clip": False},
        # the same four with states in 8 bits; an odd number of Gaussians, so blocks end inside a tensor
        {"name": "step8 777", "op": "step", "bits": 8, "n": 777, "clip": False},
        {"name": "step8 300k clip", "op": "step", "bits": 8, "n": 300_000, "clip": True},
        {"name": "step8 3M", "op": "step", "bits": 8, "n": 3_000_000, "clip": False},
        {"name": "step8 bf16 weights", "op": "weights", "bits": 8, "width": 2000, "clip": True},
        # the norm of a small and of a large scene's gradients
        {"name": "norm 5000", "op": "norm", "bits": 32, "n": 5000, "clip": False},
        {"name": "norm 3M", "op": "norm", "bits": 32, "n": 3_000_000, "clip": False},
        # densification of a scene: a part of the rows pruned, some cloned, new ones appended
        {"name": "rows32 3M", "op": "rows", "bits": 32, "n": 3_000_000, "clip": False},
        {"name": "rows8 300001", "op": "rows", "bits": 8, "n": 300_001, "clip": False},
    ]


def draw(rng):
    op = rng.choice(("step", "step", "step", "weights", "norm", "rows"))
    case = {"op": op, "bits": rng.choice((8, 32)) if op != "norm" else 32, "clip": op in ("step", "weights") and rng.random() < 0.5}
    if op == "weights":
        case["width"] = int(round(2 ** rng.uniform(3, math.log2(2000))))
    else:
        case["n"] = int(round(2 ** rng.uniform(0, math.log2(2_900_000))))
    return case


def _shapes(case):
    """(shapes, learning rates) of the tensors of a case."""
    if case["op"] == "weights":
        w = case["width"]
        shapes = [((w, w), (w + 1,), (w // 2 + 1, 7))[i % 3] for i in range(12)]
        return shapes, [1e-3] * len(shapes)
    return [(case["n"],) + row for _, row, _ in GROUPS], [lr for _, _, lr in GROUPS]


def _sizes(case):
    return [math.prod(s) for s in _shapes(case)[0]]


def work(case):
    elements, count, bf16 = sum(_sizes(case)), len(_sizes(case)), case["op"] == "weights"
    packed = 2 * (2 + 8 / BLOCK)                                    # 8-bit states of one element, read and written
    if case["op"] == "norm":
        return {"bytes": 4 * elements + 4, "flops": 2 * elements}
    if case["op"] == "rows":
        kept, fresh, n_new = _row_counts(case["n"])
        per = elements // case["n"]
        if case["bits"] == 32:
            return {"bytes": per * (8 * kept + 8 * n_new) + 8 * n_new, "flops": per * n_new}
        return {"bytes": per * (packed / 2 * kept + (packed / 2 + 8) * n_new) + 8 * n_new, "flops": 20 * per * n_new}
    weights = (2 + 2 + 2 + 2 + 2 + 4) if bf16 else 12               # p read and written (bf16: and its remainder, the fp32 value out), g read
    states = 16 if case["bits"] == 32 else packed + 8               # 8-bit: and the values that the codes stand for
    return {"bytes": elements * (weights + states) + 64 * count, "flops": elements * (15 if case["bits"] == 32 else 45)}


def _row_counts(n):
    """(rows taken from the old state, fresh rows, all rows) after a densification of n Gaussians."""
    pruned, cloned, fresh = n // 10, n // 20, n // 20
    kept = n - pruned + cloned
    return kept, fresh, kept + fresh


# ---- 8-bit states ---------------------------------------------------------------------------------------------------

def _mix_host(x):
    x ^= x >> 16
    x = x * 0x6A09E667 & M32
    x ^= x >> 15
    x = x * 0xBB67AE85 & M32
    return x ^ (x >> 16)


def _i32(x):
    return x - (1 << 32) if x >= 1 << 31 else x


def _random_bits(n, index, step, device):
    """32 random bits for each element of tensor `index` at update `step`, as int32."""
    key = _mix_host(_mix_host(SEED + 0x9E3779B9 * (index + 1) & M32) ^ step)
    x = torch.arange(n, dtype=torch.int32, device=device) + _i32(key)
    x = x ^ ((x >> 16) & 0xFFFF)
    x = x * _i32(0x6A09E667)
    x = x ^ ((x >> 15) & 0x1FFFF)
    x = x * _i32(0xBB67AE85)
    return x ^ ((x >> 16) & 0xFFFF)


def _blocks(x):
    """x flattened to (blocks, 64), the last block padded with zeros."""
    x = x.reshape(-1)
    pad = -x.numel() % BLOCK
    return (torch.cat([x, x.new_zeros(pad)]) if pad else x).view(-1, BLOCK)


def _relative(x):
    """(x over its block's largest value, at most 1; the scales): x not negative, (blocks, 64)."""
    scale = x.amax(dim=1, keepdim=True)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    return torch.clamp(x * inverse, max=1.0), scale


def _pack(m, u, random=None):
    """Codes (n, 2) and scales (blocks, 2) of first moments m and roots of second moments u; without random bits to the nearest level."""
    n = m.numel()
    r = _blocks(random) if random is not None else None
    xm, sm = _relative(_blocks(m.abs()))
    xu, su = _relative(_blocks(u))
    rm = (r & 0xFFFF) if r is not None else 32768
    ru = ((r >> 16) & 0xFFFF) if r is not None else 32768
    cm = 127 + ((xm.view(torch.int32) + rm * 16 - ONE) >> 20)
    lowest = 1.25 * 2.0 ** -16
    cm = torch.where(cm < 1, (xm * (65536.0 / lowest) > rm).to(torch.int32), cm)
    cm = cm + torch.where(_blocks(m) < 0, 128, 0) * (cm > 0)
    cu = 255 + ((xu.view(torch.int32) + ru * 8 - ONE) >> 19)
    cu = torch.where(xu > 0, cu.clamp(min=1), torch.zeros_like(cu))
    codes = torch.stack([cm.reshape(-1)[:n], cu.reshape(-1)[:n]], dim=1).to(torch.uint8)
    return codes, torch.cat([sm, su], dim=1)


def _unpack(codes, scales, shape):
    """(m, u) that the codes stand for."""
    c = codes.reshape(-1, 2).to(torch.int32)
    n = c.shape[0]
    s = scales.repeat_interleave(BLOCK, dim=0)[:n]
    mag = c[:, 0] & 127
    m = torch.where(mag > 0, (ONE - ((127 - mag) << 20)).view(torch.float32), 0.0) * s[:, 0]
    m = torch.where(c[:, 0] > 127, -m, m)
    u = torch.where(c[:, 1] > 0, (ONE - ((255 - c[:, 1]) << 19)).view(torch.float32), 0.0) * s[:, 1]
    return m.view(shape), u.view(shape)


# ---- fp32 values behind bf16 parameters ---------------------------------------------------------------------------

def _joined(p, low):
    """The fp32 value of a bf16 parameter and its remainder."""
    return ((p.view(torch.int16).to(torch.int32) << 16) + low.to(torch.int32)).view(torch.float32)


def _split(x):
    """x rounded to bf16 (halves away from zero) and the remainder in units of fp32's last place."""
    bits = x.view(torch.int32)
    high = (bits + 0x8000) >> 16
    return high.to(torch.int16).view(torch.bfloat16), (bits - (high << 16)).to(torch.int16)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    shapes, lrs = _shapes(case)
    bf16 = case["op"] == "weights"

    def normal(shape):
        return torch.randn(shape, generator=gen, device=dev)

    params = [normal(s) for s in shapes]
    if bf16:
        grads = [normal(s) * 1e-3 for s in shapes]
        typical = [torch.full((s[0],) + (1,) * (len(s) - 1), 1e-3, device=dev) for s in shapes]
    else:
        # gradients of a Gaussian share a size that spreads over decades; those outside the view have none
        n = case["n"]
        size = torch.exp(normal((n,)) * 1.5 - 9.0)
        seen = size * (torch.rand((n,), generator=gen, device=dev) < 0.7)
        sh = normal((n, 16, 3)) * seen.view(n, 1, 1)
        grads = [normal(s) * seen.view((n,) + (1,) * (len(s) - 1)) if name not in ("f_dc", "f_rest") else
                 sh[:, :1] if name == "f_dc" else sh[:, 1:] for (name, _, _), s in zip(GROUPS, shapes)]
        typical = [size.view((n,) + (1,) * (len(s) - 1)) for s in shapes]
    if case["op"] == "norm":
        return {"case": case, "grads": grads}
    m = [normal(s) * t * 0.3 for s, t in zip(shapes, typical)]
    u = [(normal(s) * 0.2).exp() * t for s, t in zip(shapes, typical)]
    low = None
    if bf16:
        params, low = (list(x) for x in zip(*(_split(p) for p in params)))
        grads = [g.to(torch.bfloat16) for g in grads]
    state = {"case": case, "lrs": lrs, "step": STEP, "grads": grads, "low": low}
    if case["bits"] == 8:
        state["codes"], state["scales"] = (list(x) for x in zip(*(_pack(a, b) for a, b in zip(m, u))))
        state["codes"] = [c.view(s + (2,)) for c, s in zip(state["codes"], shapes)]
    else:
        state["m"], state["v"] = m, [x * x for x in u]
    if case["op"] == "rows":
        kept, fresh, n_new = _row_counts(n)
        old = torch.arange(n, device=dev)[torch.rand((n,), generator=gen, device=dev).argsort()[: n - n // 10].sort().values]
        more = torch.randint(0, n, (kept - old.numel(),), generator=gen, device=dev)
        state["index"] = torch.cat([old, more, torch.full((fresh,), -1, dtype=torch.int64, device=dev)])
    state["params"] = params
    if own:  # the optimizer that a training program keeps, its states as they are after STEP updates
        import importlib
        impl = importlib.import_module("gaussian-splatting_amd")
        state["params"] = [torch.nn.Parameter(p) for p in params]
        opt = impl.FusedAdamW([{"params": [p], "lr": lr} for p, lr in zip(state["params"], lrs)], lr=0.0, betas=BETAS, eps=EPS,
                              weight_decay=WEIGHT_DECAY, state_bits=case["bits"], seed=SEED)
        for k, (p, g) in enumerate(zip(state["params"], grads)):
            p.grad = g
            opt.state[p] = {"step": torch.tensor(float(STEP))}
            opt.state[p].update({"moment_codes": state["codes"][k], "moment_scales": state["scales"][k]} if case["bits"] == 8
                                else {"exp_avg": state["m"][k], "exp_avg_sq": state["v"][k]})
            if bf16:
                opt.state[p]["param_low"] = low[k]
        state["opt"] = opt
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------

def _norm(grads):
    """sqrt of the sum of squares over all tensors, the sum in 64 bits."""
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()


def _step_one(state, k, coef):
    """The AdamW update of tensor k, in place; returns its new value, first and second moment."""
    b1, b2 = BETAS
    t, lr, eight = state["step"], state["lrs"][k], state["case"]["bits"] == 8
    p, g = state["params"][k], state["grads"][k].float()
    low = state["low"][k] if state["low"] is not None else None
    x = p if low is None else _joined(p, low)
    g = g if coef is None else g * coef
    if eight:
        m, u = _unpack(state["codes"][k], state["scales"][k], p.shape)
        v = u * u
    else:
        m, v = state["m"][k], state["v"][k]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    u = v.sqrt()
    denom = u * (1.0 / math.sqrt(1 - b2 ** t)) + EPS
    x = x * (1 - lr * WEIGHT_DECAY) - (m / denom) * (lr / (1 - b1 ** t))
    if low is None:
        p.copy_(x)
    else:
        high, rest = _split(x)
        p.copy_(high)
        low.copy_(rest)
    if eight:
        codes, scales = _pack(m, u, _random_bits(m.numel(), k, t, m.device))
        state["codes"][k].copy_(codes.view(state["codes"][k].shape))
        state["scales"][k].copy_(scales)
        m, u = _unpack(codes, scales, p.shape)
        v = u * u
    else:
        state["m"][k].copy_(m)
        state["v"][k].copy_(v)
    return (p, m, v) if low is None else (p, x, m, v)


def _rows_one(state, k, index, shape):
    """(first, second moments) of the selected rows of tensor k; rows outside the old ones are fresh."""
    taken = (index >= 0) & (index < shape[0])
    at = torch.where(taken, index, torch.zeros_like(index))
    taken = taken.view((-1,) + (1,) * (len(shape) - 1))
    if state["case"]["bits"] == 32:
        return tuple(torch.where(taken, x[k][at], torch.zeros_like(x[k][at])) for x in (state["m"], state["v"]))
    m, u = (torch.where(taken, x[at], torch.zeros_like(x[at])) for x in _unpack(state["codes"][k], state["scales"][k], shape))
    m, u = _unpack(*_pack(m, u), m.shape)
    return m, u * u


def run(state):
    case = state["case"]
    if own:
        import importlib
        impl = importlib.import_module("gaussian-splatting_amd")
        if case["op"] == "norm":
            return impl.grad_norm(state["grads"])
        opt, params = state["opt"], state["params"]
        if case["op"] == "rows":
            states = opt.gather_state(params, state["index"])
            return [(x["exp_avg"], x["exp_avg_sq"]) for x in opt.unpacked(states=states)]
        opt.step(max_norm=1.0 if case["clip"] else None)
        parts = opt.unpacked(params)
        out = [(p.detach(), x["exp_avg"], x["exp_avg_sq"]) if p.dtype == torch.float32 else
               (p.detach(), x["param"], x["exp_avg"], x["exp_avg_sq"]) for p, x in zip(params, parts)]
        return (out, opt.last_grad_norm) if case["clip"] else out
    if case["op"] == "norm":
        return _norm(state["grads"])
    shapes, _ = _shapes(case)
    if case["op"] == "rows":
        return [_rows_one(state, k, state["index"], s) for k, s in enumerate(shapes)]
    state["step"] += 1
    coef = norm = None
    if case["clip"]:
        norm = _norm(state["grads"])
        coef = torch.clamp(1.0 / (norm + 1e-6), max=1.0)
    out = [_step_one(state, k, coef) for k in range(len(shapes))]
    return (out, norm) if case["clip"] else out


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def _exact_states(state, k, shape):
    """First moment and second moment of tensor k before the pass, in 64 bits: level q of an octave scale is (1 + (q mod L) / L) 2^(q div L)."""
    if state["case"]["bits"] == 32:
        return state["m"][k].double(), state["v"][k].double()
    codes, scales = state["codes"][k].reshape(-1, 2), state["scales"][k]

    def level(code, top, per):
        q = code - top
        return torch.where(code > 0, torch.pow(2.0, torch.div(q, per, rounding_mode="floor").double()) * (1 + (q % per).double() / per), 0.0)

    m, v = [], []
    piece = 1 << 22                                       # elements at a time: a multiple of BLOCK
    for at in range(0, codes.shape[0], piece):
        c = codes[at:at + piece].long()
        s = scales[at // BLOCK:(at + piece) // BLOCK].double().repeat_interleave(BLOCK, dim=0)[:c.shape[0]]
        m.append(level(c[:, 0] % 128, 127, 8) * s[:, 0] * (1 - 2 * (c[:, 0] // 128)).double())
        v.append((level(c[:, 1], 255, 16) * s[:, 1]) ** 2)
    return torch.cat(m).view(shape), torch.cat(v).view(shape)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    grads = [g.double() for g in state["grads"]]
    norm = sum(float((g * g).sum()) for g in grads) ** 0.5
    if case["op"] == "norm":
        return torch.tensor(norm, dtype=torch.float64)
    shapes, lrs = _shapes(case)
    if case["op"] == "rows":
        if case["bits"] == 8:
            return None                                   # which of two levels a value goes to has no 64-bit answer
        index = state["index"]
        out = []
        for k, s in enumerate(shapes):
            pair = []
            for x in _exact_states(state, k, s):
                y = torch.zeros((index.numel(),) + s[1:], dtype=torch.float64, device=x.device)
                y[index >= 0] = x[index[index >= 0]]
                pair.append(y)
            out.append(tuple(pair))
        return out
    t = STEP + 1
    scale = min(1.0, 1.0 / (norm + 1e-6)) if case["clip"] else 1.0
    out = []
    for k, s in enumerate(shapes):
        m, v = _exact_states(state, k, s)
        x = state["params"][k].double() if state["low"] is None else _joined(state["params"][k], state["low"][k]).double()
        g = grads[k] * scale
        m = BETAS[0] * m + (1 - BETAS[0]) * g
        v = BETAS[1] * v + (1 - BETAS[1]) * g ** 2
        new = x - lrs[k] * WEIGHT_DECAY * x - lrs[k] * (m / (1 - BETAS[0] ** t)) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS)
        states = (m, v) if case["bits"] == 32 else (None, None)
        out.append((new,) + (() if state["low"] is None else (new,)) + states)
    return (out, torch.tensor(norm, dtype=torch.float64)) if case["clip"] else out
