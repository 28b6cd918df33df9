"""GPU: FusedAdamW, grad_norm, gather_state / replace_params and unpacked (csrc/adamw.hip through the C-ABI).

Against torch.optim.AdamW bit for bit (32-bit states), against the formulas in float64 with bounds counted in roundings, against the
oracle's 8-bit codes one by one (oracle/adamw_oracle.py).  With e = 2^-24, half a step of float32 relative to the value, the
update of one element makes at most these roundings:
    m      beta, 1 - beta, two products, a sum (or their fma form)              <= 5 e (|beta1 m| + |(1 - beta1) g|)
    v      the same, g * g, and u * u where u is what is kept                   <= 8 e v
    u, d   half of v's, the root, bc2, the quotient or product, eps, the sum    <= 10 e d
    update m's, d's, the division (1 ulp = 2 e), the step size, the product     <= 15 e |update| + 5 e |step| size / d
    p      1 - lr wd, the product, the sum                                      <= 3 e |p| + e |new p|
Clipping adds the coefficient (norm, + 1e-6, division, max_norm: 4) and its product to g: 5 e of g, 10 e of g^2; 11 e covers it in
|update|.  A bfloat16 parameter adds half a step of bfloat16 to the parameter, none to the value behind it.
"""
import importlib
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from oracle import adamw_oracle as orc  # noqa: E402

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
SIZES = [1, 2, 63, 64, 65, 255, 257, 2047, 2049, 100_003]


@pytest.fixture(scope="module")
def impl():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return importlib.import_module("gaussian-splatting_amd")


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _np(t):
    t = t.detach()
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy()


def _bits16(t):
    return t.detach().view(torch.int16).cpu().numpy().view(np.uint16)


def _inputs(n, seed, decades=3.0):
    """p, g, m, u of n elements: gradients whose size spreads over decades, a fifth of them zero."""
    r = np.random.default_rng(seed)
    size = np.exp(r.normal(0, decades, n) - 6)
    g = (r.standard_normal(n) * size * (r.random(n) < 0.8)).astype(np.float32)
    m = (r.standard_normal(n) * size * 0.3).astype(np.float32)
    u = (np.exp(r.normal(0, 0.3, n)) * size).astype(np.float32)
    return r.standard_normal(n).astype(np.float32), g, m, u


HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-15, weight_decay=0.02)


def _put(opt, p, t, m, u, bits, low=None):
    """Gives p the state of t updates; returns the float64 moments that the state stands for."""
    dev = p.device
    state = {"step": torch.tensor(float(t))}
    if bits == 8:
        codes, scales = orc.pack(m, u)
        state["moment_codes"] = torch.from_numpy(codes).to(dev).view(p.shape + (2,))
        state["moment_scales"] = torch.from_numpy(scales).to(dev)
        s = np.repeat(scales, 64, axis=0)[:m.size]
        out = orc.level_m(codes[:, 0], s[:, 0]), orc.level_u(codes[:, 1], s[:, 1]) ** 2
    else:
        v = u * u
        state["exp_avg"], state["exp_avg_sq"] = torch.from_numpy(m).to(dev).view(p.shape), torch.from_numpy(v).to(dev).view(p.shape)
        out = m.astype(np.float64), v.astype(np.float64)
    if low is not None:
        state["param_low"] = torch.from_numpy(low).to(dev).view(p.shape)
    opt.state[p] = state
    return out


def _check_value(got, start, ref, upd, size, d, t, clip=False, hyper=HYPER):
    step = hyper["lr"] / (1 - hyper["betas"][0] ** t)
    tol = E * (3 * np.abs(start) + np.abs(ref) + (26 if clip else 15) * upd + (10 if clip else 5) * step * size / d) + 1e-44
    err = np.abs(got.astype(np.float64) - ref)
    assert np.all(err <= tol), (float((err / tol).max()), int((err > tol).sum()))


# ---- the step ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 777, 40_000])
def test_32_bit_states_equal_torch_adamw_bit_for_bit(impl, dev, n):
    shapes = {"xyz": (n, 3), "f_rest": (n, 15, 3), "opacity": (n, 1), "scalar": ()}
    gen = torch.Generator().manual_seed(n)
    start = {k: torch.randn(s, generator=gen) for k, s in shapes.items()}
    a = {k: torch.nn.Parameter(v.to(dev)) for k, v in start.items()}
    b = {k: torch.nn.Parameter(v.to(dev)) for k, v in start.items()}

    def groups(p):
        return [{"params": [p["xyz"]], "lr": 1.6e-4, "weight_decay": 0.0}, {"params": [p["f_rest"], p["opacity"]], "lr": 0.02},
                {"params": [p["scalar"]], "betas": (0.8, 0.95), "eps": 1e-8}]

    ref = torch.optim.AdamW(groups(a), lr=1e-3, eps=1e-15, weight_decay=0.1, foreach=True)
    opt = impl.FusedAdamW(groups(b), lr=1e-3, eps=1e-15, weight_decay=0.1)
    for t in range(1, 6):
        for o in (ref, opt):
            o.param_groups[0]["lr"] = 1.6e-4 * 0.9 ** t
        for k in shapes:
            g = torch.randn(shapes[k], generator=gen) * 10 ** (torch.rand((), generator=gen) * 4 - 3)
            a[k].grad, b[k].grad = g.to(dev), g.to(dev)
        if t == 3:
            a["opacity"].grad = b["opacity"].grad = None          # skipped: its count stays behind the others'
        ref.step()
        opt.step()
        for k in shapes:
            s, r = opt.state[b[k]], ref.state[a[k]]
            assert torch.equal(s["exp_avg"], r["exp_avg"]) and torch.equal(s["exp_avg_sq"], r["exp_avg_sq"]), (k, t)
            assert torch.equal(a[k], b[k]), (k, t)
            assert float(s["step"]) == float(r["step"]) == (t if k != "opacity" or t < 3 else t - 1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("n", SIZES)
def test_step_against_float64(impl, dev, n, clip, bf16, bits):
    p, g, m, u = _inputs(n, n + bits)
    t = 7
    low = None
    if bf16:
        high, low = orc.split(p)
        param = torch.nn.Parameter(torch.from_numpy(high.view(np.int16)).to(dev).view(torch.bfloat16))
        param.grad = torch.from_numpy(g).to(dev).bfloat16()
        g = _np(param.grad)
    else:
        param = torch.nn.Parameter(torch.from_numpy(p.copy()).to(dev))
        param.grad = torch.from_numpy(g).to(dev)
    opt = impl.FusedAdamW([param], state_bits=bits, seed=5, **HYPER)
    m64, v64 = _put(opt, param, t - 1, m, u, bits, low)
    norm = math.sqrt(float((g.astype(np.float64) ** 2).sum()))
    max_norm = 0.25 * norm if clip else None
    if clip and norm == 0:
        max_norm = 1.0
    before = param.grad.clone()
    opt.step(max_norm=max_norm)
    assert torch.equal(param.grad, before)                        # gradients are never rewritten
    coef = min(1.0, max_norm / (norm + 1e-6)) if clip else 1.0
    ref, m1, v1, upd, size, d = orc.step64(p, g, m64, v64, t, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], coef)
    state = opt.state[param]
    assert float(state["step"]) == t
    value = opt.unpacked([param])[0]
    _check_value(_np(value["param"]), p, ref, upd, size, d, t, clip)
    if bf16:
        x = _np(value["param"])
        assert np.array_equal(orc.join(_bits16(param), _np(state["param_low"])).view(np.uint32), x.view(np.uint32))
        assert np.all(np.abs(_np(param) - x) <= np.abs(x) * 2.0 ** -8 + 2.0 ** -134)
    if bits == 32:
        assert np.all(np.abs(_np(state["exp_avg"]) - m1) <= (10 if clip else 5) * E * size + 1e-44)
        assert np.all(np.abs(_np(state["exp_avg_sq"]) - v1) <= (18 if clip else 8) * E * v1 + 1e-44)
    else:
        codes, scales = _np(state["moment_codes"]).reshape(-1, 2), _np(state["moment_scales"])
        s = np.repeat(scales, 64, axis=0)[:n].astype(np.float64)
        # off by less than one level of its octave, the first moment at the bottom by its lowest level
        for col, level, x, per, low_level in ((0, orc.level_m, m1, 8, 1.25 * 2.0 ** -16), (1, orc.level_u, np.sqrt(v1), 16, 2.0 ** -15.87)):
            got = level(codes[:, col], s[:, col])
            gap = np.exp2(np.floor(np.log2(np.maximum(np.abs(x) / s[:, col], low_level)))) * s[:, col] / per
            assert np.all(np.abs(got - x) <= np.maximum(gap, low_level * s[:, col]) * (1 + 1e-5) + 12 * E * (size if col == 0 else x)), col
        assert np.all((codes[:, 1] > 0) | (v1 < 1e-44))           # a second moment is never rounded away


@pytest.mark.parametrize("stochastic", [False, True])
@pytest.mark.parametrize("n", SIZES)
def test_codes_equal_the_oracles_one_by_one(impl, dev, n, stochastic):
    p, g, m, u = _inputs(n, 3 * n + 1)
    first, param = (torch.nn.Parameter(torch.from_numpy(x.copy()).to(dev)) for x in (np.ones(5, np.float32), p))
    opt = impl.FusedAdamW([first, param], state_bits=8, stochastic_rounding=stochastic, seed=123, **HYPER)
    _put(opt, param, 0, m, u, 8)
    codes, scales = orc.pack(m, u)
    for t in range(1, 4):
        param.grad = torch.from_numpy(g).to(dev)
        opt.step()
        rnd = orc.random_bits(n, 123, 1, t) if stochastic else None
        _, codes, scales = orc.step8(p, g, codes, scales, t, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], rnd)
        assert np.array_equal(_np(opt.state[param]["moment_scales"]), scales), t
        assert np.array_equal(_np(opt.state[param]["moment_codes"]).reshape(-1, 2), codes), t
        value = opt.unpacked([param])[0]
        mm, uu = orc.unpack(codes, scales)
        assert np.array_equal(_np(value["exp_avg"]), mm) and np.array_equal(_np(value["exp_avg_sq"]), uu * uu)
        g = (g * np.float32(-1.7)).astype(np.float32)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_results_do_not_depend_on_alignment_or_strides(impl, dev, shift, dtype, bits):
    """The same tensors as views that start `shift` elements into their storage, and gradients that are column ranges of a wider
    tensor or transposed: the same bits as from fresh contiguous ones."""
    gen = torch.Generator().manual_seed(shift)
    shapes = [(300, 15, 3), (301, 1, 3), (1000,), (65, 64), (1, 7)]
    opts, params = [], []
    for variant in range(3):
        gen.manual_seed(shift)
        ps = []
        for s in shapes:
            x = torch.randn(s, generator=gen).to(dtype)
            g = torch.randn(s, generator=gen).to(dtype)
            if variant:
                store = torch.zeros(x.numel() + 16, dtype=dtype, device=dev)
                view = store[shift:shift + x.numel()].view(s)
                view.copy_(x)
                p = torch.nn.Parameter(view)
                assert p.data_ptr() == view.data_ptr()
            else:
                p = torch.nn.Parameter(x.to(dev))
            if variant == 1:
                wide = torch.full((s[0], math.prod(s[1:]) + 5), float("nan"), dtype=dtype, device=dev)
                gv = wide[:, 2:2 + math.prod(s[1:])]
                gv.copy_(g.view(s[0], -1))
                p.grad = gv.unflatten(1, s[1:]) if len(s) > 1 else gv[:, 0]
            elif variant == 2 and len(s) == 2:
                p.grad = g.t().contiguous().to(dev).t()
            else:
                p.grad = g.to(dev)
            ps.append(p)
        opt = impl.FusedAdamW(ps, lr=0.01, eps=1e-8, weight_decay=0.1, state_bits=bits, seed=1)
        for _ in range(3):
            opt.step(max_norm=0.5)
        opts.append(opt)
        params.append(ps)
    for k in range(len(shapes)):
        for v in (1, 2):
            assert torch.equal(params[0][k], params[v][k]), (k, v)
            for name, x in opts[0].state[params[0][k]].items():
                assert torch.equal(x, opts[v].state[params[v][k]][name]), (k, v, name)
    assert torch.equal(opts[0].last_grad_norm, opts[1].last_grad_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_of_all_sizes_types_and_states(impl, dev, bits):
    """150 tensors, several launches, groups of both types and both forms of state: each as if it were alone."""
    gen = torch.Generator().manual_seed(2)
    sizes = [0, 1, 3, 64, 65, 1000, 4097] * 22
    params = [torch.nn.Parameter(torch.randn(n, generator=gen).to(dev, torch.bfloat16 if i % 3 == 0 else torch.float32)) for i, n in enumerate(sizes[:150])]
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    groups = [{"params": params[:70], "state_bits": 40 - bits}, {"params": params[70:], "state_bits": bits, "lr": 0.3}]
    opt = impl.FusedAdamW(groups, lr=0.1, seed=4)
    for _ in range(2):
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen).to(dev, p.dtype)
        before = [p.grad.clone() for p in params]
        opt.step()
        for i, (p, q) in enumerate(zip(params, alone)):
            q.grad = before[i]
            if not hasattr(q, "opt"):
                # the tensor's place in the optimizer is part of the random bits: parameters without gradients before it
                dummies = [torch.nn.Parameter(torch.zeros(1, device=dev)) for _ in range(i)]
                q.opt = impl.FusedAdamW(dummies + [q], lr=0.1 if i < 70 else 0.3, seed=4, state_bits=40 - bits if i < 70 else bits)
            q.opt.step()
            assert torch.equal(p, q), i
            for name, x in opt.state[p].items():
                assert torch.equal(x, q.opt.state[q][name]), (i, name)


def test_seeds_and_repeatability(impl, dev):
    def run(seed, stochastic=True):
        p = torch.nn.Parameter(torch.ones(5000, device=dev))
        opt = impl.FusedAdamW([p], lr=0.1, state_bits=8, seed=seed, stochastic_rounding=stochastic)
        gen = torch.Generator().manual_seed(0)
        for _ in range(3):
            p.grad = torch.randn(5000, generator=gen).to(dev)
            opt.step()
        return opt.state[p]["moment_codes"]
    assert torch.equal(run(1), run(1)) and torch.equal(run(1, False), run(2, False))
    assert (run(1) != run(2)).float().mean() > 0.3


def test_stochastic_rounding_follows_a_slow_second_moment(impl, dev):
    """Gradients of constant size after a long rest: v has to grow to their square within 1 / (1 - beta2) updates, by less than a level
    each.  Element 0 of each block keeps the scale high.  u after T updates is u_T = g sqrt(1 - beta2^T); a run of one element
    scatters by less than a quarter of it, the mean of 64 * 63 independent ones by less than 1 / 60 of that."""
    n, T = 64 * 64, 600
    p = torch.nn.Parameter(torch.zeros(n, device=dev))
    opt = impl.FusedAdamW([p], lr=0.0, state_bits=8, betas=(0.9, 0.99), weight_decay=0.0)
    g = torch.full((n,), 1e-2, device=dev)
    g[::64] = 1.0
    p.grad = g
    for _ in range(T):
        opt.step()
    u = opt.unpacked([p])[0]["exp_avg_sq"].sqrt().view(64, 64)[:, 1:]
    expect = 1e-2 * math.sqrt(1 - 0.99 ** T)
    assert abs(float(u.mean()) - expect) <= expect * (0.25 / 60 * 5 + 1 / 32)     # 5 sigma, and the curvature of the root over a level
    m = opt.unpacked([p])[0]["exp_avg"].view(64, 64)[:, 1:]
    assert abs(float(m.mean()) - 1e-2) <= 1e-2 * (0.25 / 60 * 5)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_and_non_finite_gradients(impl, dev, bits):
    p = torch.nn.Parameter(torch.ones(256, device=dev))
    opt = impl.FusedAdamW([p], lr=0.1, state_bits=bits, weight_decay=0.5, eps=1e-8)
    p.grad = torch.zeros(256, device=dev)
    opt.step()                                    # nothing but the decay
    assert torch.equal(p.detach(), torch.full_like(p, 1 - 0.1 * 0.5))
    got = opt.unpacked([p])[0]
    assert not got["exp_avg"].any() and not got["exp_avg_sq"].any()
    p.grad = torch.ones(256, device=dev)
    p.grad[70] = float("nan")
    p.grad[200] = float("inf")
    opt.step()
    x = p.detach()
    bad = torch.zeros(256, dtype=torch.bool, device=dev)
    bad[70] = bad[200] = True
    assert torch.equal(x.isnan(), bad)
    p.grad = torch.ones(256, device=dev)
    opt.step()
    if bits == 8:                                 # the whole block of the NaN, the infinity's own element
        bad[64:128] = True
        got = opt.unpacked([p])[0]
        assert not got["exp_avg"][192:200].any()  # the infinity's neighbours start over while it is there
    assert torch.equal(p.detach().isnan(), bad)
    # a NaN norm reaches everything, as with torch.nn.utils.clip_grad_norm_
    q = torch.nn.Parameter(torch.ones(100, device=dev))
    opt = impl.FusedAdamW([q], lr=0.1, state_bits=bits)
    q.grad = torch.ones(100, device=dev)
    q.grad[3] = float("nan")
    opt.step(max_norm=1.0)
    assert q.detach().isnan().all() and opt.last_grad_norm.isnan()


def test_tiny_moments_and_huge_ratios_stay_bounded(impl, dev):
    """Within a block: gradients over 30 decades.  No update exceeds what Adam allows, |m| / u <= (1 - beta1) / sqrt(1 - beta2) with the
    first update's corrections: lr (1 + a level of m) each."""
    n = 64 * 50
    gen = torch.Generator().manual_seed(1)
    g = (10 ** (torch.rand(n, generator=gen) * 30 - 18)).to(dev)
    p = torch.nn.Parameter(torch.zeros(n, device=dev))
    opt = impl.FusedAdamW([p], lr=1.0, state_bits=8, eps=1e-30, weight_decay=0.0)
    p.grad = g
    opt.step()
    assert torch.isfinite(p).all() and float(p.detach().abs().max()) <= 1.0 + 20 * E
    for _ in range(20):
        before = p.detach().clone()
        opt.step()
        assert torch.isfinite(p).all()
        assert float((p.detach() - before).abs().max()) <= 1.5      # u of 0 would give g / eps


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_beyond_32_bits(impl, dev, bits):
    """2^32 + 130 elements: the ends of the tensor, and both sides of element 2^32, against the oracle."""
    n = (1 << 32) + 130
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=dev))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    opt = impl.FusedAdamW([p], state_bits=bits, seed=3, **HYPER)
    r = np.random.default_rng(0)
    at = [0, (1 << 31) - 64, (1 << 32) - 64, (1 << 32) + 64]
    vals = []
    for a in at:
        g = torch.from_numpy(r.standard_normal(66 if a == at[-1] else 128).astype(np.float32)).bfloat16()
        p.grad[a:a + g.numel()] = g.to(dev)
        vals.append(g.float().numpy())
    norm = impl.grad_norm([p.grad])
    assert abs(float(norm) - math.sqrt(sum(float((v.astype(np.float64) ** 2).sum()) for v in vals))) <= float(norm) * 2 * E
    opt.step()
    state = opt.state[p]
    for a, g in zip(at, vals):
        k = g.size
        if bits == 8:
            blocks = (k + 63) // 64
            _, codes, scales = orc.step8(np.zeros(k), g, np.zeros((k, 2), np.uint8), np.zeros((blocks, 2), np.float32), 1, HYPER["lr"],
                                         *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], orc.random_bits(k, 3, 0, 1, first=a))
            assert np.array_equal(_np(state["moment_codes"][a:a + k]), codes), a
            assert np.array_equal(_np(state["moment_scales"][a // 64:a // 64 + blocks]), scales), a
        else:
            assert np.all(np.abs(_np(state["exp_avg"][a:a + k]) - 0.1 * g.astype(np.float64)) <= 5 * E * np.abs(g)), a
        ref = orc.step64(np.zeros(k), g, np.zeros(k), np.zeros(k), 1, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])[0]
        assert np.all(np.abs(_np(p[a:a + k]) - ref) <= np.abs(ref) * (2.0 ** -8 + 30 * E)), a
    assert not p[200:1 << 20].any()
    index = torch.tensor([n - 1, 0, 1 << 32, -1], device=dev)
    got = opt.gather_state([p], index)[0]
    full = opt.unpacked(states=[got])[0]["exp_avg"]
    expect = np.array([vals[3][-1], vals[0][0], 0.0, 0.0]) * 0.1
    expect[2] = vals[2][64] * 0.1
    assert np.all(np.abs(_np(full) - expect) <= np.abs(expect) * (2.0 ** -3 if bits == 8 else 1e-6))


# ---- the norm -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [[1], [0, 5], [64, 8191, 8192, 8193], [3, 1_000_003], [7] * 200, [0]])
def test_grad_norm_against_float64(impl, dev, sizes):
    gen = torch.Generator().manual_seed(len(sizes))
    for dtypes in ((torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)):
        grads = [(torch.randn(n, generator=gen) * 10 ** (torch.rand((), generator=gen) * 8 - 4)).to(dev, dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]
        ref = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        got = impl.grad_norm(grads)
        assert got.shape == () and got.dtype == torch.float32
        assert abs(float(got) - ref) <= ref * 1.001 * E
        assert torch.equal(impl.grad_norm(grads + [None]), got)            # the same order every time


def test_grad_norm_range_strides_and_non_finite(impl, dev):
    big = torch.full((1000,), 1e30, device=dev)
    assert abs(float(impl.grad_norm(big)) / (1e30 * math.sqrt(1000)) - 1) <= 4 * E        # squares pass fp32's range
    small = torch.full((1000,), 1e-30, device=dev)
    assert abs(float(impl.grad_norm([small])) / (1e-30 * math.sqrt(1000)) - 1) <= 4 * E
    assert float(impl.grad_norm(torch.zeros(70, device=dev))) == 0.0
    x = torch.randn(50, 16, 3, device=dev)
    for view in (x[:, :1], x[:, 1:], x.transpose(0, 2), x[0, 0, 0].expand(9), x[::3, 2]):
        assert abs(float(impl.grad_norm([view])) / float(view.double().square().sum().sqrt()) - 1) <= 1.001 * E
    x[3, 4, 1] = float("inf")
    assert float(impl.grad_norm([x])) == float("inf")
    x[2, 2, 2] = float("nan")
    assert math.isnan(float(impl.grad_norm([x])))
    with pytest.raises(RuntimeError, match="bfloat16"):
        impl.grad_norm(torch.ones(4, dtype=torch.float16, device=dev))
    with pytest.raises(RuntimeError, match="bfloat16"):
        impl.grad_norm(torch.ones(4, dtype=torch.int64, device=dev))


def test_clip_matches_torch_and_takes_a_given_norm(impl, dev):
    gen = torch.Generator().manual_seed(8)
    shapes = [(500, 3), (77,), (500, 15, 3)]
    a, b, c = ([torch.nn.Parameter(torch.ones(s, device=dev)) for s in shapes] for _ in range(3))
    ref = torch.optim.AdamW(a, lr=0.01, foreach=True)
    opt, given = impl.FusedAdamW(b, lr=0.01), impl.FusedAdamW(c, lr=0.01)
    for scale in (1e-4, 1.0, 50.0):                                 # below and above the limit
        for x, y, z in zip(a, b, c):
            g = (torch.randn(x.shape, generator=gen) * scale).to(dev)
            x.grad, y.grad, z.grad = g.clone(), g, g
        norm = torch.nn.utils.clip_grad_norm_(a, 1.0)
        ref.step()
        opt.step(max_norm=1.0)
        given.step(max_norm=1.0, grad_norm=impl.grad_norm([z.grad for z in c]))
        assert abs(float(opt.last_grad_norm) / float(norm) - 1) <= 64 * E      # torch's norms of the tensors are fp32 sums
        for x, y, z in zip(a, b, c):
            assert torch.equal(y, z)
            assert float((x - y).detach().abs().max()) <= 1e-6                  # lr 0.01 times the relative difference, and a rounding of 1
    opt.step()
    assert opt.last_grad_norm is None
    for bad in (1.0, torch.ones((), device=dev, dtype=torch.float64), torch.ones(2, device=dev), torch.ones(())):
        with pytest.raises(ValueError, match="grad_norm"):
            opt.step(max_norm=1.0, grad_norm=bad)


# ---- rows -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n,m", [(1, 1), (5, 0), (0, 7), (777, 900), (4096, 1000), (20_001, 30_011)])
def test_gather_state(impl, dev, n, m, bits, dtype):
    r = np.random.default_rng(n + m)
    rows = [(3,), (1, 3), (15, 3), (1,), (4,), ()]
    params = [torch.nn.Parameter(torch.zeros((n,) + s, dtype=dtype, device=dev)) for s in rows]
    opt = impl.FusedAdamW(params, state_bits=bits, lr=0.1)
    raw = []
    for p in params:
        _, _, mm, uu = _inputs(p.numel(), 5)
        low = r.integers(-30000, 30000, p.numel()).astype(np.int16) if dtype == torch.bfloat16 else None
        _put(opt, p, 11, mm, uu, bits, low)
        raw.append((mm, uu, low))
    index = r.integers(0, max(n, 1), m) if n else np.zeros(m, np.int64)
    index[r.random(m) < 0.1] = -1
    if m > 4:
        index[:4] = (n, -(1 << 40), 1 << 40, np.iinfo(np.int64).min)       # all outside: fresh rows
        index[5] = index[6]
    taken = (index >= 0) & (index < n)
    kept = {id(p): {k: v.clone() for k, v in opt.state[p].items()} for p in params}
    got = opt.gather_state(params, torch.from_numpy(index).to(dev))
    for p, s, state, (mm, uu, low) in zip(params, rows, got, raw):
        assert float(state["step"]) == 11 and state["step"].data_ptr() != opt.state[p]["step"].data_ptr()
        for k, v in kept[id(p)].items():
            assert torch.equal(v, opt.state[p][k])                          # the old state is as it was
        per = math.prod(s)
        full = lambda x: np.where(taken.reshape(-1, 1), x.reshape(n, per)[np.where(taken, index, 0)], 0) if n else np.zeros((m, per), x.dtype)  # noqa: E731
        if bits == 32:
            assert np.array_equal(_np(state["exp_avg"]).reshape(m, per), full(mm))
            assert np.array_equal(_np(state["exp_avg_sq"]).reshape(m, per), full(uu * uu))
        else:
            a, b = orc.unpack(*orc.pack(mm, uu))
            codes, scales = orc.pack(full(a).astype(np.float32).reshape(-1), full(b).astype(np.float32).reshape(-1))
            assert np.array_equal(_np(state["moment_codes"]).reshape(-1, 2), codes)
            assert np.array_equal(_np(state["moment_scales"]), scales)
            assert state["moment_codes"].shape == (m,) + s + (2,)
        if low is not None:
            assert np.array_equal(_np(state["param_low"]).reshape(m, per), full(low))


def test_replace_params_prunes_and_appends(impl, dev):
    """The reference's surgery: prune by mask, clone, append; the step afterwards continues with the rows' own moments."""
    gen = torch.Generator().manual_seed(4)
    n = 1000
    shapes = [(n, 3), (n, 15, 3), (n, 1)]
    params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(dev)) for s in shapes]
    other = torch.nn.Parameter(torch.zeros(7, device=dev))
    opt = impl.FusedAdamW([{"params": [p], "lr": 0.01 * (k + 1), "state_bits": 32 if k else 8} for k, p in enumerate(params)] + [{"params": [other]}], lr=0.1)
    for p in params + [other]:
        p.grad = torch.randn(p.shape, generator=gen).to(dev)
    opt.step()
    mask = torch.rand(n, generator=gen).to(dev) > 0.3
    index = torch.cat([mask.nonzero()[:, 0], torch.arange(20, device=dev), torch.full((10,), -1, device=dev)])
    new = [torch.nn.Parameter(p.detach()[index.clamp(min=0)]) for p in params]
    before = [{k: v.clone() for k, v in opt.state[p].items()} for p in params]
    opt.replace_params(params, new, index)
    assert [g["params"][0] is q for g, q in zip(opt.param_groups, new + [other])] == [True] * 4
    assert all(p not in opt.state for p in params) and other in opt.state
    for k, q in enumerate(new[1:], 1):
        expect = torch.where((index >= 0).view((-1,) + (1,) * (q.dim() - 1)), before[k]["exp_avg"][index.clamp(min=0)], torch.zeros((), device=dev))
        assert torch.equal(opt.state[q]["exp_avg"], expect) and float(opt.state[q]["step"]) == 1
    for q in new:
        q.grad = torch.randn(q.shape, generator=gen).to(dev)
    opt.step()
    assert float(opt.state[new[0]]["step"]) == 2 and float(opt.state[other]["step"]) == 2
    # a parameter without a state is replaced too; refused: what the reference's torch surgery would leave behind for 8 bits
    fresh = torch.nn.Parameter(torch.zeros(3, device=dev))
    opt.add_param_group({"params": [fresh]})
    opt.replace_params([fresh], [torch.nn.Parameter(torch.zeros(2, device=dev))], torch.tensor([0, -1], device=dev))
    q = new[0]
    opt.state[q]["moment_codes"] = opt.state[q]["moment_codes"][:5]
    with pytest.raises(RuntimeError, match="replace_params"):
        opt.step()
    twin = torch.nn.Parameter(new[2].detach().clone())
    opt.add_param_group({"params": [twin]})
    with pytest.raises(ValueError, match="already"):
        opt.replace_params([new[2]], [twin], torch.arange(twin.shape[0], device=dev))


# ---- graphs, streams, errors ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_steps_count_on(impl, dev, dtype, bits):
    """A captured, clipped step replayed with new gradients and learning rates, other work in between: the same bits as eager steps."""
    gen = torch.Generator().manual_seed(6)
    shapes = [(1000, 3), (333,), (64, 65)]
    start = [torch.randn(s, generator=gen).to(dtype) for s in shapes]
    a, b = ([torch.nn.Parameter(x.to(dev)) for x in start] for _ in range(2))
    lr = torch.tensor(0.02, device=dev)
    opt = impl.FusedAdamW([{"params": a[:1], "lr": lr}, {"params": a[1:], "betas": (0.8, 0.99)}], lr=0.01, state_bits=bits, capturable=True, seed=2)
    ref = impl.FusedAdamW([{"params": b[:1], "lr": 0.02}, {"params": b[1:], "betas": (0.8, 0.99)}], lr=0.01, state_bits=bits, seed=2)
    for p, q in zip(a, b):
        p.grad = torch.zeros_like(p)
        q.grad = torch.zeros_like(q)

    def feed(k):
        new = float(np.float32(0.02 * 0.9 ** k))
        lr.fill_(new)
        ref.param_groups[0]["lr"] = new
        for p, q in zip(a, b):
            g = (torch.randn(p.shape, generator=gen) * 3).to(dev, dtype)
            p.grad.copy_(g)
            q.grad.copy_(g)

    feed(0)
    opt.step(max_norm=2.0)
    ref.step(max_norm=2.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(max_norm=2.0)
    for k in range(1, 6):
        feed(k)
        graph.replay()
        ref.step(max_norm=2.0)
        junk = torch.randn(1 << 16, device=dev).sum()                       # the program's own work and waits between replays
        torch.cuda.synchronize()
        assert torch.isfinite(junk)
        assert torch.equal(opt.last_grad_norm, ref.last_grad_norm)
        for p, q in zip(a, b):
            assert float(opt.state[p]["step"]) == float(ref.state[q]["step"]) == k + 1
            assert torch.equal(p, q), k
            for name in opt.state[p]:
                if name != "step":
                    assert torch.equal(opt.state[p][name], ref.state[q][name]), (k, name)
    opt.step(max_norm=2.0)                                                   # and eager again
    assert float(opt.state[a[0]]["step"]) == 7


def test_capture_refusals(impl, dev):
    p = torch.nn.Parameter(torch.ones(10, device=dev))
    p.grad = torch.ones(10, device=dev)
    for capturable, message in ((False, "capturable=True"), (True, "before the capture")):
        opt = impl.FusedAdamW([p], capturable=capturable)
        if not capturable:
            opt.step()
        before = p.detach().clone()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=message):
            with torch.cuda.graph(graph):
                opt.step()
        torch.cuda.synchronize()
        assert torch.equal(p.detach(), before) and (capturable or float(opt.state[p]["step"]) == 1)


def test_counts_move_to_the_gpu_outside_captures_only(impl, dev):
    """capturable switched on for states that count on the host: refused during a capture, moved by the next eager step."""
    p = torch.nn.Parameter(torch.ones(10, device=dev))
    p.grad = torch.ones(10, device=dev)
    opt = impl.FusedAdamW([p], lr=0.1)
    opt.step()
    opt.param_groups[0]["capturable"] = True
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), before) and not opt.state[p]["step"].is_cuda
    opt.step()
    assert opt.state[p]["step"].is_cuda and float(opt.state[p]["step"]) == 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    opt.param_groups[0]["capturable"] = False
    opt.step()
    assert float(opt.state[p]["step"]) == 4
    q = torch.nn.Parameter(torch.ones(10, device=dev))
    q.grad = torch.ones(10, device=dev)
    ref = torch.optim.AdamW([q], lr=0.1)
    for _ in range(4):
        ref.step()
    assert torch.equal(p, q)


def test_steps_on_two_streams(impl, dev):
    """Two optimizers at once on streams of their own: no shared workspace."""
    gen = torch.Generator().manual_seed(1)
    grads = [torch.randn(200_003, generator=gen).to(dev) for _ in range(4)]
    ref = []
    for k in range(2):
        q = torch.nn.Parameter(torch.zeros(200_003, device=dev))
        o = impl.FusedAdamW([q], lr=0.1, state_bits=8, capturable=True)
        for j in range(6):
            q.grad = grads[2 * k + j % 2]
            o.step(max_norm=3.0)
        ref.append(q.detach().clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    params = [torch.nn.Parameter(torch.zeros(200_003, device=dev)) for _ in range(2)]
    opts = [impl.FusedAdamW([p], lr=0.1, state_bits=8, capturable=True) for p in params]
    torch.cuda.synchronize()
    for j in range(6):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                params[k].grad = grads[2 * k + j % 2]
                opts[k].step(max_norm=3.0)
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(params[k].detach(), ref[k])


def test_gpu_refusals_leave_everything_as_it_was(impl, dev):
    p = torch.nn.Parameter(torch.ones(64, device=dev))
    q = torch.nn.Parameter(torch.ones(64, device=dev))
    opt = impl.FusedAdamW([{"params": [p]}, {"params": [q], "state_bits": 8}], lr=0.1)
    p.grad, q.grad = torch.ones(64, device=dev), torch.ones(64, device=dev)
    opt.step()
    before = [x.detach().clone() for x in (p, q)]

    def refused(error, match, **kw):
        with pytest.raises(error, match=match):
            opt.step(**kw)
        assert torch.equal(p.detach(), before[0]) and torch.equal(q.detach(), before[1])
        assert float(opt.state[p]["step"]) == 1 and float(opt.state[q]["step"]) == 1

    group = opt.param_groups[1]
    for key, value, error in (("betas", (0.9, 1.0), ValueError), ("eps", -1.0, ValueError), ("state_bits", 16, ValueError),
                              ("amsgrad", True, NotImplementedError), ("maximize", True, NotImplementedError)):
        old = group[key]
        group[key] = value
        refused(error, "FusedAdamW")
        group[key] = old
    codes = opt.state[q]["moment_codes"]
    for bad in (codes[:, :1], codes.float(), codes.cpu(), codes.view(32, 2, 2)):
        opt.state[q]["moment_codes"] = bad
        refused(RuntimeError, "does not match")
    opt.state[q]["moment_codes"] = codes
    group["state_bits"] = 32
    refused(RuntimeError, "does not match")
    group["state_bits"] = 8
    # sparse gradients, and two parameters in the same memory
    e = torch.nn.Parameter(torch.ones(8, 2, device=dev))
    e.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 2), (8, 2)).to(dev)
    with pytest.raises(RuntimeError, match="dense"):
        impl.FusedAdamW([e], lr=0.1).step()
    store = torch.ones(100, device=dev)
    x, y = torch.nn.Parameter(store[:60]), torch.nn.Parameter(store[59:])
    x.grad, y.grad = torch.ones(60, device=dev), torch.ones(41, device=dev)
    with pytest.raises(RuntimeError, match="share memory"):
        impl.FusedAdamW([x, y], lr=0.1).step()
    z = torch.nn.Parameter(torch.ones(4, 5, device=dev).t())
    z.grad = torch.ones(5, 4, device=dev)
    with pytest.raises(RuntimeError, match="contiguous"):
        impl.FusedAdamW([z], lr=0.1).step()
    h = torch.nn.Parameter(torch.ones(4, device=dev, dtype=torch.float16))
    h.grad = torch.ones(4, device=dev, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="bfloat16"):
        impl.FusedAdamW([h], lr=0.1).step()
    with pytest.raises(RuntimeError, match="one GPU"):
        opt.gather_state([p], torch.zeros(3, dtype=torch.int64))
    # neighbours in one storage are no overlap
    x, y = torch.nn.Parameter(store[:60]), torch.nn.Parameter(store[60:])
    x.grad, y.grad = torch.ones(60, device=dev), torch.ones(40, device=dev)
    impl.FusedAdamW([x, y], lr=0.1).step()
    assert torch.unique(store).numel() == 1


def test_backward_through_a_stepped_parameter_is_noticed(impl, dev):
    p = torch.nn.Parameter(torch.ones(4, device=dev))
    loss = (p * p).sum()
    p.grad = torch.ones(4, device=dev)
    impl.FusedAdamW([p], lr=0.1).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_continues_bit_for_bit(impl, dev, dtype, bits, tmp_path):
    gen = torch.Generator().manual_seed(3)
    grads = [torch.randn(100, 7, generator=gen).to(dev, dtype) for _ in range(6)]
    p = torch.nn.Parameter(torch.ones(100, 7, device=dev, dtype=dtype))
    opt = impl.FusedAdamW([p], lr=0.1, state_bits=bits, seed=17)
    for g in grads[:3]:
        p.grad = g
        opt.step()
    torch.save({"p": p.detach(), "o": opt.state_dict()}, tmp_path / "c.pt")
    saved = torch.load(tmp_path / "c.pt", weights_only=True, map_location="cpu")
    q = torch.nn.Parameter(saved["p"].to(dev))
    new = impl.FusedAdamW([q], lr=0.5, state_bits=bits)
    new.load_state_dict(saved["o"])
    for g in grads[3:]:
        p.grad, q.grad = g, g
        opt.step()
        new.step()
    assert torch.equal(p, q)
    for k, v in opt.state[p].items():
        assert torch.equal(v, new.state[q][k]), k


def test_bf16_parameter_keeps_small_updates_and_outside_writes(impl, dev):
    """1000 updates of 1e-5 on a bfloat16 1.0, whose step is 2^-7: the value behind it moves by all of them; a
    value written from outside is taken up, to half a step."""
    p = torch.nn.Parameter(torch.ones(100, device=dev, dtype=torch.bfloat16))
    opt = impl.FusedAdamW([p], lr=1e-5, weight_decay=0.0, eps=0.0)
    p.grad = torch.ones_like(p)
    for _ in range(1000):
        opt.step()
    got = opt.unpacked([p])[0]["param"]
    assert float((got - (1 - 1000 * 1e-5)).abs().max()) <= 1000 * (E + 15 * E * 1e-5)
    with torch.no_grad():
        p.fill_(5.0)
    got = opt.unpacked([p])[0]["param"]
    assert float((got - 5.0).abs().max()) <= 5.0 * 2.0 ** -8
    opt.state[p]["param_low"].copy_(torch.arange(-50, 50, dtype=torch.int16, device=dev) * 600)
    for zero in (0.0, -0.0):                      # a remainder of the old value must not borrow through the sign
        with torch.no_grad():
            p.fill_(zero)
        got = opt.unpacked([p])[0]["param"]
        assert float(got.abs().max()) <= 2.0 ** -126            # half a step of bfloat16 at zero is a subnormal
        q = torch.nn.Parameter(p.detach().clone())
        twin = impl.FusedAdamW([q], lr=1e-5, weight_decay=0.5, state_bits=8)
        twin.state[q] = {"step": torch.tensor(0.0), "moment_codes": torch.zeros(100, 2, dtype=torch.uint8, device=dev),
                         "moment_scales": torch.zeros(2, 2, device=dev), "param_low": opt.state[p]["param_low"].clone()}
        q.grad = torch.ones_like(q)
        twin.step()
        assert torch.equal(q.detach(), torch.full_like(q, -1e-5))


# ---- together, as a training loop uses them -------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_training_loop_with_densification(impl, dev, bits):
    """Rasterize, loss, backward, clipped step, statistics, prune and append, checkpoint: one loop over the framework's own entry
    points.  The 32-bit run is checked against torch.optim.AdamW and clip_grad_norm_ on the same gradients at every step."""
    syn = importlib.import_module("gaussian-splatting_amd.synthetic")
    sc = syn.make_scene(1500, 16, 64, 96, seed=1)
    settings = impl.GaussianRasterizationSettings(
        image_height=sc.H, image_width=sc.W, tanfovx=sc.tanfovx, tanfovy=sc.tanfovy, bg=sc.bg.to(dev), scale_modifier=1.0,
        viewmatrix=sc.viewmatrix.to(dev), projmatrix=sc.projmatrix.to(dev), sh_degree=sc.sh_degree, campos=sc.campos.to(dev),
        prefiltered=False, debug=False)
    names = ("means3D", "shs", "opacities", "scales", "rotations")
    params = {k: torch.nn.Parameter(getattr(sc, k).to(dev)) for k in names}
    gt = torch.rand(3, sc.H, sc.W, generator=torch.Generator().manual_seed(1)).to(dev)

    def groups(p):
        return [{"params": [p[k]], "lr": lr, "name": k} for k, lr in zip(names, (1.6e-4, 2.5e-3, 0.01, 1e-3, 1e-3))]

    opt = impl.FusedAdamW(groups(params), lr=0.0, eps=1e-15, weight_decay=1e-3, state_bits=bits)
    for it in range(6):
        n = params["means3D"].shape[0]
        screen = torch.zeros(n, 3, device=dev, requires_grad=True)
        image, radii, _, _ = impl.GaussianRasterizer(settings)(
            means3D=params["means3D"], means2D=screen, shs=params["shs"], colors_precomp=None, opacities=params["opacities"],
            scales=params["scales"], rotations=params["rotations"], cov3D_precomp=None)
        impl.l1_ssim_loss(image, gt, lambda_dssim=0.2).backward()
        acc, den, mr = torch.zeros(n, 1, device=dev), torch.zeros(n, 1, device=dev), torch.zeros(n, device=dev)
        opt.update_densify_stats(viewspace_grad=screen.grad, radii=radii, xyz_gradient_accum=acc, denom=den, max_radii2D=mr)
        assert torch.equal(mr, radii.clamp(min=0).float())
        twin = {k: torch.nn.Parameter(p.detach().clone()) for k, p in params.items()}
        ref = torch.optim.AdamW(groups(twin), lr=0.0, eps=1e-15, weight_decay=1e-3, foreach=True)
        if bits == 32:
            for k in names:
                twin[k].grad = params[k].grad.clone()
                if opt.state.get(params[k]):
                    ref.state[twin[k]] = {a: b.clone() for a, b in opt.state[params[k]].items()}
        norm = impl.grad_norm([p.grad for p in params.values()])
        opt.step(max_norm=0.5 * float(norm))
        assert torch.equal(opt.last_grad_norm, norm)
        if bits == 32:
            torch.nn.utils.clip_grad_norm_(list(twin.values()), 0.5 * float(norm))
            ref.step()
            for k in names:
                # the two norms differ by a few roundings, Adam's update by as much of itself (its size is at most 8 lr here)
                assert float((twin[k] - params[k]).detach().abs().max()) <= 2e-6 * max(1.0, float(params[k].detach().abs().max())), (it, k)
        for p in params.values():
            assert torch.isfinite(p).all()
            p.grad = None
        if it % 2 == 1:
            keep = ((acc / den.clamp(min=1))[:, 0] < (acc / den.clamp(min=1))[:, 0].quantile(0.9)).nonzero()[:, 0]
            index = torch.cat([keep, keep[:50], torch.full((25,), -1, device=dev)])
            old = [params[k] for k in names]
            new = [torch.nn.Parameter(p.detach()[index.clamp(min=0)].contiguous()) for p in old]
            opt.replace_params(old, new, index)
            params = dict(zip(names, new))
    assert params["means3D"].shape[0] != 1500
    sd = opt.state_dict()
    other = impl.FusedAdamW(groups({k: torch.nn.Parameter(p.detach().clone()) for k, p in params.items()}), lr=0.0, state_bits=bits)
    other.load_state_dict(sd)
    assert float(other.state[other.param_groups[0]["params"][0]]["step"]) == 6


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 43, 1000, 70_001])
@pytest.mark.parametrize("cuts", [(1, 3, 48), (3, 48), (45, 48), (5, 9, 20, 41), (24, 48)])
def test_column_ranges_of_one_matrix(impl, dev, n, cuts, dtype, bits):
    """Gradients that are neighbouring column ranges of one (n, 48) matrix (their workgroups alternate, the norm reads them as one),
    in both orders and with a gap: the same bits as from copies."""
    gen = torch.Generator().manual_seed(n)
    matrix = torch.randn(n, 48, generator=gen).to(dev, dtype)
    edges = [0, *cuts]
    ranges = list(zip(edges, edges[1:]))
    for order in (ranges, ranges[::-1], ranges[::2]):
        results = []
        for copy in (False, True):
            params = [torch.nn.Parameter(torch.ones(n, b - a, device=dev, dtype=dtype)) for a, b in order]
            for p, (a, b) in zip(params, order):
                p.grad = matrix[:, a:b].contiguous() if copy else matrix[:, a:b]
            opt = impl.FusedAdamW(params, lr=0.01, state_bits=bits, seed=3)
            for _ in range(2):
                opt.step(max_norm=1.0)
            results.append((params, opt))
        (pa, oa), (pb, ob) = results
        exact = math.sqrt(sum(float(p.grad.double().square().sum()) for p in pb))
        for o in (oa, ob):
            assert abs(float(o.last_grad_norm) - exact) <= 1.001 * E * exact
        if torch.equal(oa.last_grad_norm, ob.last_grad_norm):        # fp64 sums of another order may round to either neighbour
            for p, q in zip(pa, pb):
                assert torch.equal(p, q)
                for name, x in oa.state[p].items():
                    assert torch.equal(x, ob.state[q][name]), name


def test_column_ranges_in_a_captured_step(impl, dev):
    """Counts on the device together with alternating workgroups: every tensor finds its own scalars."""
    matrix = torch.randn(3000, 48, generator=torch.Generator().manual_seed(0)).to(dev)
    runs = []
    for capturable in (False, True):
        params = [torch.nn.Parameter(torch.ones(3000, w, device=dev)) for w in (45, 3)]
        params[0].grad, params[1].grad = matrix[:, 3:], matrix[:, :3]
        opt = impl.FusedAdamW([{"params": [params[0]], "lr": 0.5}, {"params": [params[1]], "lr": 0.001}], capturable=capturable)
        for _ in range(3):
            opt.step()
        runs.append(params)
    for p, q in zip(*runs):
        assert torch.equal(p, q)


def test_unpacked_of_mixed_states(impl, dev):
    """All kinds at once, empty tensors and missing states among them: every result is its own."""
    gen = torch.Generator().manual_seed(11)
    shapes = [(7, 3), (0, 3), (65,), (), (130, 2), (3, 0)]
    groups, params = [], []
    for bits in (8, 32):
        for dtype in (torch.float32, torch.bfloat16):
            ps = [torch.nn.Parameter(torch.randn(s, generator=gen).to(dev, dtype)) for s in shapes]
            params += ps
            groups.append({"params": ps, "state_bits": bits})
    bare = torch.nn.Parameter(torch.ones(5, device=dev, dtype=torch.bfloat16))
    opt = impl.FusedAdamW(groups + [{"params": [bare]}], lr=0.1)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(dev, p.dtype)
    opt.step()
    got = opt.unpacked(params + [bare])
    assert len(opt.unpacked()) == len(params) and set(got[-1]) == {"param"} and got[-1]["param"].dtype == torch.float32
    for p, x in zip(params, got):
        s = opt.state[p]
        if "moment_codes" in s:
            m, u = orc.unpack(_np(s["moment_codes"]).reshape(-1, 2), _np(s["moment_scales"]))
            expect = m, u * u
        else:
            expect = _np(s["exp_avg"]).reshape(-1), _np(s["exp_avg_sq"]).reshape(-1)
        for name, y in zip(("exp_avg", "exp_avg_sq"), expect):
            assert x[name].shape == p.shape and x[name].dtype == torch.float32
            assert np.array_equal(_np(x[name]).reshape(-1), y), name
        value = orc.join(_bits16(p).reshape(-1), _np(s["param_low"]).reshape(-1)) if p.dtype == torch.bfloat16 else _np(p).reshape(-1)
        assert x["param"].shape == p.shape and np.array_equal(_np(x["param"]).reshape(-1), value)
    with pytest.raises(ValueError, match="not a parameter"):
        stranger = torch.nn.Parameter(torch.ones(5, device=dev))
        opt.state[stranger] = dict(opt.state[params[0]])
        opt.unpacked([stranger])
    with pytest.raises(RuntimeError, match="not a state"):
        opt.unpacked(states=[{"moment_codes": torch.zeros(5, 2, device=dev), "moment_scales": torch.zeros(1, 2, device=dev)}])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,row_len,width", [(5, 2047, 2049), (5, 2048, 2100), (4, 4097, 5000), (3, 8191, 8192), (3, 8192, 8200), (3, 9000, 9001),
                                                (2, 40_000, 70_000), (70, 4, 5), (70, 5, 5000)])
def test_long_rows(impl, dev, rows, row_len, width, dtype):
    """Rows around and beyond a workgroup's chunk: strided gradients of the step and the norm, and the selection of such rows."""
    gen = torch.Generator().manual_seed(row_len)
    wide = torch.full((rows, width), float("nan"))
    wide[:, 1:1 + row_len] = torch.randn(rows, row_len, generator=gen)
    wide = wide.to(dev, dtype)
    start = torch.randn(rows, row_len, generator=gen).to(dev, dtype)
    index = torch.tensor([rows - 1, 0, -1, rows - 1, rows], device=dev)
    for bits in (32, 8):
        a, b = torch.nn.Parameter(start.clone()), torch.nn.Parameter(start.clone())
        a.grad = wide[:, 1:1 + row_len]
        b.grad = a.grad.contiguous()
        opts = [impl.FusedAdamW([p], lr=0.1, state_bits=bits, seed=1) for p in (a, b)]
        for _ in range(2):
            for o in opts:
                o.step(max_norm=1e9)
        exact = float(b.grad.double().square().sum().sqrt())
        for o in opts:
            assert abs(float(o.last_grad_norm) - exact) <= 1.001 * E * exact
        assert torch.equal(a, b)
        for name, x in opts[0].state[a].items():
            assert torch.equal(x, opts[1].state[b][name]), name
        old, new = opts[0].unpacked([a])[0], opts[0].gather_state([a], index)
        got = opts[0].unpacked(states=new)[0]
        for name in ("exp_avg", "exp_avg_sq"):
            expect = _np(old[name])[[rows - 1, 0, 0, rows - 1, 0]]
            expect[[2, 4]] = 0
            if bits == 8:
                x = expect if name == "exp_avg" else np.sqrt(expect)
                m, u = (x, np.zeros_like(x)) if name == "exp_avg" else (np.zeros_like(x), x)
                packed = orc.unpack(*orc.pack(m.reshape(-1).astype(np.float32), u.reshape(-1).astype(np.float32)))
                expect = (packed[0] if name == "exp_avg" else packed[1] ** 2).reshape(expect.shape)
            assert np.array_equal(_np(got[name]), expect), (bits, name)
        if dtype == torch.bfloat16:
            low = _np(opts[0].state[a]["param_low"])[[rows - 1, 0, 0, rows - 1, 0]]
            low[[2, 4]] = 0
            assert np.array_equal(_np(new[0]["param_low"]), low)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_with_counts_on_the_device(impl, dev, bits):
    """75 tensors, three launches: captured, every tensor with its own rate and count; their rows and their values in one call."""
    gen = torch.Generator().manual_seed(5)
    a = [torch.nn.Parameter(torch.randn(40, k % 7 + 1, generator=gen).to(dev)) for k in range(75)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    rate = lambda k: float(np.float32(0.01 * (k + 1)))  # noqa: E731
    opt = impl.FusedAdamW([{"params": [p], "lr": torch.tensor(rate(k), device=dev)} for k, p in enumerate(a)], state_bits=bits, capturable=True)
    ref = impl.FusedAdamW([{"params": [p], "lr": rate(k)} for k, p in enumerate(b)], state_bits=bits)
    for p, q in zip(a, b):
        p.grad = torch.randn(p.shape, generator=gen).to(dev)
        q.grad = p.grad.clone()
    for k, (p, q) in enumerate(zip(a, b)):          # counts of their own: the first tensors are a few updates ahead
        if k < 20:
            others = [x.grad for x in a], [x.grad for x in b]
            for x in a + b:
                x.grad = None
            p.grad, q.grad = others[0][k], others[1][k]
            opt.step()
            ref.step()
            for x, g in zip(a + b, others[0] + others[1]):
                x.grad = g
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(max_norm=3.0)
    for _ in range(3):
        graph.replay()
        ref.step(max_norm=3.0)
        torch.cuda.synchronize()
    for k, (p, q) in enumerate(zip(a, b)):
        assert float(opt.state[p]["step"]) == float(ref.state[q]["step"]) == (5 if k < 20 else 4)
        assert torch.equal(p, q), k
    index = torch.arange(39, -1, -1, device=dev)
    for o, ps in ((opt, a), (ref, b)):
        values, rows = o.unpacked(ps), o.unpacked(states=o.gather_state(ps, index))
        alone = [o.unpacked([p])[0] for p in ps]
        for x, y, z in zip(values, rows, alone):
            assert torch.equal(x["exp_avg"], z["exp_avg"]) and torch.equal(x["exp_avg_sq"], z["exp_avg_sq"])
            # reversed rows: exact in 32 bits; in 8 a level of the first moment is off by at most half an eighth of its octave
            tol = 0.0 if bits == 32 else 1 / 16 + 1e-6
            low = 0.0 if bits == 32 else float(x["exp_avg"].abs().max()) * 1.25 * 2.0 ** -17
            assert bool(((y["exp_avg"] - x["exp_avg"][index]).abs() <= tol * x["exp_avg"][index].abs() + low).all())
