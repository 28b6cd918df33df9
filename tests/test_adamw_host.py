"""CPU: the host side of FusedAdamW / grad_norm -- argument checks of the Python classes and of the C entry points (which refuse
before any launch), the descriptor structs against the header, and the oracle of the 8-bit format against its definition."""
import ctypes as C
import importlib
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from oracle import adamw_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def impl():
    return importlib.import_module("gaussian-splatting_amd")


@pytest.fixture(scope="module")
def adamw():
    return importlib.import_module("gaussian-splatting_amd.adamw")


def test_descriptor_structs_match_the_header(impl, adamw):
    names = ["GsAdamWTensor", "GsGradTensor", "GsAdamWRows", "GsAdamWUnpack"]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "gsplat.h"\nint main(void){\n'
    for n in names:
        src += f'printf("{n} %zu\\n", sizeof({n}));\n'
        for field, _ in getattr(impl._lib, n)._fields_:
            src += f'printf("{n}.{field} %zu\\n", offsetof({n}, {field}));\n'
    src += "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "t.c"), "w") as f:
            f.write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "t.c"), "-o", os.path.join(d, "t")])
        out = dict(line.split() for line in subprocess.check_output([os.path.join(d, "t")], text=True).splitlines())
    for n in names:
        cls = getattr(impl._lib, n)
        assert int(out[n]) == C.sizeof(cls)
        for field, _ in cls._fields_:
            assert int(out[f"{n}.{field}"]) == getattr(cls, field).offset, (n, field)
    # the packed forms: every field in its place (a count up from 1 in the order of the struct)
    for pack, cls in ((adamw._STEP, impl._lib.GsAdamWTensor), (adamw._GRAD, impl._lib.GsGradTensor), (adamw._ROWS, impl._lib.GsAdamWRows),
                      (adamw._UNPACK, impl._lib.GsAdamWUnpack)):
        packed = pack(*range(1, len(cls._fields_) + 1))
        assert len(packed) == C.sizeof(cls)
        got = cls.from_buffer_copy(packed)
        assert [getattr(got, field) for field, _ in cls._fields_] == list(range(1, len(cls._fields_) + 1))
    assert impl._lib.load().gs_adamw_block() == adamw.BLOCK == orc.BLOCK


def test_python_refusals(impl):
    p = torch.nn.Parameter(torch.randn(4, 3))
    for kw in ({"amsgrad": True}, {"maximize": True}, {"differentiable": True}):
        with pytest.raises(NotImplementedError):
            impl.FusedAdamW([p], **kw)
    with pytest.raises(ValueError, match="state_bits"):
        impl.FusedAdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="state_bits"):
        impl.FusedAdamW([{"params": [p], "state_bits": 4}])
    for kw in ({"lr": -1.0}, {"eps": -1.0}, {"betas": (1.0, 0.9)}, {"weight_decay": -0.1}):
        with pytest.raises(ValueError):
            impl.FusedAdamW([p], **kw)
    opt = impl.FusedAdamW([p], lr=1e-3)
    opt.step()                                    # nothing has a gradient: nothing to do
    assert not opt.state
    p.grad = torch.randn(4, 3)
    with pytest.raises(RuntimeError, match="GPU"):
        opt.step()
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-1.0)
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=float("nan"))
    with pytest.raises(ValueError, match="both"):
        opt.step(grad_norm=torch.ones(()))
    assert not opt.state
    with pytest.raises(RuntimeError, match="GPU"):
        impl.grad_norm([p.grad])
    with pytest.raises(ValueError):
        impl.grad_norm([None])
    index = torch.arange(4)
    with pytest.raises(ValueError, match="int64"):
        opt.gather_state([p], torch.ones(4, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="GPU"):
        opt.gather_state([p], index)
    with pytest.raises(ValueError, match="same number of rows"):
        opt.gather_state([torch.nn.Parameter(torch.zeros(()))], index)
    q = torch.nn.Parameter(torch.randn(4, 3))
    with pytest.raises(ValueError):
        opt.replace_params([q], [torch.nn.Parameter(torch.randn(4, 3))], index)      # not one of its parameters
    with pytest.raises(ValueError, match="cannot take the place"):
        opt.replace_params([p], [torch.nn.Parameter(torch.randn(5, 3))], index)
    with pytest.raises(ValueError, match="each once"):
        opt.replace_params([p, p], [q, torch.nn.Parameter(torch.randn(4, 3))], index)
    with pytest.raises(ValueError, match="int64"):
        opt.replace_params([p], [q], [0, 1, 2, 3])
    with pytest.raises(ValueError, match="not both"):
        opt.unpacked([p], states=[])
    assert opt.gather_state([], index) == []


def test_group_options_and_torch_class(impl):
    a, b = torch.nn.Parameter(torch.randn(4)), torch.nn.Parameter(torch.randn(4))
    opt = impl.FusedAdamW([{"params": [a], "state_bits": 8, "seed": 3}], lr=0.1, weight_decay=0.2, seed=9)
    opt.add_param_group({"params": [b], "stochastic_rounding": False})
    assert isinstance(opt, torch.optim.AdamW)
    g, h = opt.param_groups
    assert (g["state_bits"], g["seed"], g["stochastic_rounding"]) == (8, 3, True)
    assert (h["state_bits"], h["seed"], h["stochastic_rounding"], h["weight_decay"]) == (32, 9, False, 0.2)
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(1))], "state_bits": 7})
    import copy
    import pickle
    other = pickle.loads(pickle.dumps(opt))
    assert other.param_groups[0]["state_bits"] == 8 and copy.deepcopy(opt).param_groups[0]["seed"] == 3
    other.add_param_group({"params": [torch.nn.Parameter(torch.zeros(1))]})
    assert other.param_groups[-1]["seed"] == 9 and other.last_grad_norm is None
    assert len(opt.param_groups) == 2             # the refused group was not added


def test_load_state_dict_keeps_types(impl):
    """The base class casts every floating state to the parameter's type and integer codes with it; here each keeps its own."""
    p, q = torch.nn.Parameter(torch.randn(5, 3).bfloat16()), torch.nn.Parameter(torch.randn(70))
    opt = impl.FusedAdamW([{"params": [p], "state_bits": 8}, {"params": [q]}], lr=0.1)
    opt.state[p] = {"step": torch.tensor(3.0), "moment_codes": torch.randint(0, 256, (5, 3, 2), dtype=torch.uint8),
                    "moment_scales": torch.rand(1, 2), "param_low": torch.randint(-9, 9, (5, 3), dtype=torch.int16)}
    opt.state[q] = {"step": torch.tensor(4.0), "exp_avg": torch.randn(70), "exp_avg_sq": torch.rand(70)}
    p2, q2 = torch.nn.Parameter(p.detach().clone()), torch.nn.Parameter(q.detach().clone())
    new = impl.FusedAdamW([{"params": [p2], "state_bits": 8}, {"params": [q2]}], lr=0.7)
    new.load_state_dict(opt.state_dict())
    for a, b in ((p, p2), (q, q2)):
        assert set(opt.state[a]) == set(new.state[b])
        for k, x in opt.state[a].items():
            y = new.state[b][k]
            assert y.dtype == x.dtype and torch.equal(x, y) and y.data_ptr() != x.data_ptr(), k
    assert new.param_groups[0]["lr"] == 0.1
    # torch's own AdamW state goes into 32-bit groups and is refused by 8-bit ones
    r = torch.nn.Parameter(torch.randn(6))
    ref = torch.optim.AdamW([r], lr=0.3)
    r.grad = torch.randn(6)
    ref.step()
    s = torch.nn.Parameter(r.detach().clone())
    into = impl.FusedAdamW([s], lr=0.5)
    into.load_state_dict(ref.state_dict())
    assert torch.equal(into.state[s]["exp_avg"], ref.state[r]["exp_avg"]) and into.param_groups[0]["state_bits"] == 32
    eight = impl.FusedAdamW([torch.nn.Parameter(r.detach().clone())], lr=0.5, state_bits=8)
    with pytest.raises(ValueError, match="8 bits"):
        eight.load_state_dict(ref.state_dict())
    assert eight.param_groups[0]["lr"] == 0.5


def test_gradient_layouts(adamw):
    """Rows that are contiguous in themselves are taken in place, everything else is copied."""
    base = torch.arange(10 * 16 * 3, dtype=torch.float32).view(10, 16, 3)
    for view, expect in ((base, (480, 1, 0)), (base[:, :1], (10, 3, 48)), (base[:, 1:], (10, 45, 48)), (base[:, 1:][:, :, :1], None),
                         (base.transpose(0, 1), None), (base[0, 0, 0].expand(5), None), (base[::2], (5, 48, 96)),
                         (base[:, 0, 0], (10, 1, 48)), (base[:1, 1:], (45, 1, 0)), (torch.zeros(()), (1, 1, 0)),
                         (torch.zeros(0, 3), (0, 1, 0)), (base[:, 1:2, 1:2], (10, 1, 48)), (base.as_strided((4, 6), (3, 1)), None)):
        t, rows, row_len, stride = adamw._matrix(view)
        if expect is None:
            assert t.is_contiguous() and t.data_ptr() != view.data_ptr() and (rows, row_len, stride) == (view.numel(), 1, 0)
        else:
            assert t.data_ptr() == view.data_ptr() and (rows, row_len, stride) == expect
        flat = t.as_strided((rows, row_len), (stride or row_len, 1)) if rows else t
        assert torch.equal(flat.reshape(-1), view.reshape(-1))


def test_c_refusals_before_any_launch(impl):
    L = impl._lib
    lib = L.load()
    buf = C.create_string_buffer(4096)
    at = (C.addressof(buf) + 255) & ~255

    def tensor(**kw):
        t = L.GsAdamWTensor(param=at, grad=at, exp_avg=at, exp_avg_sq=at, rows=4, grad_row_stride=0, step=1, lr=0.1, beta1=0.9, beta2=0.99,
                            eps=1e-8, weight_decay=0.0, row_len=3)
        for k, v in kw.items():
            setattr(t, k, v)
        return (L.GsAdamWTensor * 1)(t)

    def step(arr, bf16=0, bits=32, norm=None, max_norm=1.0, scalars=None):
        return lib.gs_adamw_step(1, arr, bf16, bits, 1, norm, max_norm, scalars, None)

    cases = [(dict(), dict(bits=16), b"state_bits"), (dict(rows=-1), {}, b"shape"), (dict(row_len=0), {}, b"shape"),
             (dict(param=None), {}, b"null"), (dict(grad=None), {}, b"null"), (dict(exp_avg=None), {}, b"null"),
             (dict(exp_avg_sq=None), {}, b"null"), (dict(), dict(bf16=1), b"param_low"), (dict(grad_row_stride=2), {}, b"grad_row_stride"),
             (dict(beta1=1.0), {}, b"betas"), (dict(beta2=-0.1), {}, b"betas"), (dict(eps=-1.0), {}, b"eps"), (dict(step=0), {}, b"step"),
             (dict(step_dev=at), {}, b"scalars"), (dict(), dict(scalars=at), b"scalars"), (dict(step_dev=at), dict(scalars=at + 4), b"aligned"),
             (dict(lr_dev=at), {}, b"lr on the device"), (dict(param=at + 2), {}, b"misaligned"), (dict(exp_avg_sq=at + 4), dict(bits=8), b"misaligned"),
             (dict(), dict(norm=at, max_norm=-1.0), b"max_norm"), (dict(), dict(norm=at, max_norm=float("nan")), b"max_norm"),
             (dict(rows=1 << 41, row_len=1), {}, b"shape"), (dict(rows=1 << 39, row_len=1), {}, b"workgroups"), (dict(rows=1 << 32, row_len=1 << 20), {}, b"shape")]
    for fields, args, message in cases:
        rc = step(tensor(**fields), **args)
        assert rc == -1 and message in lib.gs_last_error(), (fields, args, lib.gs_last_error())
    assert lib.gs_adamw_step(-1, None, 0, 32, 1, None, 0.0, None, None) == -1
    assert lib.gs_adamw_step(0, None, 0, 32, 1, None, 0.0, None, None) == 0            # nothing to do

    def grad(**kw):
        t = L.GsGradTensor(grad=at, rows=20000, row_stride=0, row_len=1, bf16=0)
        for k, v in kw.items():
            setattr(t, k, v)
        return (L.GsGradTensor * 1)(t)

    size = lib.gs_grad_norm_workspace_bytes(1, grad())
    assert size >= 8
    for arr, out, ws, n in ((grad(grad=None), at, at, size), (grad(), None, at, size), (grad(), at, at, size - 1), (grad(), at, None, size),
                            (grad(rows=-5), at, at, size), (grad(row_stride=1, row_len=2), at, at, 1 << 20), (grad(grad=at + 2), at, at, size),
                            (grad(), at, at + 4, size)):
        assert lib.gs_grad_norm(1, arr, out, ws, n, None) == -1

    def rows(**kw):
        t = L.GsAdamWRows(src_exp_avg=at, src_exp_avg_sq=at, dst_exp_avg=at + 1024, dst_exp_avg_sq=at + 2048, row_len=3)
        for k, v in kw.items():
            setattr(t, k, v)
        return (L.GsAdamWRows * 1)(t)

    for arr, bits, n_src, n_dst, index in ((rows(), 4, 4, 4, at), (rows(), 32, -1, 4, at), (rows(), 32, 4, 4, None), (rows(row_len=0), 32, 4, 4, at),
                                           (rows(src_exp_avg=None), 32, 4, 4, at), (rows(dst_exp_avg_sq=None), 32, 4, 4, at),
                                           (rows(src_param_low=at), 32, 4, 4, at), (rows(dst_exp_avg_sq=at + 2052), 8, 4, 4, at),
                                           (rows(), 32, 4, 4, at + 4)):
        assert lib.gs_adamw_gather_rows(1, arr, bits, n_src, n_dst, index, None) == -1

    for kw in (dict(codes=at, numel=4), dict(param_bf16=at, numel=4), dict(codes=at + 1, scales=at, exp_avg=at, exp_avg_sq=at, numel=4),
               dict(codes=at, scales=at, exp_avg=at, exp_avg_sq=at, numel=-1)):
        assert lib.gs_adamw_unpack(1, (L.GsAdamWUnpack * 1)(L.GsAdamWUnpack(**kw)), None) == -1


def test_oracle_levels_agree_with_the_definition():
    """The bit patterns of the format against 2^(q div L) (1 + (q mod L) / L), exactly; the codes of every level round-trip."""
    codes = np.arange(256)
    m, u = orc.unpack(np.stack([codes, codes], 1).astype(np.uint8), np.ones((4, 2), np.float32))
    assert np.array_equal(m.astype(np.float64), orc.level_m(codes, 1.0)) and np.array_equal(u.astype(np.float64), orc.level_u(codes, 1.0))
    assert np.all(np.diff(u) > 0) and np.all(np.diff(m[:128]) > 0) and m[1] == 1.25 * 2.0 ** -16 and u[255] == m[127] == 1.0
    for k in range(4):                            # blocks of 64 that hold 1.0, so that the scale is 1
        part = np.concatenate([codes[64 * k: 64 * k + 63], [255]])
        mm, uu = np.where(part == 255, np.float32(1), m[part]), u[part]
        back, s = orc.pack(mm, uu)
        assert np.array_equal(s, np.ones((1, 2), np.float32))
        assert np.array_equal(back[:, 1], part)
        assert np.array_equal(orc.unpack(back, s)[0], mm)


def test_oracle_rounding_is_nearest_or_unbiased():
    rng = np.random.default_rng(5)
    x = np.exp(rng.uniform(np.log(2.0 ** -15), 0, 63 * 64)).astype(np.float32).reshape(63, 64)
    x[:, 0] = 1.0
    x = x.reshape(-1)
    codes, s = orc.pack(x * np.where(rng.random(x.size) < 0.5, -1, 1).astype(np.float32), x)
    for col, level, per in ((0, orc.level_m, 8), (1, orc.level_u, 16)):
        err = np.abs(np.abs(level(codes[:, col], 1.0)) - x)
        gap = np.exp2(np.floor(np.log2(x.astype(np.float64)))) / per
        assert np.all(err <= gap / 2 * (1 + 1e-6))
    # stochastic: the mean over many draws; a draw is off by at most a gap, so its variance is at most gap^2 / 4
    draws = 4000
    y = np.full(64, np.float32(0.3))
    y[0] = 1.0
    total = np.zeros((2, 64))
    for t in range(draws):
        c, s = orc.pack(y, y, orc.random_bits(64, 11, 0, t + 1))
        total += np.stack([orc.level_m(c[:, 0], 1.0), orc.level_u(c[:, 1], 1.0)])
    mean = total / draws
    for row, per in ((0, 8), (1, 16)):
        gap = 0.25 / per
        assert abs(mean[row, 1:].mean() - 0.3) <= 5 * gap / 2 / np.sqrt(draws * 63) + gap / 65536
        assert np.all(np.abs(mean[row, 1:] - 0.3) <= 5 * gap / 2 / np.sqrt(draws) + gap / 65536)


def test_oracle_split_of_bf16():
    rng = np.random.default_rng(6)
    x = np.concatenate([rng.standard_normal(1000).astype(np.float32), np.array([0.0, -0.0, 1.0, 3.3895e38, -3.3895e38, 1e-40], np.float32)])
    high, low = orc.split(x)
    assert np.array_equal(orc.join(high, low).view(np.uint32), x.view(np.uint32))
    near = torch.from_numpy(x[:1000]).to(torch.bfloat16).float().numpy()
    got = torch.from_numpy(high[:1000].view(np.int16)).view(torch.bfloat16).float().numpy()
    assert np.all(np.abs(got - x[:1000]) <= np.abs(x[:1000]) * 2.0 ** -8) and (got != near).mean() < 0.01


def _norm_worker(rank, world, port, tmp):
    import sys
    import torch.distributed as dist
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        par = importlib.import_module("gaussian-splatting_amd.parallel")
        mine = torch.tensor([3.0, 4.0][rank])
        got = par.reduce_grad_norm(mine)
        assert got.shape == () and got.dtype == torch.float32 and float(got) == 5.0 and float(mine) == [3.0, 4.0][rank]
        assert float(par.reduce_grad_norm(torch.tensor([3e30, 4e30][rank]))) == float(torch.tensor(5e30))       # the squares pass float32's range
        assert torch.isnan(par.reduce_grad_norm(torch.tensor([1.0, float("nan")][rank])))
        open(os.path.join(tmp, f"ok{rank}"), "w").write("ok")
    finally:
        dist.destroy_process_group()


def test_norm_of_sharded_gradients_gloo(tmp_path):
    import socket
    import torch.multiprocessing as mp
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    mp.spawn(_norm_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    assert (tmp_path / "ok0").exists() and (tmp_path / "ok1").exists()
    par = importlib.import_module("gaussian-splatting_amd.parallel")
    assert float(par.reduce_grad_norm(torch.tensor(2.0))) == 2.0                                                 # no process group
