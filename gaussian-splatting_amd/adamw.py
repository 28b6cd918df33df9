"""AdamW over many tensors with moments in 32 or in 8 bits, the global gradient norm, and the state's rows.

``FusedAdamW`` stands beside ``FusedAdam`` (optimizer.py) for training with decoupled weight decay: a
``torch.optim.AdamW`` whose ``step()`` is one HIP launch per 32 tensors (gs_adamw_step).  Beyond torch's class:

    state_bits=8            two bytes of state per element instead of eight (a Gaussian model's moments: 472 -> 133 bytes per
                            Gaussian of SH degree 3), rounded stochastically from a seed: the same seed gives the same bits
    step(max_norm=...)      clips by the global norm inside the step: no pass that rewrites the gradients
    bfloat16 parameters     the fp32 value is kept (16 more bits of state), so small updates are not lost
    capturable=True         counts (and learning rates given as GPU tensors) are read on the GPU: the step can be captured
                            in a graph and replayed
    replace_params(...)     the reference's optimizer surgery (scene/gaussian_model.py:461-530) for states in either form
    grad_norm(grads)        the global norm alone

32-bit states of float32 parameters are bit-identical to torch.optim.AdamW's on the same GPU.  No CPU path.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib
from .optimizer import FusedAdam
from .profiling import stage as _stage

BLOCK = 64                                       # GS_ADAMW_BLOCK: elements that share a pair of scales
_STEP = struct.Struct("@7P3q5diIIi")             # GsAdamWTensor
_GRAD = struct.Struct("@P2q2i")                  # GsGradTensor
_TYPES = (torch.float32, torch.bfloat16)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _table(struct_type, packed):
    return (struct_type * len(packed)).from_buffer(bytearray(b"".join(packed)))


def _matrix(g):
    """(tensor to keep alive, rows, row length, row stride) of a gradient: rows that are contiguous in themselves are taken where they are."""
    if g.is_contiguous():
        return g, g.numel(), 1, 0
    if g.shape[0] > 1:
        row_len = 1
        for size, stride in zip(reversed(g.shape[1:]), reversed(g.stride()[1:])):
            if size != 1 and stride != row_len:
                break
            row_len *= size
        else:
            if row_len <= g.stride(0) and 0 < row_len < 1 << 31:
                return g, g.shape[0], row_len, g.stride(0)
    return g.contiguous(), g.numel(), 1, 0


def _check_grad(g, what):
    if g.layout != torch.strided or not g.is_cuda:
        raise RuntimeError(f"{what} must be a dense tensor on the GPU (no CPU path)")
    if g.dtype not in _TYPES:
        raise RuntimeError(f"{what} must be float32 or bfloat16, not {g.dtype}")


def _norm(mats, dev):
    """Launches gs_grad_norm over (matrix, is_bf16) pairs on the current stream of `dev`, the current device."""
    lib = _lib.load()
    arr = _table(_lib.GsGradTensor, [_GRAD.pack(g.data_ptr(), rows, stride, row_len, bf16) for (g, rows, row_len, stride), bf16 in mats])
    size = lib.gs_grad_norm_workspace_bytes(len(mats), arr)
    ws = torch.empty(max(size, 8), dtype=torch.uint8, device=dev)
    out = torch.empty((), dtype=torch.float32, device=dev)
    _lib.check(lib.gs_grad_norm(len(mats), arr, _ptr(out), _ptr(ws), size, C.c_void_p(torch.cuda.current_stream().cuda_stream)),
               "gs_grad_norm")
    return out


@torch.no_grad()
def grad_norm(grads):
    """sqrt of the sum of squares over all given tensors (None is skipped) as a 0-d float32 GPU tensor.

    float32 and bfloat16, any strides; accumulated in fp64 in a fixed order, so it neither overflows before its result does nor
    depends on scheduling.  Nothing is synchronised.  For gradients sharded over ranks, all-reduce the square of the result
    and pass its root to ``FusedAdamW.step(max_norm=..., grad_norm=...)``."""
    grads = [grads] if torch.is_tensor(grads) else [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grad_norm needs at least one tensor")
    for g in grads:
        _check_grad(g, "grad_norm: a gradient")
        if g.device != grads[0].device:
            raise RuntimeError("grad_norm: all gradients must live on one device")
    with torch.cuda.device(grads[0].device), _stage("grad_norm"):
        return _norm([(_matrix(g), g.dtype == torch.bfloat16) for g in grads], grads[0].device)


class FusedAdamW(torch.optim.AdamW):
    """AdamW on float32 or bfloat16 GPU parameters; see the module's docstring for what it adds to torch's class.

    ``state_bits``, ``stochastic_rounding`` and ``seed`` may differ between parameter groups, as every other option.
    State of a parameter: ``step``; ``exp_avg`` and ``exp_avg_sq`` (float32) or, with 8 bits, ``moment_codes`` (uint8,
    shape + (2,)) and ``moment_scales`` (float32, (ceil(numel / 64), 2)); for bfloat16 parameters ``param_low`` (int16).
    ``last_grad_norm`` is the norm that the last step clipped by (None without clipping)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *, state_bits=32,
                 stochastic_rounding=True, seed=0, capturable=False, **kw):
        if amsgrad or kw.pop("maximize", False) or kw.pop("differentiable", False):
            raise NotImplementedError("FusedAdamW: amsgrad / maximize / differentiable are not implemented")
        for k in ("foreach", "fused"):
            kw.pop(k, None)
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, foreach=False,
                         capturable=capturable, **kw)
        self._own_defaults = {"state_bits": state_bits, "stochastic_rounding": bool(stochastic_rounding), "seed": int(seed)}
        self.defaults.update(self._own_defaults)
        for group in self.param_groups:
            self._complete(group)
        self.last_grad_norm = None

    def _complete(self, group):
        for k, v in self._own_defaults.items():
            group.setdefault(k, v)
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {group['state_bits']!r}")

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if hasattr(self, "_own_defaults"):       # not yet while the base class adds the first groups
            self._complete(self.param_groups[-1])

    # ---- the step ---------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None, *, max_norm=None, grad_norm=None):
        """One AdamW update of every parameter that has a .grad (others are skipped, as in torch).

        ``max_norm``: gradients are multiplied by min(1, max_norm / (norm + 1e-6)) inside the update, the rule of
        torch.nn.utils.clip_grad_norm_, and are themselves left as they are; norm is over all gradients of this step, or
        ``grad_norm`` (one float32 on the GPU) where the caller has it."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if max_norm is None:
            if grad_norm is not None:
                raise ValueError("grad_norm is the norm that max_norm clips: give both")
        elif not float(max_norm) >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        work, dev = self._collect()
        self.last_grad_norm = None
        if not work:
            return loss
        if grad_norm is not None and (not torch.is_tensor(grad_norm) or grad_norm.device != dev or grad_norm.dtype != torch.float32
                                      or grad_norm.numel() != 1):
            raise ValueError("grad_norm must be one float32 on the parameters' device")
        with torch.cuda.device(dev), _stage("adamw"):
            capturing = torch.cuda.is_current_stream_capturing()
            if capturing:
                self._check_capture(work)
            mats = [_matrix(g) for _, _, _, g, _ in work]
            if max_norm is not None and grad_norm is None:
                grad_norm = _norm([(m, g.dtype == torch.bfloat16) for m, (_, _, _, g, _) in zip(mats, work)], dev)
            self._launch(work, mats, grad_norm, max_norm, dev)
        self.last_grad_norm = grad_norm
        torch.autograd.graph.increment_version([p for _, p, _, _, _ in work])
        return loss

    def _collect(self):
        """Everything that the step updates, checked before anything changes: [(group, param, index, grad, state or None)]."""
        work, dev, index, spans = [], None, -1, []
        for group in self.param_groups:
            if group["amsgrad"] or group["maximize"] or group["differentiable"]:
                raise NotImplementedError("FusedAdamW: amsgrad / maximize / differentiable are not implemented")
            beta1, beta2 = group["betas"]
            if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0 and group["eps"] >= 0.0 and group["state_bits"] in (8, 32)):
                raise ValueError(f"FusedAdamW: betas {group['betas']}, eps {group['eps']}, state_bits {group['state_bits']}: betas are in "
                                 "[0, 1), eps is not negative, state_bits is 8 or 32")
            for p in group["params"]:
                index += 1
                g = p.grad
                if g is None:
                    continue
                if not p.is_cuda or p.dtype not in _TYPES or not p.is_contiguous():
                    raise RuntimeError("FusedAdamW needs contiguous float32 or bfloat16 parameters on the GPU (no CPU path)")
                _check_grad(g, "FusedAdamW: a gradient")
                if g.dtype != p.dtype or g.device != p.device:
                    raise RuntimeError("FusedAdamW needs gradients of the parameter's type on its device")
                if dev is None:
                    dev = p.device
                elif dev != p.device:
                    raise RuntimeError("FusedAdamW: all parameters must live on one device")
                state = self.state.get(p) or None
                if state is not None:
                    self._check_state(p, state, group["state_bits"])
                if p.numel():
                    spans.append((p.data_ptr(), p.numel() * p.element_size()))
                work.append((group, p, index, g, state))
        spans.sort()
        for (a, size), (b, _) in zip(spans, spans[1:]):
            if a + size > b:
                raise RuntimeError("FusedAdamW: two parameters share memory (or one is listed twice)")
        return work, dev

    @staticmethod
    def _check_state(p, state, bits):
        if bits == 8:
            a, b = state.get("moment_codes"), state.get("moment_scales")
            good = (a is not None and b is not None and a.dtype == torch.uint8 and a.shape == p.shape + (2,)
                    and b.shape == ((p.numel() + BLOCK - 1) // BLOCK, 2))
        else:
            a, b = state.get("exp_avg"), state.get("exp_avg_sq")
            good = a is not None and b is not None and a.dtype == torch.float32 and a.shape == p.shape and b.shape == p.shape
        low = state.get("param_low") if p.dtype == torch.bfloat16 else None
        if p.dtype == torch.bfloat16:
            good = good and low is not None and low.dtype == torch.int16 and low.shape == p.shape and low.is_contiguous() and low.device == p.device
        if not good or b.dtype != torch.float32 or not (a.is_contiguous() and b.is_contiguous()) or a.device != p.device or b.device != p.device:
            raise RuntimeError(f"FusedAdamW: optimizer state does not match its parameter (shape {tuple(p.shape)}, {p.dtype}, state_bits {bits}); "
                               "replace_params() takes states along when rows are pruned or added")

    @staticmethod
    def _fresh_state(p, bits, capturable):
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device if capturable else "cpu")}
        if bits == 8:
            state["moment_codes"] = torch.zeros(p.shape + (2,), dtype=torch.uint8, device=p.device)
            state["moment_scales"] = torch.zeros(((p.numel() + BLOCK - 1) // BLOCK, 2), dtype=torch.float32, device=p.device)
        else:
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if p.dtype == torch.bfloat16:
            state["param_low"] = torch.zeros(p.shape, dtype=torch.int16, device=p.device)
        return state

    @staticmethod
    def _check_capture(work):
        for group, p, _, _, state in work:
            if not group["capturable"]:
                raise RuntimeError("FusedAdamW: a step that is captured needs capturable=True (its counts would stay where they are at every replay)")
            if state is None or not (torch.is_tensor(state["step"]) and state["step"].is_cuda):
                raise RuntimeError("FusedAdamW: run one step before the capture (states made during a capture would be cleared by every replay)")

    def _launch(self, work, mats, norm, max_norm, dev):
        lib = _lib.load()
        buckets, keep, counted = {}, [], []
        for (group, p, index, g, state), (gk, rows, row_len, stride) in zip(work, mats):
            bits, on_gpu = group["state_bits"], bool(group["capturable"])
            if state is None:
                state = self.state[p] = self._fresh_state(p, bits, on_gpu)
            lr, step, lr_dev, step_dev, t = group["lr"], state["step"], 0, 0, 0
            if on_gpu:
                if not torch.is_tensor(step) or step.device != dev or step.dtype != torch.float32:
                    step = state["step"] = torch.as_tensor(step, dtype=torch.float32).to(dev)
                step_dev = step.data_ptr()
                if torch.is_tensor(lr) and lr.is_cuda:
                    lr = lr.to(device=dev, dtype=torch.float32)
                    if lr.numel() != 1:
                        raise ValueError("FusedAdamW: lr must be one number")
                    keep.append(lr)
                    lr_dev, lr = lr.data_ptr(), 0.0
            else:
                t = int(step) + 1
                counted.append(state)
            low = 0
            if p.dtype == torch.bfloat16:
                low = state["param_low"].data_ptr()
            a, b = (state["moment_codes"], state["moment_scales"]) if bits == 8 else (state["exp_avg"], state["exp_avg_sq"])
            beta1, beta2 = group["betas"]
            buckets.setdefault((p.dtype == torch.bfloat16, bits, group["stochastic_rounding"], on_gpu), []).append(
                _STEP.pack(p.data_ptr(), gk.data_ptr(), low, a.data_ptr(), b.data_ptr(), step_dev, lr_dev, rows, stride, t, float(lr),
                           beta1, beta2, group["eps"], group["weight_decay"], row_len, group["seed"] & 0xFFFFFFFF, index, 0))
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        for (bf16, bits, stochastic, on_gpu), packed in buckets.items():
            scalars = torch.empty(4 * len(packed), dtype=torch.float32, device=dev) if on_gpu else None
            _lib.check(lib.gs_adamw_step(len(packed), _table(_lib.GsAdamWTensor, packed), bf16, bits, stochastic, _ptr(norm),
                                         0.0 if max_norm is None else float(max_norm), _ptr(scalars), stream), "gs_adamw_step")
        for state in counted:                    # after the launch: a refused call leaves the counts as they were
            state["step"] += 1

    @torch.no_grad()
    def update_densify_stats(self, viewspace_grad=None, radii=None, xyz_gradient_accum=None, denom=None, max_radii2D=None):
        """The densification statistics of FusedAdam.update_densify_stats (train.py:184-193)."""
        if radii is None:
            raise ValueError("update_densify_stats needs radii (the rasterizer's second output)")
        stats = FusedAdam._check_stats(viewspace_grad, radii, xyz_gradient_accum, denom, max_radii2D)
        FusedAdam._launch(self, [], stats, radii.device)

    # ---- rows -------------------------------------------------------------------------------------------------------
    def _group_of(self, p):
        for group in self.param_groups:
            for q in group["params"]:
                if q is p:
                    return group
        raise ValueError("not a parameter of this optimizer")

    @torch.no_grad()
    def gather_state(self, params, index):
        """States for tensors whose row i is row ``index[i]`` of each of ``params``: a list of state dicts in their order.

        ``index``: (M,) int64 on the GPU.  The same row may be taken more than once; an index outside 0..rows-1 (-1) gives a
        fresh row: moments zero.  All ``params`` have the same number of rows.  Counts are taken over; a parameter that
        has no state yet gives an empty dict.  Nothing of the optimizer changes; one launch per 32 tensors."""
        params = list(params)
        if not params:
            return []
        if not torch.is_tensor(index) or index.dtype != torch.int64 or index.dim() != 1:
            raise ValueError("index must be a 1-d int64 tensor (of a mask: mask.nonzero()[:, 0])")
        n, m = (params[0].shape[0] if params[0].dim() else -1), index.shape[0]
        buckets, out, keep = {}, [], []
        for p in params:
            if p.dim() < 1 or p.shape[0] != n:
                raise ValueError("gather_state: all params need the same number of rows")
            if not p.is_cuda or p.device != params[0].device or index.device != p.device:
                raise RuntimeError("gather_state: params and index must live on one GPU (no CPU path)")
            bits = self._group_of(p)["state_bits"]
            state = self.state.get(p) or None
            if state is None:
                out.append({})
                continue
            self._check_state(p, state, bits)
            step = state["step"]
            new = {"step": step.clone() if torch.is_tensor(step) else step}
            shape = (m,) + tuple(p.shape[1:])
            row_len = 1
            for d in p.shape[1:]:
                row_len *= d
            if row_len >= 1 << 31:
                raise ValueError(f"gather_state: rows of {row_len} elements are too long")
            if bits == 8:
                names = ("moment_codes", "moment_scales")
                new["moment_codes"] = torch.empty(shape + (2,), dtype=torch.uint8, device=p.device)
                new["moment_scales"] = torch.empty(((m * row_len + BLOCK - 1) // BLOCK, 2), dtype=torch.float32, device=p.device)
            else:
                names = ("exp_avg", "exp_avg_sq")
                new["exp_avg"] = torch.empty(shape, dtype=torch.float32, device=p.device)
                new["exp_avg_sq"] = torch.empty(shape, dtype=torch.float32, device=p.device)
            low = state.get("param_low")
            if low is not None:
                new["param_low"] = torch.empty(shape, dtype=torch.int16, device=p.device)
            if row_len:
                buckets.setdefault(bits, []).append(_lib.GsAdamWRows(
                    state[names[0]].data_ptr(), state[names[1]].data_ptr(), None if low is None else low.data_ptr(), new[names[0]].data_ptr(),
                    new[names[1]].data_ptr(), None if low is None else new["param_low"].data_ptr(), row_len, 0))
            out.append(new)
        lib = _lib.load()
        with torch.cuda.device(params[0].device), _stage("adamw_rows"):
            index = index.contiguous()
            stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
            for bits, rows in buckets.items():
                _lib.check(lib.gs_adamw_gather_rows(len(rows), (_lib.GsAdamWRows * len(rows))(*rows), bits, n, m, _ptr(index), stream),
                           "gs_adamw_gather_rows")
        return out

    def replace_params(self, old, new, index):
        """Puts ``new[k]`` in the place of ``old[k]`` in its group, with the state of the rows ``index`` (see gather_state): the
        reference's _prune_optimizer and cat_tensors_to_optimizer (scene/gaussian_model.py:476-530) in one call."""
        old, new = list(old), list(new)
        if len(old) != len(new) or len({id(p) for p in old}) != len(old) or len({id(p) for p in new}) != len(new):
            raise ValueError("replace_params: as many new parameters as old ones, each once")
        for p, q in zip(old, new):
            if not torch.is_tensor(q) or not q.is_leaf:
                raise ValueError("replace_params: new parameters must be leaf tensors")
            if q.dtype != p.dtype or q.device != p.device or p.dim() < 1 or tuple(q.shape) != tuple(index.shape) + tuple(p.shape[1:]):
                raise ValueError(f"replace_params: {tuple(q.shape)} {q.dtype} cannot take the place of {tuple(p.shape)} {p.dtype} with index {tuple(index.shape)}")
        places = [self._group_of(p)["params"] for p in old]
        others = {id(q) for group in self.param_groups for q in group["params"]} - {id(p) for p in old}
        if any(id(q) in others for q in new):
            raise ValueError("replace_params: a new parameter is already one of this optimizer's")
        states = self.gather_state(old, index)
        for p in old:
            self.state.pop(p, None)
        at = [next(i for i, r in enumerate(place) if r is p) for p, place in zip(old, places)]
        for place, i, q, state in zip(places, at, new, states):
            place[i] = q
            if state:
                self.state[q] = state

    # ---- what states stand for ----------------------------------------------------------------------------------------
    @torch.no_grad()
    def unpacked(self, params=None, *, states=None):
        """[{"param", "exp_avg", "exp_avg_sq"}] in float32 for ``params`` (all that have a state), or for ``states`` as gather_state
        returns them (without "param").  What is kept in float32 already is returned itself, the rest is
        computed by one launch per 32 tensors: 8-bit moments, and the values behind bfloat16 parameters."""
        if states is not None:
            if params is not None:
                raise ValueError("unpacked: params or states, not both")
            pairs = [(None, s) for s in states]
        else:
            if params is None:
                params = [p for group in self.param_groups for p in group["params"] if self.state.get(p)]
            pairs = [(p, self.state.get(p) or {}) for p in params]
        out, packed, dev = [], [], None
        for p, s in pairs:
            got, codes, low = {}, s.get("moment_codes"), s.get("param_low")
            if p is not None and s:
                self._check_state(p, s, self._group_of(p)["state_bits"])
            entry = _lib.GsAdamWUnpack()
            if codes is not None:
                scales = s["moment_scales"]
                if not (codes.is_cuda and codes.is_contiguous() and scales.is_contiguous()) or codes.dtype != torch.uint8 or \
                        scales.dtype != torch.float32 or scales.shape != ((codes.numel() // 2 + BLOCK - 1) // BLOCK, 2) or scales.device != codes.device:
                    raise RuntimeError("unpacked: not a state of FusedAdamW on the GPU")
                got["exp_avg"] = torch.empty(codes.shape[:-1], dtype=torch.float32, device=codes.device)
                got["exp_avg_sq"] = torch.empty_like(got["exp_avg"])
                entry.codes, entry.scales = codes.data_ptr(), scales.data_ptr()
                entry.exp_avg, entry.exp_avg_sq, entry.numel = got["exp_avg"].data_ptr(), got["exp_avg_sq"].data_ptr(), got["exp_avg"].numel()
            elif s:
                got["exp_avg"], got["exp_avg_sq"] = s["exp_avg"], s["exp_avg_sq"]
            if p is not None:
                got["param"] = p.detach()
                if p.dtype == torch.bfloat16 and low is not None:
                    got["param"] = torch.empty(p.shape, dtype=torch.float32, device=p.device)
                    entry.param_bf16, entry.param_low, entry.param, entry.numel = p.data_ptr(), low.data_ptr(), got["param"].data_ptr(), p.numel()
            out.append(got)
            if entry.numel:
                here = codes.device if codes is not None else p.device
                if dev not in (None, here):
                    raise RuntimeError("unpacked: all tensors must live on one device")
                dev = here
                packed.append(entry)
        if packed:
            with torch.cuda.device(dev), _stage("adamw_unpack"):
                _lib.check(_lib.load().gs_adamw_unpack(len(packed), (_lib.GsAdamWUnpack * len(packed))(*packed),
                                                       C.c_void_p(torch.cuda.current_stream().cuda_stream)), "gs_adamw_unpack")
        return out

    # ---- checkpoints --------------------------------------------------------------------------------------------------
    def load_state_dict(self, state_dict):
        """torch's, but every state keeps its own type (the base class casts it to the parameter's) and memory.  A
        state_dict of torch.optim.AdamW / Adam or FusedAdam is taken by groups with state_bits=32."""
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        bits = [group.get("state_bits", mine["state_bits"]) for group, mine in zip(state_dict["param_groups"], self.param_groups)
                for _ in group["params"]]
        for i, b in zip(saved, bits):
            state = state_dict["state"].get(i)
            if state and ("moment_codes" if b == 8 else "exp_avg") not in state:
                raise ValueError(f"state_dict holds no states in {b} bits for parameter {i}")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            self._complete(group)
        params = [(group, p) for group in self.param_groups for p in group["params"]]
        for i, (group, p) in zip(saved, params):
            state = state_dict["state"].get(i)
            if not state:
                continue
            names = ("moment_codes", "moment_scales") if group["state_bits"] == 8 else ("exp_avg", "exp_avg_sq")
            mine = {"step": torch.as_tensor(state["step"], dtype=torch.float32).to(p.device if group["capturable"] else "cpu", copy=True)}
            for name in names:
                mine[name] = state[name].to(p.device, torch.uint8 if name == "moment_codes" else torch.float32, copy=True).contiguous()
            if p.dtype == torch.bfloat16:
                low = state.get("param_low")
                mine["param_low"] = (torch.zeros(p.shape, dtype=torch.int16, device=p.device) if low is None
                                     else low.to(p.device, torch.int16, copy=True).contiguous())
            self.state[p] = mine
