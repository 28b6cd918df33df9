"""AdamW over many tensors with moments in 32 or in 8 bits, the global gradient norm, and the state's rows.

``FusedAdamW`` stands beside ``FusedAdam`` (optimizer.py) for training with decoupled weight decay: a
``torch.optim.AdamW`` whose ``step()`` is one HIP launch per 32 tensors (gs_adamw_step).  Beyond torch's class:

    state_bits=8            two bytes of state per element instead of eight (a Gaussian model's moments: 472 -> 125 bytes per
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

import struct

import torch

from . import _lib
from .optimizer import FusedAdam
from .profiling import stage as _stage

BLOCK = 64                                       # GS_ADAMW_BLOCK: elements that share a pair of scales
_F32, _BF16 = torch.float32, torch.bfloat16

_stream = torch._C._cuda_getCurrentRawStream     # of a device index; torch.cuda.current_stream() takes 2.5 us to make its object

# The descriptors of include/gsplat.h as packed bytes: a step describes every tensor anew, and a small model's step takes as long as that does.
_STEP = struct.Struct("@7P3q5diIIi").pack        # GsAdamWTensor
_GRAD = struct.Struct("@P2q2i").pack             # GsGradTensor
_ROWS = struct.Struct("@6P2i").pack              # GsAdamWRows
_UNPACK = struct.Struct("@7Pq").pack             # GsAdamWUnpack


class _On:
    """The device context of a call, entered only where the device is not the current one already."""
    __slots__ = ("ctx",)

    def __init__(self, dev):
        self.ctx = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)


def _matrix(g):
    """(tensor to keep alive, rows, row length, row stride) of a gradient: rows that are contiguous in themselves are taken where they are."""
    if g.is_contiguous():
        return g, g.numel(), 1, 0
    shape, strides = g.shape, g.stride()
    if shape[0] > 1:
        row_len = 1
        for d in range(len(shape) - 1, 0, -1):
            if strides[d] != row_len and shape[d] != 1:
                break
            row_len *= shape[d]
        else:
            if 0 < row_len <= strides[0] and row_len < 1 << 31:
                return g, shape[0], row_len, strides[0]
    return g.detach().contiguous(), g.numel(), 1, 0


def _refuse_grad(g, what):
    if g.layout is not torch.strided or not g.is_cuda:
        raise RuntimeError(f"{what} must be a dense tensor on the GPU (no CPU path)")
    raise RuntimeError(f"{what} must be float32 or bfloat16, not {g.dtype}")


def _norm(mats, dev, stream):
    """Launches gs_grad_norm over matrices of _matrix() on `stream` of `dev`, the current device."""
    lib = _lib.load()
    table = b"".join([_GRAD(g.data_ptr(), rows, stride, row_len, g.dtype is _BF16) for g, rows, row_len, stride in mats])
    size = lib.gs_grad_norm_workspace_bytes(len(mats), table)
    ws = torch.empty(max(size, 8), dtype=torch.uint8, device=dev)
    out = torch.empty((), dtype=_F32, device=dev)
    _lib.check(lib.gs_grad_norm(len(mats), table, out.data_ptr(), ws.data_ptr(), size, stream), "gs_grad_norm")
    return out


def grad_norm(grads):
    """sqrt of the sum of squares over all given tensors (None is skipped) as a 0-d float32 GPU tensor.

    float32 and bfloat16, any strides; accumulated in fp64 in a fixed order, so it neither overflows before its result does nor
    depends on scheduling.  Nothing is synchronised.  For gradients sharded over ranks, pass the result through
    ``parallel.reduce_grad_norm`` and on to ``FusedAdamW.step(max_norm=..., grad_norm=...)``."""
    grads = [grads] if torch.is_tensor(grads) else [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grad_norm needs at least one tensor")
    dev = grads[0].device
    for g in grads:
        if g.layout is not torch.strided or not g.is_cuda or g.dtype is not _F32 and g.dtype is not _BF16:
            _refuse_grad(g, "grad_norm: a gradient")
        if g.get_device() != dev.index:
            raise RuntimeError("grad_norm: all gradients must live on one device")
    with _On(dev), _stage("grad_norm"):
        return _norm([_matrix(g) for g in grads], dev, _stream(dev.index))


def _counts_on(step, dev):
    return torch.is_tensor(step) and step.dtype is _F32 and step.get_device() == dev.index


class _Plan:
    """One step's launches: packed descriptors by kernel form, what has to live until they are made, and the tensors (fresh) whose
    state or count on the GPU has to be made first."""
    __slots__ = ("dev", "params", "mats", "fresh", "counted", "keep", "buckets")

    def __init__(self):
        self.dev, self.params, self.mats, self.fresh, self.counted, self.keep, self.buckets = None, [], [], [], [], [], {}

    def add(self, p, group, options, index, mat, state):
        g, rows, row_len, stride = mat
        lr_dev, lr, beta1, beta2, eps, weight_decay, seed = options
        bits, on_gpu, step, step_dev, t = group["state_bits"], bool(group["capturable"]), state["step"], 0, 0
        if on_gpu:
            step_dev = step.data_ptr()
        else:
            t = int(step) + 1
            self.counted.append((state, step, t))
        if bits == 8:
            a, b = state["moment_codes"], state["moment_scales"]
        else:
            a, b = state["exp_avg"], state["exp_avg_sq"]
        bf16 = p.dtype is _BF16
        key = (bf16, bits, group["stochastic_rounding"], on_gpu)
        packed = self.buckets.get(key)
        if packed is None:
            packed = self.buckets[key] = []
        packed.append(_STEP(p.data_ptr(), g.data_ptr(), state["param_low"].data_ptr() if bf16 else 0, a.data_ptr(), b.data_ptr(), step_dev, lr_dev,
                            rows, stride, t, lr, beta1, beta2, eps, weight_decay, row_len, seed, index, 0))


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
        self.defaults.update(state_bits=state_bits, stochastic_rounding=bool(stochastic_rounding), seed=int(seed))
        for group in self.param_groups:
            self._complete(group)

    last_grad_norm = None

    def _complete(self, group):
        for k in ("state_bits", "stochastic_rounding", "seed"):
            group.setdefault(k, self.defaults[k])
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {group['state_bits']!r}")

    def add_param_group(self, param_group):
        if "state_bits" in self.defaults:        # not yet while the base class adds the first groups
            self._complete(param_group)
        super().add_param_group(param_group)

    # ---- the step ---------------------------------------------------------------------------------------------------
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
        plan = self._plan()
        self.last_grad_norm = None
        dev = plan.dev
        if dev is None:
            return loss
        if grad_norm is not None and (not torch.is_tensor(grad_norm) or grad_norm.device != dev or grad_norm.dtype is not _F32
                                      or grad_norm.numel() != 1):
            raise ValueError("grad_norm must be one float32 on the parameters' device")
        with _On(dev), _stage("adamw"):
            if (plan.counted or plan.fresh) and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedAdamW: a step that is captured needs capturable=True, or its counts would stay where they are at every replay"
                                   if plan.counted or not all(group["capturable"] for _, group, _, _ in plan.fresh) else
                                   "FusedAdamW: run one step before the capture: states and counts made during it would be made again by every replay")
            states = self.state
            for p, group, index, mat in plan.fresh:
                state = states.get(p) or None
                if state is None:
                    state = states[p] = self._fresh_state(p, group["state_bits"], group["capturable"])
                elif group["capturable"]:
                    state["step"] = torch.as_tensor(state["step"], dtype=_F32).to(dev)
                plan.add(p, group, self._options(group, dev, plan.keep), index, mat, state)
            stream = _stream(dev.index)
            if max_norm is not None and grad_norm is None:
                grad_norm = _norm(plan.mats, dev, stream)
            lib = _lib.load()
            for (bf16, bits, stochastic, on_gpu), packed in plan.buckets.items():
                scalars = torch.empty(4 * len(packed), dtype=_F32, device=dev) if on_gpu else None
                _lib.check(lib.gs_adamw_step(len(packed), b"".join(packed), bf16, bits, stochastic, None if grad_norm is None else grad_norm.data_ptr(),
                                             0.0 if max_norm is None else float(max_norm), None if scalars is None else scalars.data_ptr(),
                                             stream), "gs_adamw_step")
        for state, step, t in plan.counted:      # after the launches: a refused call leaves the counts as they were
            if torch.is_tensor(step):
                step.fill_(t)
            else:
                state["step"] = t
        self.last_grad_norm = grad_norm
        torch.autograd.graph.increment_version(plan.params)
        return loss

    def _plan(self):
        """Everything that the step updates, checked before anything changes."""
        plan, dev, index, spans, states = _Plan(), None, -1, [], self.state
        for group in self.param_groups:
            if group["amsgrad"] or group["maximize"] or group["differentiable"]:
                raise NotImplementedError("FusedAdamW: amsgrad / maximize / differentiable are not implemented")
            beta1, beta2 = group["betas"]
            bits, options = group["state_bits"], None
            if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0 and group["eps"] >= 0.0 and bits in (8, 32)):
                raise ValueError(f"FusedAdamW: betas {group['betas']}, eps {group['eps']}, state_bits {bits}: betas are in "
                                 "[0, 1), eps is not negative, state_bits is 8 or 32")
            for p in group["params"]:
                index += 1
                g = p.grad
                if g is None:
                    continue
                dtype = p.dtype
                if not p.is_cuda or dtype is not _F32 and dtype is not _BF16 or not p.is_contiguous():
                    raise RuntimeError("FusedAdamW needs contiguous float32 or bfloat16 parameters on the GPU (no CPU path)")
                if g.layout is not torch.strided:
                    _refuse_grad(g, "FusedAdamW: a gradient")
                if dev is None:
                    dev = p.device
                if g.dtype is not dtype or p.get_device() != dev.index or g.get_device() != dev.index:
                    raise RuntimeError("FusedAdamW: all parameters must live on one device, with gradients of their type there")
                n = p.numel()
                if n:
                    start = p.data_ptr()
                    spans.append((start, start + n * (4 if dtype is _F32 else 2)))
                plan.params.append(p)
                state = states.get(p) or None
                if state is not None:
                    self._check_state(p, state, bits)
                mat = _matrix(g)
                plan.mats.append(mat)
                if state is None or group["capturable"] and not _counts_on(state["step"], dev):
                    plan.fresh.append((p, group, index, mat))
                    continue
                if options is None:
                    options = self._options(group, dev, plan.keep)
                plan.add(p, group, options, index, mat, state)
        spans.sort()
        end = 0
        for start, stop in spans:
            if start < end:
                raise RuntimeError("FusedAdamW: two parameters share memory (or one is listed twice)")
            end = stop
        plan.dev = dev
        return plan

    @staticmethod
    def _options(group, dev, keep):
        """What the descriptors of a group's tensors have in common: (lr_dev, lr, beta1, beta2, eps, weight_decay, seed)."""
        lr, lr_dev = group["lr"], 0
        if group["capturable"] and torch.is_tensor(lr) and lr.is_cuda:
            lr = lr.detach().to(device=dev, dtype=_F32)
            if lr.numel() != 1:
                raise ValueError("FusedAdamW: lr must be one number")
            keep.append(lr)
            lr_dev, lr = lr.data_ptr(), 0.0
        return (lr_dev, float(lr), *group["betas"], group["eps"], group["weight_decay"], group["seed"] & 0xFFFFFFFF)

    @staticmethod
    def _check_state(p, state, bits):
        dev, shape = p.get_device(), p.shape
        if bits == 8:
            a, b = state.get("moment_codes"), state.get("moment_scales")
            good = (a is not None and b is not None and a.dtype is torch.uint8 and a.shape == shape + (2,)
                    and b.shape == ((p.numel() + BLOCK - 1) // BLOCK, 2))
        else:
            a, b = state.get("exp_avg"), state.get("exp_avg_sq")
            good = a is not None and b is not None and a.dtype is _F32 and a.shape == shape and b.shape == shape
        if p.dtype is _BF16:
            low = state.get("param_low")
            good = good and low is not None and low.dtype is torch.int16 and low.shape == shape and low.is_contiguous() and low.get_device() == dev
        if not good or b.dtype is not _F32 or not (a.is_contiguous() and b.is_contiguous()) or a.get_device() != dev or b.get_device() != dev:
            raise RuntimeError(f"FusedAdamW: optimizer state does not match its parameter (shape {tuple(shape)}, {p.dtype}, state_bits {bits}); "
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
        dev, m = params[0].device, index.shape[0]
        n = params[0].shape[0] if params[0].dim() else -1
        group_of = {q: group for group in self.param_groups for q in group["params"]}
        buckets, out = {}, []
        for p in params:
            if p.dim() < 1 or p.shape[0] != n:
                raise ValueError("gather_state: all params need the same number of rows")
            if not p.is_cuda or p.device != dev or index.device != dev:
                raise RuntimeError("gather_state: params and index must live on one GPU (no CPU path)")
            if p not in group_of:
                raise ValueError("not a parameter of this optimizer")
            bits = group_of[p]["state_bits"]
            state = self.state.get(p) or None
            if state is None:
                out.append({})
                continue
            self._check_state(p, state, bits)
            step = state["step"]
            new = {"step": step.clone() if torch.is_tensor(step) else step}
            row = p.shape[1:]
            shape, row_len = (m,) + row, row.numel()
            if row_len >= 1 << 31:
                raise ValueError(f"gather_state: rows of {row_len} elements are too long")
            if bits == 8:
                a, b = state["moment_codes"], state["moment_scales"]
                x = new["moment_codes"] = a.new_empty(shape + (2,))
                y = new["moment_scales"] = b.new_empty(((m * row_len + BLOCK - 1) // BLOCK, 2))
            else:
                a, b = state["exp_avg"], state["exp_avg_sq"]
                x = new["exp_avg"] = a.new_empty(shape)
                y = new["exp_avg_sq"] = a.new_empty(shape)
            low_from = low_to = 0
            if p.dtype is _BF16:
                low_from, new["param_low"] = state["param_low"].data_ptr(), state["param_low"].new_empty(shape)
                low_to = new["param_low"].data_ptr()
            if row_len:
                buckets.setdefault(bits, []).append(_ROWS(a.data_ptr(), b.data_ptr(), low_from, x.data_ptr(), y.data_ptr(), low_to, row_len, 0))
            out.append(new)
        lib = _lib.load()
        with _On(dev), _stage("adamw_rows"):
            index = index.contiguous()
            for bits, rows in buckets.items():
                _lib.check(lib.gs_adamw_gather_rows(len(rows), b"".join(rows), bits, n, m, index.data_ptr(), _stream(dev.index)), "gs_adamw_gather_rows")
        return out

    def replace_params(self, old, new, index):
        """Puts ``new[k]`` in the place of ``old[k]`` in its group, with the state of the rows ``index`` (see gather_state): the
        reference's _prune_optimizer and cat_tensors_to_optimizer (scene/gaussian_model.py:476-530) in one call."""
        old, new = list(old), list(new)
        if not torch.is_tensor(index):
            raise ValueError("index must be a 1-d int64 tensor (of a mask: mask.nonzero()[:, 0])")
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
        group_of = {q: group for group in self.param_groups for q in group["params"]} if states is None else None
        for p, s in pairs:
            got, numel = {}, 0
            codes = m = v = x = low = scales = 0          # addresses
            if p is not None and s:
                if p not in group_of:
                    raise ValueError("not a parameter of this optimizer")
                self._check_state(p, s, group_of[p]["state_bits"])
            c = s.get("moment_codes")
            if c is not None:
                scale, here, numel = s["moment_scales"], c.device, c.numel() // 2
                if p is None and (not (c.is_cuda and c.is_contiguous() and scale.is_contiguous()) or c.dtype is not torch.uint8 or
                                  scale.dtype is not _F32 or scale.device != here or c.shape[-1:] != (2,) or
                                  scale.shape != ((numel + BLOCK - 1) // BLOCK, 2)):
                    raise RuntimeError("unpacked: not a state of FusedAdamW on the GPU")
                got["exp_avg"] = t = torch.empty_like(p) if p is not None and p.dtype is _F32 else scale.new_empty(c.shape[:-1])
                got["exp_avg_sq"] = w = torch.empty_like(t)
                codes, scales, m, v = c.data_ptr(), scale.data_ptr(), t.data_ptr(), w.data_ptr()
            elif s:
                got["exp_avg"], got["exp_avg_sq"] = s["exp_avg"], s["exp_avg_sq"]
            bits16 = 0
            if p is not None:
                if p.dtype is _F32 or not s:
                    got["param"] = p.detach() if p.dtype is _F32 else p.detach().float()
                else:
                    here, numel = p.device, p.numel()
                    got["param"] = t = torch.empty(p.shape, dtype=_F32, device=here)
                    bits16, low, x = p.data_ptr(), s["param_low"].data_ptr(), t.data_ptr()
            out.append(got)
            if numel:
                if dev is None:
                    dev = here
                elif dev != here:
                    raise RuntimeError("unpacked: all tensors must live on one device")
                packed.append(_UNPACK(codes, scales, bits16, low, m, v, x, numel))
        if packed:
            with _On(dev), _stage("adamw_unpack"):
                _lib.check(_lib.load().gs_adamw_unpack(len(packed), b"".join(packed), _stream(dev.index)), "gs_adamw_unpack")
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
        super().load_state_dict({**state_dict, "state": {}})
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
