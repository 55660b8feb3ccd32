"""Parameter update of the train step on the HIP kernels (csrc/step.hip):
torch.nn.utils.clip_grad_norm_ and torch.optim.AdamW (trainer.py:216-221,
hparams: AdamW, clip 0.5) over a device table of parameter slots, so a step
is three launches (sum of squares, clip, AdamW) whatever the tensor count.

Drop-in surface: ``AdamW`` takes torch.optim.AdamW's arguments (amsgrad,
maximize, capturable, differentiable off) and keeps its state layout
(state[p] = {'step', 'exp_avg', 'exp_avg_sq'}), so state_dicts load either way;
``clip_grad_norm_`` has torch's signature for the 2-norm and returns the
total norm as a device tensor. Both need contiguous CUDA tensors of one
storage type per call: fp32, or the bf16 / fp16 of a model.to(bfloat16) /
.half() run (ABI 10: torch's foreach AdamW rounding reproduced in the kernel).
There is no CPU path.

``AdamW(..., state_bits=32)`` keeps both moments in fp32 whatever the parameters' type,
``state_bits=8`` keeps m and sqrt(v) in one byte an element with a power of two for each 128
(csrc/adamw.hip: the table of tensors travels in the kernel's arguments, 48 a launch).
``adamw32_`` and ``adamw8_`` are the same steps on tensors in hand.
"""
from __future__ import annotations


import operator

import numpy as np
import torch

from . import _native as N

SUMSQ_DOUBLES = 2049   # SE_SUMSQ_DOUBLES (include/sehip.h)
_SLOT = np.dtype([("param", "<u8"), ("grad", "<u8"), ("exp_avg", "<u8"), ("exp_avg_sq", "<u8"),
                  ("numel", "<i8"), ("offset", "<i8")])


def _slot_table(rows, device):
    """Device array of se_tensor_slot for [(param, grad, exp_avg, exp_avg_sq)]
    (None -> NULL). Returns (table, nslots, total)."""
    arr = np.zeros(len(rows), dtype=_SLOT)
    off = 0
    for i, (p, g, m, v) in enumerate(rows):
        n = g.numel()
        arr[i] = (N.ptr(p) or 0, g.data_ptr(), N.ptr(m) or 0, N.ptr(v) or 0, n, off)
        off += n
    host = torch.from_numpy(arr.view(np.uint8)).pin_memory()
    return host.to(device, non_blocking=True), len(rows), off


def _check(ts):
    """The storage-type code (SE_DTYPE_*) shared by every tensor, or RuntimeError."""
    dt = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda or t.dtype not in N.DTYPES or not t.is_contiguous() or (dt is not None and t.dtype != dt):
            raise RuntimeError("sehip optim: parameters and gradients must be contiguous CUDA tensors of one "
                               "storage type (fp32, bf16 or fp16; there is no CPU path)")
        dt = t.dtype
    return N.DTYPES[dt] if dt is not None else 0


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ (2-norm): scales every .grad in place by
    min(max_norm / (total_norm + 1e-6), 1) and returns total_norm (device fp32).
    Sum of squares in fp64 (torch: fp32 per-tensor norms)."""
    if float(norm_type) != 2.0:
        raise NotImplementedError("sehip clip_grad_norm_: only the 2-norm (the reference's)")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    code = _check(grads)
    dev = grads[0].device
    table, n, total = _slot_table([(None, g, None, None) for g in grads], dev)
    sumsq = torch.empty(SUMSQ_DOUBLES, device=dev, dtype=torch.float64)
    norm = torch.empty(1, device=dev, dtype=torch.float32)
    st = N.stream_of(grads[0])
    N.check(N.lib().se_grad_sumsq(table.data_ptr(), n, total, sumsq.data_ptr(), code, st), "se_grad_sumsq")
    if error_if_nonfinite and not torch.isfinite(sumsq[0]).item():   # [0] = the total (SE_SUMSQ_DOUBLES)
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` "
                           "is non-finite, so it cannot be clipped")
    N.check(N.lib().se_clip_grads(table.data_ptr(), n, total, sumsq.data_ptr(), float(max_norm), norm.data_ptr(),
                                  code, st), "se_clip_grads")
    return norm.view(())


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW on se_adamw_step: one launch per (parameter group, step
    count). Parameters of a group normally share their step count; one that
    missed steps (no gradient on some iterations, or a loaded state_dict with
    per-parameter steps) is updated by its own launch with its own bias
    corrections, as torch tracks the step per parameter.

    state_bits (a group may have its own, and its own seed) None: the moments in the parameters' type (torch's state layout). 32: state[p] =
    {'step', 'exp_avg', 'exp_avg_sq'} with fp32 moments. 8: {'step', 'exp_avg', 'exp_avg_scale',
    'exp_avg_root', 'exp_avg_root_scale'}, e4m3 values of m and sqrt(v) and their e8m0 powers of two,
    rounded stochastically from `seed`: the replicas of a data-parallel run, given one seed and the same
    gradients, keep the same states."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False,
                 *, maximize=False, foreach=None, capturable=False, differentiable=False, fused=None,
                 state_bits=None, seed=0):
        if amsgrad or maximize or capturable or differentiable:
            raise NotImplementedError("sehip AdamW: amsgrad / maximize / capturable / differentiable")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, maximize=False,
                        foreach=None, capturable=False, differentiable=False, fused=None)
        if state_bits is not None:
            defaults.update(state_bits=state_bits, seed=int(seed))
        self._seed = int(seed)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        """As torch's; a group may have its own state_bits and seed."""
        bits = param_group.get("state_bits", self.defaults.get("state_bits")) if isinstance(param_group, dict) else None
        if bits is not None:
            if bits not in (8, 32):
                raise ValueError(f"sehip AdamW: state_bits {bits!r} (None, 8 or 32)")
            param_group["state_bits"] = int(bits)
            param_group["seed"] = int(param_group.get("seed", getattr(self, "_seed", 0)))
        super().add_param_group(param_group)

    def load_state_dict(self, state_dict):
        """As torch's, but the moments of state_bits 8 / 32 keep their own type (torch casts a state to its
        parameter's). A state without the keys or types of this optimizer's state_bits is refused before anything
        is replaced; None and 32 take moments of any floating type of 16 bits or more."""
        given = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [(p, g.get("state_bits")) for g in self.param_groups for p in g["params"]]
        if len(ids) != len(mine):   # torch says which group differs
            return super().load_state_dict(state_dict)
        keep = []
        for i, (p, bits) in zip(ids, mine):
            if i not in given:
                continue
            if bits is None:   # torch would take 8-bit codes, without their scales, for numbers
                for key in ("exp_avg", "exp_avg_sq") if given[i] else ():
                    t = given[i].get(key)
                    if t is None or not t.is_floating_point() or t.element_size() == 1:
                        raise ValueError(f"sehip AdamW: the loaded state has no {key} for state_bits=None")
                continue
            keep.append((p, "step", torch.as_tensor(given[i]["step"]).clone()))
            want = _state_like(p, bits)
            for key, like in want.items():
                t = given[i].get(key)
                if t is None or t.shape != like.shape or (
                        t.dtype != like.dtype if bits == 8 else not t.is_floating_point() or t.element_size() == 1):
                    raise ValueError(f"sehip AdamW: the loaded state has no {key} for state_bits={bits}")
                keep.append((p, key, t.to(device=p.device, dtype=like.dtype, copy=True)))
        own = [{k: g[k] for k in ("state_bits", "seed") if k in g} for g in self.param_groups]
        super().load_state_dict(state_dict)
        for g, o in zip(self.param_groups, own):   # the layout of the state is this optimizer's, not the file's
            g.pop("state_bits", None)
            g.update({**o, **({"seed": g["seed"]} if "seed" in o and "seed" in g else {})})
        for p, key, t in keep:
            self.state[p][key] = t

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for at, group in enumerate(self.param_groups):
            if group.get("state_bits") is not None:
                self._step_multi(at, group)
                continue
            by_step: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("sehip AdamW: sparse gradients")
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] += 1
                s = int(st["step"].item())   # a CPU tensor, as torch's non-capturable AdamW
                by_step.setdefault(s, []).append((p, p.grad.resolve_neg(), st["exp_avg"], st["exp_avg_sq"]))
            b1, b2 = group["betas"]
            for step_val, rows in sorted(by_step.items()):
                by_dtype: dict = {}
                for r in rows:
                    by_dtype.setdefault(r[0].dtype, []).append(r)
                for rs in by_dtype.values():
                    code = _check([t for r in rs for t in r])
                    table, n, total = _slot_table(rs, rs[0][0].device)
                    N.check(N.lib().se_adamw_step(table.data_ptr(), n, total, float(group["lr"]), float(b1),
                                                  float(b2), float(group["eps"]), float(group["weight_decay"]),
                                                  step_val, code, N.stream_of(rs[0][0])), "se_adamw_step")
        return loss

    def _step_multi(self, at, group):
        bits = group["state_bits"]
        calls: dict = {}
        for p in group["params"]:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError("sehip AdamW: sparse gradients")
            st = self.state[p]
            if len(st) == 0:
                st["step"] = torch.tensor(0.0)
                st.update(_state_like(p, bits, torch.zeros))
            calls.setdefault((int(st["step"].item()) + 1, p.dtype, p.device), []).append(p)
        kw = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"])
        for call, ((step, _, _), ps) in enumerate(sorted(calls.items(), key=lambda c: c[0][0])):
            sts = [self.state[p] for p in ps]
            states = [[st[k] for st in sts] for k in _STATE_KEYS[bits]]
            if bits == 8:   # random bits of the group's own, and of each call's (which counts its tensors from 0)
                adamw8_(ps, [p.grad for p in ps], *states, step=step, seed=group["seed"] + 0x10001 * at + (call << 32), **kw)
            else:
                adamw32_(ps, [p.grad for p in ps], *states, step=step, **kw)
            for st in sts:   # counted once the launch has gone through
                st["step"] += 1


_dtype_of = operator.attrgetter("dtype")
SCALE_BLOCK = 128   # SE_ADAMW_BLOCK (include/sehip.h)
_STATE_KEYS = {32: ("exp_avg", "exp_avg_sq"),
               8: ("exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale")}
_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _state_like(p, bits, new=torch.empty):
    """The moments of a parameter: what AdamW keeps for it (new = torch.zeros), or their shapes and types."""
    if new is torch.empty:
        p = torch.empty(p.shape, device="meta")
    if bits == 32:
        return {k: new(p.shape, device=p.device, dtype=torch.float32) for k in _STATE_KEYS[32]}
    blocks = -(-p.numel() // SCALE_BLOCK)
    return {k: new(blocks if k.endswith("scale") else p.shape, device=p.device, dtype=torch.uint8).view(
        _E8 if k.endswith("scale") else _F8) for k in _STATE_KEYS[8]}


_TENSOR = np.dtype([("param", "<u8"), ("grad", "<u8"), ("exp_avg", "<u8"), ("exp_avg_sq", "<u8"),
                    ("exp_avg_scale", "<u8"), ("exp_avg_sq_scale", "<u8"), ("numel", "<i8")])   # se_adamw_tensor


def _multi(params, columns, types, bits, step, lr, betas, eps, weight_decay, seed):
    """se_adamw_multi over `params` and the columns grad, exp_avg, exp_avg_sq (, their scales)."""
    n = len(params)
    if any(len(c) != n for c in columns):
        raise ValueError("sehip adamw: lists of different lengths")
    if n == 0:
        return
    if step < 1:
        raise ValueError(f"sehip adamw: step {step} (counted from 1)")
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"sehip adamw: betas {betas}")
    if any(map(torch.Tensor.is_neg, columns[0])):   # one element that is an imaginary part: negated lazily
        columns = ([g.resolve_neg() for g in columns[0]], *columns[1:])
    p0 = params[0]
    dev, dt = p0.device, p0.dtype
    if dev.type != "cuda" or dt not in N.DTYPES:
        raise RuntimeError("sehip adamw: parameters must be fp32, bf16 or fp16 CUDA tensors (there is no CPU path)")
    T = torch.Tensor
    index = p0.get_device()
    sizes = list(map(T.numel, params))
    blocks = [-(-k // SCALE_BLOCK) for k in sizes] if bits == 8 else None
    arr = np.zeros(n, dtype=_TENSOR)
    written = []
    for name, ts, ty in zip(_TENSOR.names, (params, *columns), (dt, *types)):
        want = blocks if name.endswith("scale") else sizes
        if (list(map(T.numel, ts)) != want or set(map(_dtype_of, ts)) != {ty} or set(map(T.get_device, ts)) != {index}
                or not all(map(T.is_contiguous, ts))):
            raise RuntimeError(f"sehip adamw: {name}: not all contiguous {ty} tensors of the parameters' sizes on {dev}")
        arr[name] = at = list(map(T.data_ptr, ts))
        if name == "grad":
            grads = at
        else:
            written += at
            if len(set(at)) < n and len({a for a, k in zip(at, sizes) if k}) < sum(map(bool, sizes)):
                raise RuntimeError(f"sehip adamw: the same {name} twice in the list")
    arr["numel"] = sizes
    if len(set(written)) < len(written) or not set(grads).isdisjoint(written):   # or some without elements
        full = [a for a, k in zip(written, sizes * (len(written) // n)) if k]
        if len(set(full)) < len(full) or not {a for a, k in zip(grads, sizes) if k}.isdisjoint(full):
            raise RuntimeError("sehip adamw: one tensor in two of the lists")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("sehip adamw: a captured graph would repeat this step's count and bias corrections")
    N.launch(index, "se_adamw_multi", N.lib().se_adamw_multi, arr.ctypes.data, n, N.DTYPES[dt], bits, float(lr), float(betas[0]),
             float(betas[1]), float(eps), float(weight_decay), int(step), int(seed) & 0xFFFFFFFFFFFFFFFF)
    torch.autograd.graph.increment_version([t for ts in (params, *columns[1:]) for t in ts])


@torch.no_grad()
def adamw32_(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """One AdamW step in place over lists of contiguous tensors on one GPU: parameters and gradients of one type
    (fp32, bf16, fp16), moments in fp32. step counts from 1."""
    _multi(params, (grads, exp_avgs, exp_avg_sqs), (params[0].dtype if params else None, torch.float32, torch.float32), 32,
           step, lr, betas, eps, weight_decay, 0)


@torch.no_grad()
def adamw8_(params, grads, exp_avgs, exp_avg_scales, roots, root_scales, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
            weight_decay=1e-2, seed=0):
    """One AdamW step in place whose moments are held in 8 bits: exp_avgs and roots (m and sqrt(v)) float8_e4m3fn of
    the parameters' shapes, the scales float8_e8m0fnu [ceil(numel / 128)]. m and v are rounded stochastically with a hash of
    (seed, step, place in the list, element): the same call gives the same bits."""
    _multi(params, (grads, exp_avgs, roots, exp_avg_scales, root_scales),
           (params[0].dtype if params else None, _F8, _F8, _E8, _E8), 8, step, lr, betas, eps, weight_decay, seed)
