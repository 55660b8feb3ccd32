"""BatchNorm2d + activation on the HIP kernels (csrc/bn.hip): the
ConvBlock / ConvTransposeBlock body of CARN / GCARN (BatchNorm2d + PReLU,
models/_2104_05267_carn.py:30-56) and CRN (BatchNorm2d + ELU,
models/_1809_01405_crn.py:9-45). The modules stay nn.BatchNorm2d / nn.PReLU /
nn.ELU (constructor, parameters, buffers and state_dict keys unchanged);
``bn_act(norm, act, x)`` replaces ``act(norm(x))`` with one fused forward and
backward (training: batch statistics and the running-stat update as
nn.BatchNorm2d with a float momentum; eval: running statistics).
Configurations the kernels do not cover (momentum=None, non-4-D input, other
activations) run the modules themselves.

``layer_norm(norm, x)`` replaces ``norm(x)`` of an nn.LayerNorm, forward and
backward (csrc/layernorm.hip): any leading shape, rows at any distance, fp32 / bf16 /
fp16 storage with the weight and bias in the same type or in fp32, the weight's and
bias's gradients summed in a fixed order. CPU tensors raise."""
from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native as N
from . import glue

_ACT_NONE, _ACT_PRELU, _ACT_ELU = 0, 1, 2


def _plane_stride(x):
    """Plane stride of a [B, C, H, W] tensor whose (b, c) planes are each HW
    contiguous floats at a constant stride (a row-cropped view qualifies)."""
    B, C, H, W = x.shape
    if x.stride(3) == 1 and x.stride(2) == W and x.stride(0) == C * x.stride(1) and x.stride(1) >= H * W:
        return x.stride(1)
    return None


class _BnAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act_param, rmean, rvar, training, momentum, eps, act, per_channel, alpha):
        # fp32, or bf16 / fp16 storage throughout (model.half() / .to(bfloat16)): read and
        # written in that dtype by the kernels, fp32 arithmetic
        N.require_device(x, weight, bias, act_param, rmean, rvar, dtype=x.dtype)
        dt = N.dtype_code(x)
        ps = _plane_stride(x)
        if ps is None:
            x = x.contiguous()
            ps = x.stride(1)
        B, C, H, W = x.shape
        y = torch.empty((B, C, H, W), device=x.device, dtype=x.dtype)
        save = torch.empty(2 * C, device=x.device, dtype=torch.float32)
        ws = torch.empty(int(N.lib().se_bn_workspace_size(B, C)), device=x.device, dtype=torch.uint8)
        N.check(N.lib().se_bn_fwd(x.data_ptr(), ps, B, C, H * W, N.ptr(weight), N.ptr(bias), N.ptr(rmean),
                                  N.ptr(rvar), int(training), float(momentum), float(eps), act, N.ptr(act_param),
                                  int(per_channel), float(alpha), y.data_ptr(), save.data_ptr(), dt, ws.data_ptr(),
                                  ws.numel(), N.stream_of(x)), "se_bn_fwd")
        ctx.save_for_backward(x, weight, bias, act_param, save)
        ctx.cfg = (ps, int(training), act, int(per_channel), float(alpha))
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight, bias, act_param, save = ctx.saved_tensors
        ps, training, act, per_channel, alpha = ctx.cfg
        B, C, H, W = x.shape
        gy = gy.contiguous().to(x.dtype)
        dx = torch.empty((B, C, H, W), device=x.device, dtype=x.dtype)
        dw = torch.empty(C, device=x.device, dtype=x.dtype) if weight is not None else None
        db = torch.empty(C, device=x.device, dtype=x.dtype) if bias is not None else None
        da = torch.empty_like(act_param) if act_param is not None else None
        ws = torch.empty(int(N.lib().se_bn_workspace_size(B, C)), device=x.device, dtype=torch.uint8)
        N.check(N.lib().se_bn_bwd(gy.data_ptr(), x.data_ptr(), ps, B, C, H * W, N.ptr(weight), N.ptr(bias),
                                  save.data_ptr(), training, act, N.ptr(act_param), per_channel, alpha,
                                  dx.data_ptr(), N.ptr(dw), N.ptr(db), N.ptr(da), N.dtype_code(x), ws.data_ptr(),
                                  ws.numel(), N.stream_of(gy)), "se_bn_bwd")
        return dx, dw, db, da, None, None, None, None, None, None, None, None


def bn_act(norm: nn.Module, act: nn.Module, x: torch.Tensor) -> torch.Tensor:
    """act(norm(x)) for nn.BatchNorm2d / nn.Identity `norm` and nn.PReLU / nn.ELU /
    nn.Identity `act`, fused on the HIP kernels when norm is a BatchNorm2d."""
    if not isinstance(norm, nn.BatchNorm2d) or not x.is_cuda or x.dim() != 4:
        return act(norm(x))
    if isinstance(act, nn.PReLU):
        code, param, alpha = _ACT_PRELU, act.weight, 0.0
    elif isinstance(act, nn.ELU) and not act.inplace:
        code, param, alpha = _ACT_ELU, None, float(act.alpha)
    elif isinstance(act, nn.Identity):
        code, param, alpha = _ACT_NONE, None, 0.0
    else:
        return act(norm(x))
    use_batch = norm.training or not norm.track_running_stats
    if norm.momentum is None and norm.training and norm.track_running_stats:
        return act(norm(x))     # cumulative average: needs the step count on the host
    if not use_batch and norm.running_mean is None:
        return act(norm(x))
    track = norm.training and norm.track_running_stats
    rmean = norm.running_mean if (track or not use_batch) else None
    rvar = norm.running_var if (track or not use_batch) else None
    if x.dtype not in N.DTYPES or any(t is not None and t.dtype != x.dtype
                                      for t in (norm.weight, norm.bias, param, rmean, rvar)):
        return act(norm(x))     # mixed dtypes: the modules themselves
    if track:
        norm.num_batches_tracked.add_(1)
    return _BnAct.apply(x, norm.weight, norm.bias, param, rmean, rvar, use_batch, norm.momentum or 0.0, norm.eps,
                        code, param is not None and param.numel() > 1, alpha)


def _ln_forward(x, C, weight, bias, eps, keep):
    """(y, rows of x as the kernel read them, their distance, save) of one launch; save None unless `keep`."""
    x2, ld = (x, C) if x.is_contiguous() else glue.as_rows(x, C)
    rows = x.numel() // C
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    save = x.new_empty((2, rows), dtype=torch.float32) if keep else None
    if rows:
        wt = weight if weight is not None else bias if bias is not None else x
        N.launch(x.get_device(), "se_layer_norm_fwd", N.lib().se_layer_norm_fwd, x2.data_ptr(), ld, rows, C, N.ptr(weight),
                 N.ptr(bias), eps, y.data_ptr(), N.ptr(save), N.DTYPES[x.dtype], N.DTYPES[wt.dtype])
    return y, x2, ld, save


def _ln_backward(ctx, gy):
    x, weight, save = ctx.saved_tensors
    C, ldx, bdt = ctx.cfg
    need = ctx.needs_input_grad
    rows = x.numel() // C
    wdt = weight.dtype if weight is not None else bdt or x.dtype
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    new = x.new_empty if rows else x.new_zeros
    dw = new(C, dtype=wdt) if need[1] else None
    db = new(C, dtype=wdt) if need[2] else None
    if rows:
        g2, ldg = (gy, C) if gy.is_contiguous() and gy.dtype == x.dtype and not gy.is_neg() else glue.as_rows(gy, C, x.dtype)
        lib = N.lib()
        size = lib.se_layer_norm_workspace_size(rows, C) if need[1] or need[2] else 0
        ws = x.new_empty(size, dtype=torch.uint8) if size else None
        N.launch(x.get_device(), "se_layer_norm_bwd", lib.se_layer_norm_bwd, g2.data_ptr(), ldg, x.data_ptr(), ldx, rows, C,
                 N.ptr(weight), save.data_ptr(), N.ptr(dx), N.ptr(dw), N.ptr(db), N.DTYPES[x.dtype], N.DTYPES[wdt], N.ptr(ws),
                 size)
    return dx, dw, db, None, None


_ln_backward_once = once_differentiable(_ln_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, C, eps):
        y, x2, ld, save = _ln_forward(x, C, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, save)
        ctx.cfg = (C, ld, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, gy):   # with create_graph, a result that refuses to be differentiated again
        return _ln_backward_once(ctx, gy) if torch.is_grad_enabled() else _ln_backward(ctx, gy)


def layer_norm(norm: nn.LayerNorm, x: torch.Tensor) -> torch.Tensor:
    """norm(x) on the HIP kernels: x [..., *norm.normalized_shape] on the GPU in fp32, bf16 or fp16; norm's weight
    and bias (each may be absent) both in x's type or both in fp32. The result is contiguous, in x's type. A second
    derivative and one in forward mode are refused."""
    shape, w, b = norm.normalized_shape, norm.weight, norm.bias
    k = len(shape)
    if x.shape[-k:] != shape:
        raise RuntimeError(f"sehip layer_norm: input {tuple(x.shape)} does not end in {tuple(shape)}")
    dev, dt = x.get_device(), x.dtype
    if dev < 0 or (w is not None and w.get_device() != dev) or (b is not None and b.get_device() != dev):
        raise RuntimeError("sehip layer_norm: x, weight and bias must be on one GPU (there is no CPU fallback)")
    if dt not in N.DTYPES:
        raise RuntimeError(f"sehip layer_norm: unsupported storage type {dt} (fp32, bf16, fp16)")
    wdt = dt if w is None and b is None else w.dtype if w is not None else b.dtype
    if (wdt != dt and wdt != torch.float32) or (b is not None and b.dtype != wdt):
        raise RuntimeError(f"sehip layer_norm: weight and bias {wdt}, {None if b is None else b.dtype} beside a {dt} input (both "
                           "in its type or both in fp32)")
    if not ((w is None or w.is_contiguous()) and (b is None or b.is_contiguous())):
        raise RuntimeError("sehip layer_norm: weight and bias must be contiguous")
    if x.is_neg() or (w is not None and w.is_neg()) or (b is not None and b.is_neg()):
        x, w, b = (t if t is None else t.resolve_neg() for t in (x, w, b))
    C = shape[0] if k == 1 else math.prod(shape)
    if not 0 < C <= N.INT_MAX:
        raise RuntimeError("sehip layer_norm: normalised over " + ("no elements" if C == 0 else f"{C} elements: behind 32-bit indexes"))
    if k == 1:
        return _layer_norm(x, w, b, C, norm.eps)
    # the normalised axes as one (views of w and b, so that their gradients come back in their own shapes)
    return _layer_norm(x.flatten(x.dim() - k), w if w is None else w.view(C), b if b is None else b.view(C), C,
                       norm.eps).view(x.shape)


def _layer_norm(x, w, b, C, eps):
    if (torch.is_grad_enabled() and (x.requires_grad or (w is not None and w.requires_grad)
                                     or (b is not None and b.requires_grad))) or N.followed():
        return _LayerNorm.apply(x, w, b, C, eps)
    return _ln_forward(x, C, w, b, eps, False)[0]
