"""Norms before and after a block, fused with its gate and residual scale, forward and backward, over the C ABI:

    u = N1(branch);  s = residual_scale * residual + branch_scale * gate * u;  o = N2(s)

N1 and N2 are "none", "layer" (LayerNorm) or "rms" (root-mean-square norm).  One call covers what stands between two blocks of
a residual network: the post-norm layer of BERT (out_norm="layer"), the pre-norm block of Swin (the sum, and the norm in
front of the next branch), a norm on the branch, a learned scale per channel or a gate per sample, a scaled residual.  The
reference has the LayerNorm stages of its fused layer only (cpp/bert/kernels/fused_sqq_bert.cu:3690-3782).
"""
from __future__ import annotations

import functools
from typing import Dict, Optional, Tuple, Union

import torch

from . import _lib

_NORMS = {"none": 0, "layer": 1, "rms": 2}
_VECTORS = ("branch_weight", "branch_bias", "out_weight", "out_bias")
_CODES, _rows_of, _pack, _pack_grad = _lib.DTYPE_CODES, _lib.rows_of, _lib.ResidualNorm.pack, _lib.ResidualNormGrad.pack


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows: int, cols: int, gate_rows: int) -> int:
    return _lib.load().souffle_residual_norm_backward_workspace_bytes(rows, cols, gate_rows)


def _vector(t: torch.Tensor, name: str, cols: int, device: int) -> int:
    """Address of a [cols] vector."""
    if t.get_device() != device or not t.is_contiguous() or t.shape != (cols,):
        raise ValueError(f"{name} must be a contiguous CUDA tensor of {cols} values on the same device")
    return t.data_ptr()


def _matrix(t: torch.Tensor, name: str, like: torch.Tensor, device: int):
    """(address, stride) of a matrix of the branch's shape."""
    if t.dtype != like.dtype or t.get_device() != device:
        raise ValueError(f"{name} must have the branch's type and device")
    if t.shape != like.shape:
        raise ValueError(f"{name} must have the branch's shape")
    return t.data_ptr(), _rows_of(t, name)[2]


def _front(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias, residual_scale, branch_scale,
           branch_eps, out_eps):
    """The checked head of a call record: (its first values without the outputs' strides, its input pointers, rows, columns, type of the
    vectors, gate rows)."""
    dtype, dev = branch.dtype, branch.get_device()
    code = _CODES.get(dtype)
    if dev < 0 or code is None:
        raise ValueError("branch must be a float32, float16 or bfloat16 CUDA tensor")
    n1, n2 = _NORMS.get(branch_norm), _NORMS.get(out_norm)
    if n1 is None or n2 is None:
        raise ValueError(f"norms are {', '.join(_NORMS)}: got {branch_norm}, {out_norm}")
    rows, cols, ystride = _rows_of(branch, "branch")
    r = rstride = g = gate_rows = w1 = b1 = w2 = b2 = 0
    params = None
    if residual is not None:
        r, rstride = _matrix(residual, "residual", branch, dev)
    if gate is not None:
        shape = gate.shape
        if gate.get_device() != dev or not gate.is_contiguous() or len(shape) not in (1, 2) or shape[-1] != cols:
            raise ValueError(f"gate must be a contiguous CUDA tensor [{cols}] or [gates, {cols}] on the branch's device")
        g, params, gate_rows = gate.data_ptr(), gate.dtype, shape[0] if len(shape) == 2 else 1
        if not gate_rows or rows % gate_rows:
            raise ValueError(f"gate has {gate_rows} rows, which do not divide {rows}")
    if branch_weight is not None:
        w1 = _vector(branch_weight, "branch_weight", cols, dev)
        params = _same(branch_weight, "branch_weight", params)
    if branch_bias is not None:
        b1 = _vector(branch_bias, "branch_bias", cols, dev)
        params = _same(branch_bias, "branch_bias", params)
    if out_weight is not None:
        w2 = _vector(out_weight, "out_weight", cols, dev)
        params = _same(out_weight, "out_weight", params)
    if out_bias is not None:
        b2 = _vector(out_bias, "out_bias", cols, dev)
        params = _same(out_bias, "out_bias", params)
    head = (rows, cols, code, code if params is None else _CODES.get(params, -1), n1, n2, gate_rows, residual_scale, branch_scale, branch_eps,
            out_eps, 0, rstride, ystride)
    return head, (r, branch.data_ptr(), g, w1, b1, w2, b2), rows, cols, params, gate_rows


def _same(t: torch.Tensor, name: str, dtype):
    """The one type of gate, weights and biases; `dtype`: what those before had."""
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"gate, weights and biases must share one type: {name} has {t.dtype}, others {dtype}")
    return t.dtype


def _forward(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias, residual_scale, branch_scale,
             branch_eps, out_eps, keep_sum, quantize):
    head, ptrs, rows, cols, _, _ = _front(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias,
                                          residual_scale, branch_scale, branch_eps, out_eps)
    stream = _lib.stream_on(branch.get_device())
    shape, dtype, device = branch.shape, branch.dtype, branch.device
    total = out = None
    s_ptr = o_ptr = q_ptr = scale_ptr = q_stride = 0
    if keep_sum:
        total = torch.empty(shape, dtype=dtype, device=device)
        s_ptr = total.data_ptr()
    if quantize:
        from .int8 import empty_rows
        out = q, scale = empty_rows(rows, cols, device)
        q_ptr, q_stride, scale_ptr = q.data_ptr(), (cols + 15) // 16 * 16, scale.data_ptr()
    elif out_norm != "none":
        out = torch.empty(shape, dtype=dtype, device=device)
        o_ptr = out.data_ptr()
    elif not keep_sum:
        raise ValueError("nothing to compute: neither the sum nor a norm of it is asked for")
    rc = _lib.load().souffle_residual_norm_forward(_pack(*head, cols, cols, q_stride, *ptrs, s_ptr, o_ptr, q_ptr, scale_ptr), stream)
    if rc:
        _lib.check(rc)
    return total, out


class _Differentiable(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, branch_weight, branch_bias, gate, out_weight, out_bias, branch_norm, out_norm, residual_scale, branch_scale,
                branch_eps, out_eps):
        ctx.save_for_backward(residual, branch, branch_weight, branch_bias, gate, out_weight)
        ctx.rest = dict(branch_norm=branch_norm, out_norm=out_norm, residual_scale=residual_scale, branch_scale=branch_scale,
                        branch_eps=branch_eps, out_eps=out_eps)
        ctx.set_materialize_grads(False)
        return _forward(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias, residual_scale,
                        branch_scale, branch_eps, out_eps, True, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_sum, grad_out):
        residual, branch, branch_weight, branch_bias, gate, out_weight = ctx.saved_tensors
        if ctx.rest["out_norm"] == "none":
            grad_out = None
            if grad_sum is None:
                grad_sum = torch.zeros_like(branch)
        elif grad_out is None:
            grad_out = torch.zeros_like(branch)
        contiguous = lambda t: t if t is None else t.contiguous()
        d = residual_norm_backward(contiguous(grad_sum), contiguous(grad_out), residual, branch, branch_weight=branch_weight,
                                   branch_bias=branch_bias, gate=gate, out_weight=out_weight, **ctx.rest)
        want = ctx.needs_input_grad
        names = ("residual", "branch", "branch_weight", "branch_bias", "gate", "out_weight", "out_bias")
        return tuple(d[n] if want[i] else None for i, n in enumerate(names)) + (None,) * 6


def residual_norm(residual: Optional[torch.Tensor], branch: torch.Tensor, *, branch_norm: str = "none",
                  branch_weight: Optional[torch.Tensor] = None, branch_bias: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, out_norm: str = "none", out_weight: Optional[torch.Tensor] = None,
                  out_bias: Optional[torch.Tensor] = None, residual_scale: float = 1.0, branch_scale: float = 1.0, branch_eps: float = 1e-5,
                  out_eps: float = 1e-5, keep_sum: bool = True, quantize: bool = False
                  ) -> Tuple[Optional[torch.Tensor], Union[None, torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]]:
    """(s, o) of the formula above.  residual (may be None: no such term) and branch: [..., cols] of one shape and type (float32,
    float16, bfloat16), cols <= 8192, contiguous or 2-D with rows apart.  gate: [cols], or [gates, cols] where each gate
    serves rows / gates consecutive rows.  Weights, biases and gate are all of the branch's type or all float32.
    o is None without out_norm; with `quantize` it is (int8 rows, scales) for int8.int8_linear.  `keep_sum=False` leaves s out (None).
    Asynchronous.  Differentiable (not with quantize or without the sum) in all tensors."""
    if torch.is_grad_enabled() and (branch.requires_grad or (residual is not None and residual.requires_grad)
                                    or (branch_weight is not None and branch_weight.requires_grad)
                                    or (branch_bias is not None and branch_bias.requires_grad) or (gate is not None and gate.requires_grad)
                                    or (out_weight is not None and out_weight.requires_grad)
                                    or (out_bias is not None and out_bias.requires_grad)):
        if quantize or not keep_sum:
            raise ValueError("quantize and keep_sum=False have no gradient")
        return _Differentiable.apply(residual, branch, branch_weight, branch_bias, gate, out_weight, out_bias, branch_norm, out_norm,
                                     residual_scale, branch_scale, branch_eps, out_eps)
    return _forward(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias, residual_scale, branch_scale,
                    branch_eps, out_eps, keep_sum, quantize)


def residual_norm_backward(grad_sum: Optional[torch.Tensor], grad_out: Optional[torch.Tensor], residual: Optional[torch.Tensor],
                           branch: torch.Tensor, *, branch_norm: str = "none", branch_weight: Optional[torch.Tensor] = None,
                           branch_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, out_norm: str = "none",
                           out_weight: Optional[torch.Tensor] = None, residual_scale: float = 1.0, branch_scale: float = 1.0,
                           branch_eps: float = 1e-5, out_eps: float = 1e-5) -> Dict[str, Optional[torch.Tensor]]:
    """Gradients of residual_norm's inputs under its parameters' names, for the gradients of s (None: zero) and o (None without
    out_norm).  Vectors' and gates' gradients are summed in fp32 in a fixed order and have the vectors' type; a bias's is
    returned for every LayerNorm.  Entries for what is not there are None."""
    head, ptrs, rows, cols, dtype, gate_rows = _front(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, None,
                                                      residual_scale, branch_scale, branch_eps, out_eps)
    dev = branch.get_device()
    ds = ds_stride = do = do_stride = dr_ptr = gate_ptr = 0
    if grad_sum is not None:
        ds, ds_stride = _matrix(grad_sum, "grad_sum", branch, dev)
    if grad_out is not None:
        do, do_stride = _matrix(grad_out, "grad_out", branch, dev)
    stream = _lib.stream_on(dev)
    device, shape, kind = branch.device, branch.shape, branch.dtype
    d: Dict[str, Optional[torch.Tensor]] = dict.fromkeys(("branch_weight", "branch_bias", "gate", "out_weight", "out_bias", "residual"))
    dy = torch.empty(shape, dtype=kind, device=device)
    if residual is not None:
        d["residual"] = dr = torch.empty(shape, dtype=kind, device=device)
        dr_ptr = dr.data_ptr()
    # one allocation for the vectors' gradients
    names = [n for n, there in (("branch_weight", branch_weight is not None), ("branch_bias", branch_norm == "layer"),
                                ("out_weight", out_weight is not None), ("out_bias", out_norm == "layer")) if there]
    at = dict.fromkeys(_VECTORS, 0)
    if names:
        kind = dtype or kind
        vectors = torch.empty((len(names), cols), dtype=kind, device=device)
        base, step = vectors.data_ptr(), cols * kind.itemsize
        for i, (n, t) in enumerate(zip(names, vectors.unbind(0))):
            d[n], at[n] = t, base + i * step
    if gate is not None:
        d["gate"] = dg = torch.empty_like(gate)
        gate_ptr = dg.data_ptr()
    need = _workspace_bytes(rows, cols, gate_rows)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    rc = _lib.load().souffle_residual_norm_backward(_pack_grad(
        *head, 0, 0, 0, *ptrs, 0, 0, 0, 0, ds_stride, do_stride, cols, cols, ds, do, dr_ptr, dy.data_ptr(), gate_ptr, *at.values(), ws.data_ptr(), need),
        stream)
    if rc:
        _lib.check(rc)
    d["branch"] = dy
    return d


def status() -> None:
    """Synchronises the current stream and raises SouffleError if a device-side wait of one of these calls has expired."""
    _lib.check(_lib.load().souffle_residual_norm_status(_lib.stream_ptr()))
