"""Norms before and after a block, fused with its gate and residual scale, forward and backward, over the C ABI:

    u = N1(branch);  s = residual_scale * residual + branch_scale * gate * u;  o = N2(s)

N1 and N2 are "none", "layer" (LayerNorm) or "rms" (root-mean-square norm).  One call covers what stands between two blocks of
a residual network: the post-norm layer of BERT (out_norm="layer"), the pre-norm block of Swin (the sum, and the norm in
front of the next branch), a norm on the branch, a learned scale per channel or a gate per sample, a scaled residual.  The
reference has the LayerNorm stages of its fused layer only (cpp/bert/kernels/fused_sqq_bert.cu:3690-3782).
"""
from __future__ import annotations

from typing import Dict, Optional, Tuple, Union

import torch

from . import _lib

_NORMS = {"none": 0, "layer": 1, "rms": 2}


def _vector(t: Optional[torch.Tensor], name: str, cols: int, dtype, device: int):
    """(address, dtype) of an optional [cols] vector; `dtype`: what the vectors before it had."""
    if t is None:
        return 0, dtype
    if t.get_device() != device or not t.is_contiguous() or t.shape != (cols,):
        raise ValueError(f"{name} must be a contiguous CUDA tensor of {cols} values on the same device")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"gate, weights and biases must share one type: {name} has {t.dtype}, others {dtype}")
    return t.data_ptr(), t.dtype


def _matrix(t: Optional[torch.Tensor], name: str, rows: int, cols: int, like: torch.Tensor):
    """(address, stride) of an optional matrix of the branch's shape."""
    if t is None:
        return 0, 0
    if t.dtype != like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name} must have the branch's type and device")
    if t.shape != like.shape:
        raise ValueError(f"{name} must have the branch's shape")
    return t.data_ptr(), _lib.rows_of(t, name)[2]


def _front(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias, residual_scale, branch_scale,
           branch_eps, out_eps):
    """The checked head of a call record: (its first values without the outputs' strides, its input pointers, rows, columns, type of the
    vectors, gate rows)."""
    code = _lib.DTYPE_CODES.get(branch.dtype)
    if not branch.is_cuda or code is None:
        raise ValueError("branch must be a float32, float16 or bfloat16 CUDA tensor")
    if branch_norm not in _NORMS or out_norm not in _NORMS:
        raise ValueError(f"norms are {', '.join(_NORMS)}: got {branch_norm}, {out_norm}")
    rows, cols, ystride = _lib.rows_of(branch, "branch")
    r, rstride = _matrix(residual, "residual", rows, cols, branch)
    dev, dtype, g, gate_rows = branch.get_device(), None, 0, 0
    if gate is not None:
        if gate.get_device() != dev or not gate.is_contiguous() or gate.dim() not in (1, 2) or gate.shape[-1] != cols:
            raise ValueError(f"gate must be a contiguous CUDA tensor [{cols}] or [gates, {cols}] on the branch's device")
        g, dtype, gate_rows = gate.data_ptr(), gate.dtype, gate.shape[0] if gate.dim() == 2 else 1
        if not gate_rows or rows % gate_rows:
            raise ValueError(f"gate has {gate_rows} rows, which do not divide {rows}")
    w1, dtype = _vector(branch_weight, "branch_weight", cols, dtype, dev)
    b1, dtype = _vector(branch_bias, "branch_bias", cols, dtype, dev)
    w2, dtype = _vector(out_weight, "out_weight", cols, dtype, dev)
    b2, dtype = _vector(out_bias, "out_bias", cols, dtype, dev)
    pcode = code if dtype is None else _lib.DTYPE_CODES.get(dtype, -1)
    head = (rows, cols, code, pcode, _NORMS[branch_norm], _NORMS[out_norm], gate_rows, residual_scale, branch_scale, branch_eps, out_eps, 0,
            rstride, ystride)
    return head, (r, branch.data_ptr(), g, w1, b1, w2, b2), rows, cols, dtype, gate_rows


def _forward(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias, residual_scale, branch_scale,
             branch_eps, out_eps, keep_sum, quantize):
    head, ptrs, rows, cols, _, _ = _front(residual, branch, branch_norm, branch_weight, branch_bias, gate, out_norm, out_weight, out_bias,
                                          residual_scale, branch_scale, branch_eps, out_eps)
    lib = _lib.load()
    stream = _lib.stream_on(branch.get_device())
    shape = branch.shape
    total = out = q = scale = None
    if keep_sum:
        total = torch.empty(shape, dtype=branch.dtype, device=branch.device)
    if quantize:
        from .int8 import empty_rows
        q, scale = empty_rows(rows, cols, branch.device)
    elif out_norm != "none":
        out = torch.empty(shape, dtype=branch.dtype, device=branch.device)
    elif not keep_sum:
        raise ValueError("nothing to compute: neither the sum nor a norm of it is asked for")
    _lib.check(lib.souffle_residual_norm_forward(_lib.ResidualNorm.pack(
        *head, cols, cols, q.stride(0) if q is not None else 0, *ptrs, total.data_ptr() if keep_sum else 0, out.data_ptr() if out is not None else 0,
        q.data_ptr() if q is not None else 0, scale.data_ptr() if q is not None else 0), stream))
    return total, (q, scale) if quantize else out


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
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (branch, residual, branch_weight, branch_bias, gate, out_weight,
                                                                                  out_bias)):
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
    ds, ds_stride = _matrix(grad_sum, "grad_sum", rows, cols, branch)
    do, do_stride = _matrix(grad_out, "grad_out", rows, cols, branch)
    lib = _lib.load()
    device = branch.device
    stream = _lib.stream_on(branch.get_device())
    dr = torch.empty(branch.shape, dtype=branch.dtype, device=device) if residual is not None else None
    dy = torch.empty(branch.shape, dtype=branch.dtype, device=device)
    # one allocation for the vectors' gradients: each begins on a multiple of 16 bytes where the vector path needs it
    names = [n for n, there in (("branch_weight", branch_weight is not None), ("branch_bias", branch_norm == "layer"),
                                ("out_weight", out_weight is not None), ("out_bias", out_norm == "layer")) if there]
    d: Dict[str, Optional[torch.Tensor]] = dict.fromkeys(("branch_weight", "branch_bias", "gate", "out_weight", "out_bias"))
    vectors = torch.empty(len(names), cols, dtype=dtype or branch.dtype, device=device)
    d.update(zip(names, vectors.unbind(0)))
    if gate is not None:
        d["gate"] = torch.empty_like(gate)
    ws = torch.empty(lib.souffle_residual_norm_backward_workspace_bytes(rows, cols, gate_rows), dtype=torch.uint8, device=device)
    ptr = lambda t: 0 if t is None else t.data_ptr()
    _lib.check(lib.souffle_residual_norm_backward(_lib.ResidualNormGrad.pack(
        *head, 0, 0, 0, *ptrs, 0, 0, 0, 0, ds_stride, do_stride, cols, cols, ds, do, ptr(dr), dy.data_ptr(), ptr(d["gate"]), ptr(d["branch_weight"]),
        ptr(d["branch_bias"]), ptr(d["out_weight"]), ptr(d["out_bias"]), ws.data_ptr(), ws.numel()), stream))
    d["residual"], d["branch"] = dr, dy
    return d


def status() -> None:
    """Synchronises the current stream and raises SouffleError if a device-side wait of one of these calls has expired."""
    _lib.check(_lib.load().souffle_residual_norm_status(_lib.stream_ptr()))
