"""Group norm with an activation, channels last.
(One family of `pytorch_geometric_temporal_amd.ops`; the package re-exports every name and forwards writes to its switches.)
"""
import torch

from .. import _lib
from .._lib import check_tensor, ptr, stream_of

F32 = torch.float32

from ._core import KERNEL_TIMER, _timed
from .delta import DTYPES

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2}


class GroupNormActFunction(torch.autograd.Function):
    """pgt_group_norm_act / pgt_group_norm_act_bwd on x [B, rows, C] contiguous."""

    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps, act):
        lib = _lib.get_lib()
        B, S, C = x.shape
        t = DTYPES[x.dtype]
        y = torch.empty_like(x)
        stats = torch.empty(B, groups, 2, dtype=F32, device=x.device) if S > 1 or C // groups > 512 else None
        n = int(lib._pgt_group_norm_ws_floats(B, S, C, groups, t, 0))
        ws = torch.empty(n, dtype=F32, device=x.device) if n > 0 else None
        _timed("group_norm", 2.0 * x.numel() * x.element_size() if KERNEL_TIMER else 0, lambda: lib.call(
            "pgt_group_norm_act", ptr(x), B, S, C, groups, t, ptr(weight), ptr(bias), eps, act, ptr(y), ptr(stats), ptr(ws), n,
            stream_of(lib, x)))
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.args = (groups, eps, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = _lib.get_lib()
        x, weight, bias, stats = ctx.saved_tensors
        groups, eps, act = ctx.args
        B, S, C = x.shape
        t = DTYPES[x.dtype]
        dy = dy.contiguous()
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dw = torch.empty(C, dtype=F32, device=x.device) if weight is not None and ctx.needs_input_grad[2] else None
        db = torch.empty(C, dtype=F32, device=x.device) if bias is not None and ctx.needs_input_grad[3] else None
        n = int(lib._pgt_group_norm_ws_floats(B, S, C, groups, t, 1))
        ws = torch.empty(n, dtype=F32, device=x.device) if n > 0 else None
        _timed("group_norm_bwd", 3.0 * x.numel() * x.element_size() if KERNEL_TIMER else 0, lambda: lib.call(
            "pgt_group_norm_act_bwd", ptr(x), ptr(dy), ptr(stats), B, S, C, groups, t, ptr(weight), ptr(bias), eps, act, ptr(dx), ptr(dw),
            ptr(db), ptr(ws), n, stream_of(lib, x)))
        return dx, None, dw, db, None, None


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """act(group_norm(x)) with the channels last: x [B, .., C] float32, bfloat16 or float16; statistics per sample (first axis) and group
    of C / num_groups neighbouring channels over all axes between.  For x [rows, C] every row is a sample of its own: num_groups = heads
    is the per-head norm behind a layer with heads.  weight, bias [C] float32 or None; activation None, "relu" or "silu".
    Returns x's shape and type; differentiable (once) in x, weight and bias, statistics and sums in float32, bitwise reproducible."""
    lib = _lib.get_lib()
    what = "group_norm_act"
    if not isinstance(x, torch.Tensor) or x.dtype not in DTYPES:
        raise TypeError(f"{what}: x must be a float32, bfloat16 or float16 tensor, got {getattr(x, 'dtype', type(x))}")
    check_tensor(lib, x, f"{what}: x", x.dtype)
    if x.dim() < 2:
        raise ValueError(f"{what}: x must be [batch, .., channels], got {tuple(x.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None, 'relu' or 'silu', got {activation!r}")
    C, num_groups = x.size(-1), int(num_groups)
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"{what}: {C} channels do not divide into {num_groups} groups")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            check_tensor(lib, t, f"{what}: {name}")
            if tuple(t.shape) != (C,):
                raise ValueError(f"{what}: {name} must be [{C}], got {tuple(t.shape)}")
            if t.device != x.device:
                raise ValueError(f"{what}: {name} is on {t.device}, x on {x.device}")
    rows = 1
    for n in x.shape[1:-1]:
        rows *= n
    with torch.cuda.device_of(x):
        y = GroupNormActFunction.apply(x.contiguous().view(x.size(0), rows, C), num_groups,
                                       weight.contiguous() if weight is not None else None,
                                       bias.contiguous() if bias is not None else None, float(eps), ACTIVATIONS[activation])
    return y.view(x.shape)
