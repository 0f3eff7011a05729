"""Gated linear layer act(x Wg^T) * (x Wu^T) (csrc/gated.hip), the widening half of a gated
feed-forward block. GPU tensors run the native kernels; CPU tensors (and reference mode) take the
PyTorch path below."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .functional import ACT, _C, _ref, _ref_act

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_WIDTH = 1 << 19


def _rows(x):
    r = x.reshape(-1, x.shape[-1])
    if (r.shape[1] > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < 0):
        r = r.contiguous()
    return r


class _GatedLinear(torch.autograd.Function):
    """The projections are kept in fp32 for the backward (8 bytes a hidden unit and row): computing
    them again would cost two of the forward's products, and 16-bit copies would add their rounding
    to every gradient."""

    @staticmethod
    def forward(ctx, x, wg, wu, act):
        C = _C()
        ops = C.gated_operand(x, x), C.gated_operand(wg, x), C.gated_operand(wu, x)
        h, g, u = C.gated_fwd(*ops, act, True)
        ctx.save_for_backward(g, u, *ops)
        ctx.cfg = (x.shape[1], act, wg.dtype == torch.float32)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        g, u, *ops = ctx.saved_tensors
        width, act, dw_f32 = ctx.cfg
        need_dx = ctx.needs_input_grad[0]
        need_dw = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dwg, dwu = _C().gated_bwd(_rows(dh), *ops, g, u, width, act, need_dx, need_dw, dw_f32)
        return dx, dwg, dwu, None


def gated_linear(x, w_gate, w_up, act="swish"):
    """``act(x @ w_gate.T) * (x @ w_up.T)`` with ``w_gate``, ``w_up`` [hidden, width].

    ``x`` is [..., width], or an NCHW-shaped feature map [N, width, H, W], whose pixels are the rows;
    the result has ``hidden`` in the place of ``width``. ``act``: "swish" ("silu"), "sigmoid",
    "relu" or None. fp32, bf16 and fp16 rows; the weights have the rows' type, or are fp32 masters,
    which are rounded to it and whose gradients are fp32. Sums are fp32; in 16 bits the gradients of
    the projections are rounded once to the rows' type, the operand of the products that follow.
    """
    if act not in ACT:
        raise ValueError(f"act must be one of {sorted(a for a in ACT if a)} or None, got {act!r}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"x must be fp32, bf16 or fp16, got {x.dtype}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape != w_up.shape:
        raise ValueError(f"weights must be two [hidden, width] matrices, got {tuple(w_gate.shape)} "
                         f"and {tuple(w_up.shape)}")
    width, hidden = w_gate.shape[1], w_gate.shape[0]
    axis = 1 if x.dim() == 4 else -1
    if x.shape[axis] != width:
        raise ValueError(f"x {tuple(x.shape)} has {x.shape[axis]} features, the weights {width}")
    if not (1 <= width <= MAX_WIDTH and 1 <= hidden <= MAX_WIDTH):
        raise ValueError(f"width and hidden must be 1 to {MAX_WIDTH}")
    if w_gate.dtype != w_up.dtype or w_gate.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"weights must both be {x.dtype} or fp32, got {w_gate.dtype}, {w_up.dtype}")
    if w_gate.device != x.device or w_up.device != x.device:
        raise ValueError(f"weights are on {w_gate.device} and {w_up.device}, x is on {x.device}")
    if x.dim() == 4:
        y = gated_linear(x.permute(0, 2, 3, 1).unsqueeze(0), w_gate, w_up, act)[0]
        return y.permute(0, 3, 1, 2)
    if _ref(x):
        g, u = F.linear(x, w_gate.to(x.dtype)), F.linear(x, w_up.to(x.dtype))
        return (_ref_act(g.float(), act) * u.float()).to(x.dtype)
    lead = x.shape[:-1]
    z = _rows(x)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        h = _GatedLinear.apply(z, w_gate, w_up, ACT[act])
    else:
        C = _C()
        h, _, _ = C.gated_fwd(C.gated_operand(z, z), C.gated_operand(w_gate, z),
                              C.gated_operand(w_up, z), ACT[act], False)
    return h.view(*lead, hidden)
