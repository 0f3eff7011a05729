"""Gated linear layer act(x Wg^T) * (x Wu^T) (csrc/gated.hip), the widening half of a gated
feed-forward block. GPU tensors run the native kernels; CPU tensors (and reference mode) take the
PyTorch path below."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .. import _native
from .functional import ACT, _C, _ref, _ref_act

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_WIDTH = 1 << 19


def gated_linear(x, w_gate, w_up, act="swish", dim=None):
    """``act(x @ w_gate.T) * (x @ w_up.T)`` with ``w_gate``, ``w_up`` [hidden, width].

    ``x`` is [..., width]; with four dimensions it is taken for an NCHW-shaped feature map [N, width, H,
    W], whose pixels are the rows. ``dim`` says which: -1 rows of any shape ([batch, heads, tokens,
    width]), 1 a feature map. It has to where dimensions 1 and 3 are both as long as the width. The result
    has ``hidden`` in the place of ``width``. ``act``: "swish" ("silu"), "sigmoid",
    "relu" or None. fp32, bf16 and fp16 rows; the weights have the rows' type, or are fp32 masters,
    which are rounded to it and whose gradients are fp32. Sums are fp32; in 16 bits the gradients of
    the projections are rounded once to the rows' type, the operand of the products that follow (small
    layers keep them in two parts). In fp16 what overflows there is an infinity.

    Differentiable once, in reverse mode. Forward and backward can be captured, together or apart. As with
    every autograd function, no eager graph of the same leaves may be alive while a backward is captured.
    """
    if act not in ACT:
        raise ValueError(f"act must be one of {sorted(a for a in ACT if a)} or None, got {act!r}")
    if dim not in (None, 1, -1):
        raise ValueError(f"dim must be 1 (a feature map), -1 (rows) or None, got {dim!r}")
    if dim == 1 and x.dim() != 4:
        raise ValueError(f"dim=1 is that of a feature map [N, width, H, W], x is {tuple(x.shape)}")
    if x.dim() == 4 and dim != -1:
        if w_gate.dim() == 2 and dim is None and x.shape[3] == w_gate.shape[1]:
            raise ValueError(f"x {tuple(x.shape)} ends with the weights' width {x.shape[3]}"
                             + (", and dimension 1 is as long: dim must be 1 or -1" if x.shape[1] == x.shape[3]
                                else ", but four dimensions are a feature map unless dim=-1"))
        y = gated_linear(x.permute(0, 2, 3, 1).unsqueeze(0), w_gate, w_up, act)[0]
        return y.permute(0, 3, 1, 2)
    if not _ref(x):
        return _C().gated_linear(x, w_gate, w_up, ACT[act], _native._debug)
    if x.dtype not in _FLOATS:
        raise TypeError(f"x must be fp32, bf16 or fp16, got {x.dtype}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape != w_up.shape:
        raise ValueError(f"weights must be two [hidden, width] matrices, got {tuple(w_gate.shape)} "
                         f"and {tuple(w_up.shape)}")
    width, hidden = w_gate.shape[1], w_gate.shape[0]
    if x.shape[-1] != width:
        raise ValueError(f"x {tuple(x.shape)} has {x.shape[-1]} features, the weights {width}")
    if not (1 <= width <= MAX_WIDTH and 1 <= hidden <= MAX_WIDTH):
        raise ValueError(f"width and hidden must be 1 to {MAX_WIDTH}")
    if w_gate.dtype != w_up.dtype or w_gate.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"weights must both be {x.dtype} or fp32, got {w_gate.dtype}, {w_up.dtype}")
    if w_gate.device != x.device or w_up.device != x.device:
        raise ValueError(f"weights are on {w_gate.device} and {w_up.device}, x is on {x.device}")
    g, u = F.linear(x, w_gate.to(x.dtype)), F.linear(x, w_up.to(x.dtype))
    return (_ref_act(g.float(), act) * u.float()).to(x.dtype)
