"""The norms after and before a residual block, with its gate and residual
scale, as one op: where one block ends and the next begins.

Beside bn_act (bn.py), which does the same for convolution blocks: there the
norm is over the batch, here over the last dimension (RMSNorm, LayerNorm).
GPU path: ops/hip/norm_residual.hip, with its autograd node in bindings.cpp
(a node in Python took some 25 us more of host time a call, as much as the
kernels of a batch of 256 rows).  The reference has batch norms only.
"""

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn

from . import ext, use_hip

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {None: 0, "sigmoid": 1, "silu": 2}

Norm = Union[nn.RMSNorm, nn.LayerNorm]


def _norm_args(mod: Optional[Norm], width: int, which: str):
    """(kind, weight, bias, eps) of a norm module."""
    if mod is None:
        return 0, None, None, 0.0
    if isinstance(mod, nn.RMSNorm):
        kind, bias, base = 1, None, nn.RMSNorm
    elif isinstance(mod, nn.LayerNorm):
        kind, bias, base = 2, mod.bias, nn.LayerNorm
    else:
        raise TypeError(f"{which} must be an nn.RMSNorm or nn.LayerNorm, got "
                        f"{type(mod).__name__}")
    # the formula is what the module itself would compute, and all it does
    own = mod.__dict__
    if "forward" in own or (type(mod) is not base and (
            type(mod).forward is not base.forward or
            type(mod).__call__ is not base.__call__)):
        raise TypeError(f"{which}'s forward pass is not {base.__name__}'s: "
                        f"{type(mod).__name__}")
    if own["_forward_hooks"] or own["_forward_pre_hooks"] or \
            own["_backward_hooks"] or own["_backward_pre_hooks"]:
        raise TypeError(f"{which} has hooks, which would not be called")
    if mod.normalized_shape != (width,):
        raise ValueError(f"{which} normalizes {mod.normalized_shape}, the "
                         f"last dimension is {width}")
    if mod.eps is None or not mod.eps >= 0.0:
        raise ValueError(f"{which} needs an eps of its own, got {mod.eps}")
    return kind, mod.weight, bias, mod.eps


def _check_tensors(x, branch, gate, vectors, block_type):
    """What the GPU's entry point checks by itself."""
    width = x.shape[-1]
    if block_type not in _TYPES and block_type != torch.float64:
        raise TypeError(f"the block's type must be a float type, got "
                        f"{block_type}")
    if branch is not None and branch.shape != x.shape:
        raise ValueError(f"branch is {tuple(branch.shape)}, x "
                         f"{tuple(x.shape)}")
    if x.dtype not in (torch.float32, block_type):
        raise TypeError(f"x must be float32 or of the block's type, got "
                        f"{x.dtype} with {block_type}")
    if gate is not None:
        if gate.dim() != x.dim() or gate.shape[:-1] != x.shape[:-1] or \
                gate.shape[-1] not in (1, width):
            raise ValueError(f"gate must be {tuple(x.shape)} or have 1 as "
                             f"its last dimension, got {tuple(gate.shape)}")
        if gate.dtype != block_type:
            raise TypeError(f"gate is {gate.dtype}, the branch {block_type}")
    for v in vectors:
        if v is None:
            continue
        if v.shape != (width,):
            raise ValueError(f"weights, biases and scale must be [{width}], "
                             f"got {tuple(v.shape)}")
        if v.dtype not in (torch.float32, block_type):
            raise TypeError("weights, biases and scale must be float32 or of "
                            f"the block's type, got {v.dtype}")
    if any(t is not None and t.device != x.device
           for t in (branch, gate, *vectors)):
        raise ValueError("all tensors must be on one device")


def _plain_norm(x, kind, weight, bias, eps):
    if kind == 0:
        return x
    if kind == 2:
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(y.dtype)
    return y if bias is None else y + bias.to(y.dtype)


def _plain(x, branch, gate, w1, b1, w2, b2, scale, scale_value, post, pre,
           act, eps1, eps2, out_dtype):
    """The same in elementary operations, in 32 bits (64 for float64)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    r = x.to(wide)
    if branch is not None:
        add = _plain_norm(branch.to(wide), post, w1, b1, eps1)
        if gate is not None:
            g = gate.to(wide)
            s = torch.sigmoid(g)
            add = add * (g if act == 0 else s if act == 1 else g * s)
        r = r + add * (scale_value if scale is None else scale.to(wide))
    y = _plain_norm(r, pre, w2, b2, eps2).to(out_dtype) if pre else None
    return r.to(x.dtype), y


def norm_residual(x: torch.Tensor, branch: Optional[torch.Tensor] = None, *,
                  post: Optional[Norm] = None, pre: Optional[Norm] = None,
                  gate: Optional[torch.Tensor] = None,
                  gate_act: Optional[str] = None,
                  scale: Union[None, float, torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``r = x + scale * act(gate) * post(branch);  y = pre(r)``.

    Ends one residual block and begins the next: `branch` is what a block put
    out, `post` the norm after it (sandwich norms), `pre` the norm before the
    next block.  Returns (r, y): the residual stream and the next block's
    input; y is None without `pre`.  Without `branch` (the first block) r is
    x and only y is computed.

    x: [..., width], the residual stream; float32, or of the branch's type.
    branch: x's shape; float32, bfloat16 or float16, and the type of y.
    post, pre: nn.RMSNorm or nn.LayerNorm over the last dimension, with or
        without weight and bias; None for no norm.  Only the formula is
        computed and the module not called: one with hooks or with a forward
        pass of its own is refused.
    gate: the branch's shape, or [..., 1] for one gate per token, of the
        branch's type; gate_act: None, "sigmoid" or "silu".
    scale: a number, or a tensor [width] (or of one element).  Weights,
        biases and scale are float32 or of the branch's type.
    out_dtype: type of y where there is no branch (x's by default).

    Everything is computed in 32 bits from the inputs: y is the norm of r
    before r is rounded to x's type.  Gradients flow to every tensor; x,
    branch and gate may be strided (halves of one projection) as long as the
    last dimension is dense, other layouts are copied.  On the GPU width is
    16384 at most, and only first derivatives of the backward kind are there:
    second ones, forward-mode tangents, torch.func, torch.jit.trace, make_fx
    and fake tensors are errors.
    """
    width = x.shape[-1] if x.dim() else 0
    if width < 1:
        raise ValueError(f"x must be [..., width], got {tuple(x.shape)}")
    post_kind, w1, b1, eps1 = _norm_args(post, width, "post")
    pre_kind, w2, b2, eps2 = _norm_args(pre, width, "pre")
    act = _ACTS.get(gate_act)
    if act is None:
        raise ValueError(f"gate_act must be None, 'sigmoid' or 'silu', got "
                         f"{gate_act!r}")
    if gate is None and act:
        raise ValueError("gate_act needs a gate")
    if branch is None:
        if post is not None or gate is not None or scale is not None:
            raise ValueError("post, gate and scale need a branch")
        if pre is None:
            raise ValueError("neither a branch nor a norm is given")
        block_type = out_dtype or x.dtype
    else:
        block_type = branch.dtype
        if out_dtype is not None and out_dtype != block_type:
            raise ValueError("y has the branch's type: out_dtype is for calls "
                             "without one")
    scale_value = 1.0
    if isinstance(scale, torch.Tensor):
        if scale.numel() == 1 and scale.shape != (width,):
            scale = scale.reshape(1).expand(width)
    elif scale is not None:
        scale, scale_value = None, float(scale)
    if x.is_cuda and use_hip(x):  # shapes, types, devices: checked in C++
        kind = _TYPES.get(block_type)
        if kind is None:
            raise TypeError(f"on the GPU the block's type is float32, "
                            f"bfloat16 or float16, got {block_type}")
        r, y = ext().norm_residual(x, branch, gate, w1, b1, w2, b2, scale,
                                   scale_value, post_kind, pre_kind, act,
                                   eps1, eps2, kind)
    else:
        _check_tensors(x, branch, gate, (w1, b1, w2, b2, scale), block_type)
        r, y = _plain(x, branch, gate, w1, b1, w2, b2, scale, scale_value,
                      post_kind, pre_kind, act, eps1, eps2, block_type)
    return (x if branch is None else r), y
