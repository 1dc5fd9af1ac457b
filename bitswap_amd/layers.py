"""The channels-last layer operators of bitswap_amd.hip with gradients, and the residual layer made of them.

    linear_act       s = x w^T + bias (+ res), y = act(s)       over rows of channels: a pointwise convolution with its epilogue
    group_norm_act   y = act(GN(x))                              on [n, ..., C]
    PointwiseResNetLayer   x + W2 act(W1 act(GN(x)) + b1) + b2   (Model(npoint=k) closes every conv stack with k of them)

On a HIP device they run the kernels of csrc/linear.hip, norm_act.hip and pack8.hip; on CPU tensors the same formulas in plain
torch, as the rest of the Model does there.  save8=True keeps the activations that the backward pass needs in 8 bits
(hip.Packed8: 1.03 bytes a value); the forward results do not change, the gradients are those at the saved values.  On CPU tensors
save8 changes nothing: activations are kept whole there.

First derivatives only.  A gradient of a parameter comes in the parameter's type.  To capture a training step into a graph take
its gradients with torch.autograd.grad inside the capture: `.backward()` accumulates into leaves through nodes that live as long
as any graph of the same leaves, on the stream that made them.
"""
import math

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from . import hip

ACTS = {"none": hip.ACT_NONE, "elu": hip.ACT_ELU, "silu": hip.ACT_SILU, "gelu": hip.ACT_GELU}
_PLAIN = {hip.ACT_NONE: lambda s: s, hip.ACT_ELU: F.elu, hip.ACT_SILU: F.silu, hip.ACT_GELU: F.gelu}


def _wide(dtype):
    """The type that 16-bit values are computed in."""
    return torch.float32 if dtype in (torch.bfloat16, torch.float16) else dtype


def _code(act):
    if act in ACTS:
        return ACTS[act]
    return hip._act_code(act)


def _keep(ctx, name, v, tensors):
    """Note where a saved activation (tensor, Packed8 or None) lies among the saved tensors."""
    if v is None:
        setattr(ctx, name, None)
    elif isinstance(v, hip.Packed8):
        setattr(ctx, name, (len(tensors), v.shape, v.dtype))
        tensors += [v.codes, v.exps]
    else:
        setattr(ctx, name, (len(tensors), None, None))
        tensors.append(v)


def _kept(ctx, name, tensors):
    at = getattr(ctx, name)
    if at is None:
        return None
    i, shape, dtype = at
    return tensors[i] if shape is None else hip.Packed8(tensors[i], tensors[i + 1], shape, dtype)


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, res, act, save8):
        none = act == hip.ACT_NONE
        s, y = hip.linear_act(x, w, bias, res, act=act, want_sum=True, want_act=not none)
        tensors = [w]
        _keep(ctx, "x", (hip.pack8(x) if save8 else x) if ctx.needs_input_grad[1] else None, tensors)
        _keep(ctx, "s", None if none else hip.pack8(s) if save8 else s, tensors)
        ctx.save_for_backward(*tensors)
        ctx.act, ctx.xshape, ctx.bdtype = act, x.shape, None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return s, (None if none else y)

    @staticmethod
    @once_differentiable
    def backward(ctx, gs, gy):
        if gs is None and gy is None:
            return (None,) * 6
        t = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        if not (nx or nw or nb or nr):
            return (None,) * 6
        dx, dw, db, dr = hip.linear_act_grad(_kept(ctx, "x", t), t[0], _kept(ctx, "s", t), act=ctx.act, g_sum=gs, g_act=gy, want_x=nx, want_w=nw,
                                             want_bias=nb, want_res=nr)
        return dx, dw, db.to(ctx.bdtype) if nb else None, dr, None, None


def linear_act(x, w, bias=None, res=None, act="elu", want_sum=False, save8=False):
    """act(x w^T + bias (+ res)), or (sum, act(sum)) with want_sum.  x [..., K], w [N, K], bias [N], res [..., N]."""
    act = _code(act)
    if not x.is_cuda:
        if w.dim() != 2 or w.dtype != x.dtype or x.shape[-1:] != w.shape[1:]:
            raise hip.BitswapHipError(f"linear_act: x [..., K] and w [N, K] of one type, got {tuple(x.shape)} {x.dtype} and {tuple(w.shape)} {w.dtype}")
        if bias is not None and (bias.shape != w.shape[:1] or bias.dtype not in (torch.float32, x.dtype)):
            raise hip.BitswapHipError(f"linear_act: bias must be [{w.shape[0]}] of float32 or {x.dtype}, got {tuple(bias.shape)} {bias.dtype}")
        if res is not None and (res.shape != (*x.shape[:-1], w.shape[0]) or res.dtype != x.dtype):
            raise hip.BitswapHipError(f"linear_act: res must be {(*x.shape[:-1], w.shape[0])} of {x.dtype}, got {tuple(res.shape)} {res.dtype}")
        wide = _wide(x.dtype)
        s = F.linear(x.to(wide), w.to(wide), None if bias is None else bias.to(wide))
        s = s if res is None else s + res.to(wide)
        s, y = s.to(x.dtype), _PLAIN[act](s).to(x.dtype)                # the activation sees s before its rounding
    elif torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias, res)):
        if act == hip.ACT_NONE:
            s = y = _LinearAct.apply(x, w, bias, res, act, save8)[0]
        else:
            s, y = _LinearAct.apply(x, w, bias, res, act, save8)
    else:
        s, y = hip.linear_act(x, w, bias, res, act=act, want_sum=want_sum)
    return (s, y) if want_sum else y


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, groups, eps, act, save8):
        y, stats, packed = hip.group_norm_act(x, groups, gamma, beta, eps=eps, act=act, want_stats=True, want_pack=save8)
        tensors = [stats]
        ctx.has = (gamma is not None, beta is not None)
        tensors += [v for v in (gamma, beta) if v is not None]
        _keep(ctx, "x", packed if save8 else x, tensors)
        ctx.save_for_backward(*tensors)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        t = ctx.saved_tensors
        gamma = t[1] if ctx.has[0] else None
        beta = t[1 + ctx.has[0]] if ctx.has[1] else None
        need = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dgamma, dbeta = hip.group_norm_act_grad(_kept(ctx, "x", t), t[0], ctx.groups, g, gamma, beta, act=ctx.act, want_affine=need)
        return (dx if ctx.needs_input_grad[0] else None, dgamma.to(gamma.dtype) if ctx.needs_input_grad[1] else None,
                dbeta.to(beta.dtype) if ctx.needs_input_grad[2] else None, None, None, None, None)


def group_norm_act(x, groups, gamma=None, beta=None, eps=1e-5, act="elu", save8=False):
    """act(group norm of x) on channels-last x [n, ..., C], statistics over the pixels and C / groups channels of a group."""
    act = _code(act)
    if not x.is_cuda:
        if x.dim() < 2 or x.shape[-1] < 1:
            raise hip.BitswapHipError(f"group_norm_act: expected [n, ..., C], got {tuple(x.shape)}")
        n, c = x.shape[0], x.shape[-1]
        pixels = math.prod(x.shape[1:-1])                  # (said, not -1: without images or pixels that is ambiguous)
        if groups < 1 or c % groups:
            raise hip.BitswapHipError(f"group_norm_act: {groups} groups do not divide {c} channels")
        if not eps >= 0:
            raise hip.BitswapHipError(f"group_norm_act: eps {eps}")
        given = [t for t in (gamma, beta) if t is not None]
        if any(t.shape != (c,) or t.dtype not in (torch.float32, x.dtype) or t.dtype != given[0].dtype for t in given):
            raise hip.BitswapHipError(f"group_norm_act: gamma and beta must be [{c}] of one type, float32 or {x.dtype}, got "
                                      f"{[(tuple(t.shape), t.dtype) for t in given]}")
        v = x.reshape(n, pixels, groups, c // groups).to(_wide(x.dtype))
        d = v - v.mean((1, 3), keepdim=True)
        u = (d / torch.sqrt(d.square().mean((1, 3), keepdim=True) + eps)).reshape(n, pixels, c)
        u = u if gamma is None else u * gamma
        u = u if beta is None else u + beta
        return _PLAIN[act](u).to(x.dtype).view(x.shape)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gamma, beta)):
        return _GroupNormAct.apply(x, gamma, beta, groups, eps, act, save8)
    return hip.group_norm_act(x, groups, gamma, beta, eps=eps, act=act)[0]


def groups_for(channels, most=32):
    """The largest number of groups up to `most` that divides the channels (256 -> 32, 252 -> 28, 61 -> 1)."""
    return max(g for g in range(1, min(most, channels) + 1) if channels % g == 0)


class PointwiseResNetLayer(nn.Module):
    """x + W2 act(W1 act(GN(x)) + b1) + b2 on channels-last x [n, ..., channels]: what ResNetLayer is to 3x3 convolutions, for 1x1.
    Starts close to the identity (W2 a tenth of W1's spread).  save8: see the module's text."""

    def __init__(self, channels, hidden=None, groups=None, act="elu", eps=1e-5, save8=False):
        super().__init__()
        hidden = hidden or channels
        self.groups, self.act, self.eps, self.save8 = groups or groups_for(channels), act, eps, save8
        self.gamma, self.beta = nn.Parameter(torch.ones(channels)), nn.Parameter(torch.zeros(channels))
        self.w1, self.b1 = nn.Parameter(torch.randn(hidden, channels) * channels ** -0.5), nn.Parameter(torch.zeros(hidden))
        self.w2, self.b2 = nn.Parameter(torch.randn(channels, hidden) * 0.1 * hidden ** -0.5), nn.Parameter(torch.zeros(channels))

    def forward(self, x):
        h = group_norm_act(x, self.groups, self.gamma, self.beta, eps=self.eps, act=self.act, save8=self.save8)
        t = linear_act(h, self.w1, self.b1, act=self.act, save8=self.save8)
        return linear_act(t, self.w2, self.b2, res=x, act="none", save8=self.save8)
