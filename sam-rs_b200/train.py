"""The encoder block under torch.autograd: the fused attention and LayerNorm with this library's backward passes.

    y = train.attention_relpos(q, kt, v, table, h, w, scale)   gradients to q, kt, v, table
    y = train.layer_norm(x, weight, bias, eps)                 gradients to x, weight, bias
    y, x = train.layer_norm_residual(x, weight, bias, eps)     the norm of a residual branch x + f(norm(x))
    blk = train.TrainBlock(params, heads, window); y = blk(x)  one block of the encoder

An operator's tensors are of one type (f32, f16 or bf16), as everywhere in this package: mixed ones raise, also under
autocast. The projections of TrainBlock are library matrix products, as in `Attention`; everything else of the attention is
the library's kernels in both directions. Clip what loss.backward() leaves with clip_grad_norm.
"""
import torch

from . import attention_relpos_bwd, attention_relpos_lse, layer_norm_bwd
from . import layer_norm as _layer_norm
from . import window_partition, window_unpartition


class _AttentionRelpos(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, kt, v, table, h, w, scale):
        q, kt, v, table = (t.contiguous() for t in (q, kt, v, table))
        out, lse = attention_relpos_lse(q, kt, v, table, h, w, scale)
        ctx.save_for_backward(q, kt, v, table, out, lse)
        ctx.geometry = (h, w, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, kt, v, table, out, lse = ctx.saved_tensors
        return (*attention_relpos_bwd(dout.contiguous(), q, kt, v, table, out, lse, *ctx.geometry), None, None, None)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return _layer_norm(x, weight, bias, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        return (*layer_norm_bwd(dy.contiguous(), x, weight, ctx.eps), None)


class _LayerNormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return _layer_norm(x, weight, bias, eps), x.view_as(x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dres):
        x, weight = ctx.saved_tensors
        return (*layer_norm_bwd(dy.contiguous(), x, weight, ctx.eps, dres.contiguous()), None)


def attention_relpos(q, kt, v, table, h, w, scale):
    """Differentiable attention_relpos (q/v [BH, h*w, hd], kt [BH, hd, h*w], table [(2h-1)+(2w-1), hd])."""
    return _AttentionRelpos.apply(q, kt, v, table, h, w, float(scale))


def layer_norm(x, weight, bias, eps=1e-6):
    """Differentiable layer_norm over the last dim."""
    return _LayerNorm.apply(x, weight, bias, float(eps))


def layer_norm_residual(x, weight, bias, eps=1e-6):
    """(layer_norm(x), x) for a residual branch x + f(layer_norm(x)): used so, the two gradients of x are added inside
    the norm's backward kernel."""
    return _LayerNormResidual.apply(x, weight, bias, float(eps))


class TrainBlock(torch.nn.Module):
    """A SAM ViT encoder block to train (src/sam1/encoder.rs:89-129): the parameters of `Block` (same names and
    shapes, weights as stored [out, in]) and its forward pass, differentiable. x [B, H, W, C]."""

    def __init__(self, params, heads, window, eps=1e-6):
        super().__init__()
        self.heads, self.window, self.eps = heads, window, eps
        for name, value in params.items():
            self.register_parameter(name, torch.nn.Parameter(value.detach().clone()))

    def forward(self, x):
        b, h, w, c = x.shape
        nh = self.heads
        hd = c // nh
        y, x = layer_norm_residual(x, self.norm1_w, self.norm1_b, self.eps)
        hp, wp = h, w
        wh, ww = h, w
        if self.window:
            y, hp, wp = window_partition(y, self.window)
            wh = ww = self.window
        nw, n = y.shape[0], wh * ww
        qkv = torch.nn.functional.linear(y.reshape(nw, n, c), self.qkv_w, self.qkv_b).reshape(nw, n, 3, nh, hd)
        q = qkv[:, :, 0].permute(0, 2, 1, 3).reshape(nw * nh, n, hd)
        kt = qkv[:, :, 1].permute(0, 2, 3, 1).reshape(nw * nh, hd, n)
        v = qkv[:, :, 2].permute(0, 2, 1, 3).reshape(nw * nh, n, hd)
        table = torch.cat([self.rel_pos_h, self.rel_pos_w], 0)
        a = attention_relpos(q, kt, v, table, wh, ww, float(hd) ** -0.5)
        a = a.reshape(nw, nh, n, hd).permute(0, 2, 1, 3).reshape(nw, wh, ww, c)
        if self.window:
            a = window_unpartition(a, self.window, hp, wp, (h, w), b, c)
        x = x + torch.nn.functional.linear(a, self.proj_w, self.proj_b)
        y, x = layer_norm_residual(x, self.norm2_w, self.norm2_b, self.eps)
        m = torch.nn.functional.gelu(torch.nn.functional.linear(y, self.lin1_w, self.lin1_b))
        return x + torch.nn.functional.linear(m, self.lin2_w, self.lin2_b)
