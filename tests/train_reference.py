"""The training operators' formulas in 64 bits (torch tensors on any device), for the tests of the kernels."""
import torch


def relpos_index(n, device):
    i = torch.arange(n, device=device)
    return i[:, None] - i[None, :] + n - 1


def logits(q, kt, table, h, w, scale):
    """x [bh, n, n] and the expanded tables Rh [h, h, hd], Rw [w, w, hd]."""
    bh, n, hd = q.shape
    rh = table[: 2 * h - 1][relpos_index(h, q.device)]
    rw = table[2 * h - 1:][relpos_index(w, q.device)]
    q4 = q.view(bh, h, w, hd)
    x = (scale * (q @ kt)).view(bh, h, w, h, w)
    x = x + torch.einsum("bijd,ikd->bijk", q4, rh)[..., :, None] + torch.einsum("bijd,jkd->bijk", q4, rw)[..., None, :]
    return x.view(bh, n, n), rh, rw


def attention(q, kt, v, table, h, w, scale):
    x, _, _ = logits(q, kt, table, h, w, scale)
    lse = torch.logsumexp(x, -1)
    return torch.exp(x - lse[..., None]) @ v, lse


def attention_bwd(dout, q, kt, v, table, h, w, scale):
    """(dq, dkt, dv, dtable) of a batch of heads, from the formulas."""
    bh, n, hd = q.shape
    x, rh, rw = logits(q, kt, table, h, w, scale)
    p = torch.softmax(x, -1)
    out = p @ v
    ds = p * (dout @ v.transpose(1, 2) - (dout * out).sum(-1, keepdim=True))
    dv = p.transpose(1, 2) @ dout
    dkt = scale * (q.transpose(1, 2) @ ds)
    ds5 = ds.view(bh, h, w, h, w)
    dh, dw = ds5.sum(4), ds5.sum(3)
    dq = scale * (ds @ kt.transpose(1, 2)).view(bh, h, w, hd)
    dq = dq + torch.einsum("bijk,ikd->bijd", dh, rh) + torch.einsum("bijk,jkd->bijd", dw, rw)
    q4 = q.view(bh, h, w, hd)
    dtable = torch.zeros_like(table)
    dtable[: 2 * h - 1].index_add_(0, relpos_index(h, q.device).flatten(),
                                   torch.einsum("bijk,bijd->ikd", dh, q4).reshape(h * h, hd))
    dtable[2 * h - 1:].index_add_(0, relpos_index(w, q.device).flatten(),
                                  torch.einsum("bijk,bijd->jkd", dw, q4).reshape(w * w, hd))
    return dq.reshape(bh, n, hd), dkt, dv, dtable


def attention_bwd_by_heads(dout, q, kt, v, table, h, w, scale, heads=4):
    """attention_bwd in 64 bits, a few heads at a time (the n x n tensors of large grids)."""
    parts, dtable = [], 0
    for b in range(0, q.shape[0], heads):
        *one, dt = attention_bwd(*(t[b:b + heads].double() for t in (dout, q, kt, v)), table.double(), h, w, scale)
        parts.append(one)
        dtable = dtable + dt
    return (*(torch.cat(p) for p in zip(*parts)), dtable)


def layer_norm_bwd(dy, x, weight, eps, dres=None):
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    g = dy * weight
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    c = x.shape[-1]
    return (dx if dres is None else dx + dres), (dy * xh).reshape(-1, c).sum(0), dy.reshape(-1, c).sum(0)
