"""Cases, plain forms and 64-bit values of the training operators of the encoder blocks: the attention with decomposed
relative-position bias that also returns the log of its softmax sums, its backward pass (which recomputes the
probabilities), LayerNorm's backward pass, and the global gradient norm with clipping.

`own` chooses what run() calls: elementary torch operations in 32 bits, or this package's operators."""
import importlib
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _samrs():
    return importlib.import_module("sam-rs_b200")


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the windowed layers of one image through the huge encoder: 25 windows x 16 heads
        {"name": "bwd windows bf16", "op": "attn_bwd", "h": 14, "w": 14, "bh": 400, "hd": 80, "dtype": "bf16"},
        # one window of the base encoder: the smallest call, where latency counts
        {"name": "bwd one window f16", "op": "attn_bwd", "h": 14, "w": 14, "bh": 12, "hd": 64, "dtype": "f16"},
        # a global layer of one image through the huge encoder: the largest
        {"name": "bwd global bf16", "op": "attn_bwd", "h": 64, "w": 64, "bh": 16, "hd": 80, "dtype": "bf16"},
        # a crop of a feature map with an odd number of tokens
        {"name": "bwd odd grid f16", "op": "attn_bwd", "h": 33, "w": 47, "bh": 24, "hd": 32, "dtype": "f16"},
        # 32-bit fine-tuning, the windows of a quarter of an image through the base encoder
        {"name": "bwd windows f32", "op": "attn_bwd", "h": 14, "w": 14, "bh": 75, "hd": 64, "dtype": "f32"},
        # the forward pass that keeps what the backward pass needs: windowed layers, and a small odd grid
        {"name": "fwd windows bf16", "op": "attn_fwd", "h": 14, "w": 14, "bh": 400, "hd": 80, "dtype": "bf16"},
        {"name": "fwd odd grid f32", "op": "attn_fwd", "h": 7, "w": 11, "bh": 30, "hd": 80, "dtype": "f32"},
        # norm1 / norm2 of one image, and of a batch of 8 with the residual stream's gradient added; odd rows and channels
        {"name": "norm bwd bf16", "op": "norm_bwd", "rows": 4096, "c": 1280, "dtype": "bf16", "res": False},
        {"name": "norm bwd batch bf16", "op": "norm_bwd", "rows": 32768, "c": 768, "dtype": "bf16", "res": True},
        {"name": "norm bwd odd f32", "op": "norm_bwd", "rows": 333, "c": 777, "dtype": "f32", "res": True},
        # all gradients of four blocks of the huge encoder, 16-bit, clipped into the optimiser's 32-bit buffers
        {"name": "clip blocks bf16", "op": "clip", "dim": 1280, "tensors": 52, "dtype": "bf16", "out": "f32", "max_norm": 1.0},
        # a small decoder's gradients
        {"name": "clip small f32", "op": "clip", "dim": 96, "tensors": 39, "dtype": "f32", "out": "f32", "max_norm": 0.5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn_bwd", "attn_bwd", "attn_bwd", "attn_fwd", "norm_bwd", "clip"])
    if op in ("attn_bwd", "attn_fwd"):
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        kind = rng.choice(["window", "global", "odd"])
        if kind == "window":
            h = w = 14
            hd = rng.choice([64, 80])
            bh = _log_int(rng, 4, 400)
        elif kind == "global":
            h = w = 64
            hd = rng.choice([64, 80])
            bh = rng.randint(1, 14)
        else:
            h, w = _log_int(rng, 2, 60), _log_int(rng, 2, 60)
            hd = rng.choice([16, 32, 48, 64, 80, 96, 128])
            bh = _log_int(rng, 1, 96)
        if dtype == "f32":
            bh = max(1, bh // 4)
        most = 14 * 4096.0 ** 2 * 80 / (h * w) ** 2 / hd  # no more work than the largest listed case
        return {"op": op, "h": h, "w": w, "bh": max(1, min(bh, int(most))), "hd": hd, "dtype": dtype}
    if op == "norm_bwd":
        return {"op": op, "rows": _log_int(rng, 1, 32768), "c": rng.choice([768, 1024, 1280, rng.randint(64, 1536)]),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "res": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "f16", "f32"])
    return {"op": op, "dim": _log_int(rng, 32, 1280), "tensors": rng.randint(1, 52), "dtype": dtype,
            "out": rng.choice([dtype, "f32"]), "max_norm": rng.choice([0.1, 1.0, 1e6])}


def _clip_shapes(case):
    """Parameter shapes of `tensors` / 13 encoder blocks of width dim (biases, norms, projections and rel-pos tables)."""
    c = case["dim"]
    block = [(3 * c, c), (3 * c,), (c, c), (c,), (27, max(1, c // 16)), (127, max(1, c // 16)), (c,), (c,), (4 * c, c),
             (4 * c,), (c, 4 * c), (c,), (c + 1,)]
    return [block[i % len(block)] for i in range(case["tensors"])]


# ----------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)

    s = dict(case)
    if case["op"] in ("attn_bwd", "attn_fwd"):
        h, w, bh, hd = case["h"], case["w"], case["bh"], case["hd"]
        n = h * w
        s.update(q=rnd(bh, n, hd), kt=rnd(bh, hd, n), v=rnd(bh, n, hd), table=rnd(2 * h + 2 * w - 2, hd, std=0.1),
                 scale=hd ** -0.5)
        if case["op"] == "attn_bwd":
            s["dout"] = rnd(bh, n, hd, std=0.05)
            # what the forward pass has left
            s["out"], s["lse"] = _plain_attn_fwd(s)
    elif case["op"] == "norm_bwd":
        s.update(x=rnd(case["rows"], case["c"]), dy=rnd(case["rows"], case["c"], std=0.05),
                 weight=1 + rnd(case["c"], std=0.2), eps=1e-6,
                 dres=rnd(case["rows"], case["c"], std=0.05) if case["res"] else None)
    else:
        # layers' gradients are of different sizes
        shapes = _clip_shapes(case)
        s["grads"] = [rnd(*shape, std=0.01 * (1 + i % 5)) for i, shape in enumerate(shapes)]
        s["outs"] = [torch.empty(shape, device=dev, dtype=_DTYPES[case["out"]]) for shape in shapes]
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _rel_index(n, dev):
    i = torch.arange(n, device=dev)
    return i[:, None] - i[None, :] + n - 1


def _plain_logits(s, q):
    h, w, bh = s["h"], s["w"], s["bh"]
    hd = s["hd"]
    t = s["table"].float()
    rh = t[: 2 * h - 1][_rel_index(h, t.device)]
    rw = t[2 * h - 1:][_rel_index(w, t.device)]
    x = (q @ s["kt"].float()) * s["scale"]
    q4 = q.view(bh, h, w, hd)
    bias_h = torch.einsum("bijd,ikd->bijk", q4, rh)
    bias_w = torch.einsum("bijd,jkd->bijk", q4, rw)
    x = x.view(bh, h, w, h, w) + bias_h[..., :, None] + bias_w[..., None, :]
    return x.view(bh, h * w, h * w), rh, rw


def _plain_attn_fwd(s):
    x, _, _ = _plain_logits(s, s["q"].float())
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    l = e.sum(-1, keepdim=True)
    out = (e / l) @ s["v"].float()
    return out.to(s["q"].dtype), (m + torch.log(l)).squeeze(-1)


def _plain_attn_bwd(s):
    h, w, bh, hd = s["h"], s["w"], s["bh"], s["hd"]
    dt = s["q"].dtype
    q, do = s["q"].float(), s["dout"].float()
    x, rh, rw = _plain_logits(s, q)
    p = torch.exp(x - s["lse"][..., None])
    delta = (do * s["out"].float()).sum(-1, keepdim=True)
    dv = p.transpose(1, 2) @ do
    ds = p * (do @ s["v"].float().transpose(1, 2) - delta)
    dkt = (q.transpose(1, 2) @ ds) * s["scale"]
    dq = (ds @ s["kt"].float().transpose(1, 2)) * s["scale"]
    ds = ds.view(bh, h, w, h, w)
    dh, dw = ds.sum(4), ds.sum(3)
    q4 = q.view(bh, h, w, hd)
    dq = dq.view(bh, h, w, hd) + torch.einsum("bijk,ikd->bijd", dh, rh) + torch.einsum("bijk,jkd->bijd", dw, rw)
    gh = torch.einsum("bijk,bijd->ikd", dh, q4).reshape(h * h, hd)
    gw = torch.einsum("bijk,bijd->jkd", dw, q4).reshape(w * w, hd)
    dtable = torch.cat([
        torch.zeros(2 * h - 1, hd, device=q.device).index_add_(0, _rel_index(h, q.device).flatten(), gh),
        torch.zeros(2 * w - 1, hd, device=q.device).index_add_(0, _rel_index(w, q.device).flatten(), gw)])
    return dq.reshape(bh, h * w, hd).to(dt), dkt.to(dt), dv.to(dt), dtable.to(dt)


def _plain_norm_bwd(s):
    x, dy, wt = s["x"].float(), s["dy"].float(), s["weight"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + s["eps"])
    xh = xc * rstd
    g = dy * wt
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    dt = s["x"].dtype
    return dx.to(dt), (dy * xh).sum(0).to(dt), dy.sum(0).to(dt)


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return norm, [o.copy_(g.float() * coef) for g, o in zip(s["grads"], s["outs"])]


def run(s):
    op = s["op"]
    if not own:
        plain = {"attn_fwd": _plain_attn_fwd, "attn_bwd": _plain_attn_bwd, "norm_bwd": _plain_norm_bwd, "clip": _plain_clip}
        return plain[op](s)
    samrs = _samrs()
    if op == "attn_fwd":
        return samrs.attention_relpos_lse(s["q"], s["kt"], s["v"], s["table"], s["h"], s["w"], s["scale"])
    if op == "attn_bwd":
        return samrs.attention_relpos_bwd(s["dout"], s["q"], s["kt"], s["v"], s["table"], s["out"], s["lse"], s["h"],
                                          s["w"], s["scale"])
    if op == "norm_bwd":
        return samrs.layer_norm_bwd(s["dy"], s["x"], s["weight"], s["eps"], dres=s["dres"])
    return samrs.clip_grad_norm(s["grads"], s["max_norm"], out=s["outs"]), s["outs"]


# ------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] in ("attn_bwd", "attn_fwd"):
        h, w, bh, hd, es = case["h"], case["w"], case["bh"], case["hd"], _BYTES[case["dtype"]]
        n = h * w
        table = (2 * h + 2 * w - 2) * hd * es
        if case["op"] == "attn_fwd":  # q, k, v -> out, lse; two products of n x n x hd, and the bias terms
            return {"bytes": 4 * bh * n * hd * es + 4 * bh * n + table, "flops": 4.0 * bh * n * n * hd + 2.0 * bh * n * (h + w) * hd}
        # q, k, v, out, dout, lse -> dq, dk, dv, dtable; five products, and the bias terms with their gradients
        return {"bytes": 8 * bh * n * hd * es + 4 * bh * n + 2 * table,
                "flops": 10.0 * bh * n * n * hd + 6.0 * bh * n * (h + w) * hd}
    if case["op"] == "norm_bwd":
        e = case["rows"] * case["c"]
        return {"bytes": (4 if case["res"] else 3) * e * _BYTES[case["dtype"]] + 3 * case["c"] * _BYTES[case["dtype"]],
                "flops": 15.0 * e}
    e = sum(math.prod(x) for x in _clip_shapes(case))
    return {"bytes": e * (_BYTES[case["dtype"]] + _BYTES[case["out"]]), "flops": 3.0 * e}


# ---------------------------------------------------------------------------------------- 64-bit values
def _exact_attention(q, k, v, table, h, w, scale):
    """One head in 64 bits, from the definition: every (query, key) pair's bias is a dot product with two table rows."""
    n = h * w
    i = torch.arange(n, device=q.device) // w
    j = torch.arange(n, device=q.device) % w
    by_row = q @ table.T  # [n, all table rows]
    at_h = i[:, None] - i[None, :] + (h - 1)
    at_w = j[:, None] - j[None, :] + (w - 1) + (2 * h - 1)
    x = scale * (q @ k) + by_row.gather(1, at_h) + by_row.gather(1, at_w)
    lse = torch.logsumexp(x, -1)
    return torch.softmax(x, -1) @ v, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("attn_bwd", "attn_fwd"):
        h, w = case["h"], case["w"]
        table = s["table"].double().requires_grad_(True)
        parts = []
        for b in range(case["bh"]):
            q, k, v = (s[name][b].double().requires_grad_(True) for name in ("q", "kt", "v"))
            out, lse = _exact_attention(q, k, v, table, h, w, s["scale"])
            if case["op"] == "attn_fwd":
                parts.append((out.detach(), lse.detach()))
            else:
                out.backward(s["dout"][b].double())
                parts.append((q.grad, k.grad, v.grad))
        whole = tuple(torch.stack(p) for p in zip(*parts))
        return whole if case["op"] == "attn_fwd" else whole + (table.grad,)
    if case["op"] == "norm_bwd":
        x, wt = s["x"].double().requires_grad_(True), s["weight"].double().requires_grad_(True)
        b = torch.zeros(case["c"], dtype=torch.float64, device=x.device, requires_grad=True)
        mean = x.sum(1, keepdim=True) / case["c"]
        var = ((x - mean) ** 2).sum(1, keepdim=True) / case["c"]
        y = (x - mean) / torch.sqrt(var + s["eps"]) * wt + b
        y.backward(s["dy"].double())
        dx = x.grad if s["dres"] is None else x.grad + s["dres"].double()
        return dx, wt.grad, b.grad
    total = torch.cat([g.flatten() for g in s["grads"]]).double().norm()
    scale = min(1.0, case["max_norm"] / (float(total) + 1e-6))
    return total, [g.double() * scale for g in s["grads"]]
