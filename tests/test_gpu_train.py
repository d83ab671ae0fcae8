"""The training operators on the GPU against their formulas in 64 bits: the attention's softmax sums and backward
pass, LayerNorm's backward pass, gradient clipping, and a block trained with them.

Tolerances. f32: every logit carries rounding errors of a few 2^-24 of its size (up to about 40 here), which move
P by at most about 1e-5 of itself; bound 2e-5 in the 2-norm. 16-bit: P, dS, out (through D) and the result are each
rounded once to the I/O type, independent errors of 1.65e-3 (bf16) or 2.1e-4 (f16) rms (half a step of 2^-7 or
2^-10, uniform, over numbers spread within a power of two): together 3.3e-3 and 4.2e-4; bounds 5e-3 and 1e-3 (f16:
also what falls below its normal range)."""
import pytest

from tests import train_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = {"f32": 2e-5, "f16": 1e-3, "bf16": 5e-3}
NAMES = ("dq", "dkt", "dv", "dtable")


def inputs(h, w, bh, hd, dt, dev, seed=0, table_std=0.3, dout_std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + 1000 * h + w)
    n = h * w
    shapes = [(bh, n, hd), (bh, hd, n), (bh, n, hd), (2 * h + 2 * w - 2, hd), (bh, n, hd)]
    q, kt, v, t, dout = (torch.randn(*s, generator=g, device=dev) for s in shapes)
    return [x.to(DT[dt]) for x in (q, kt, v, t * table_std, dout * dout_std)]


def rel2(got, want):
    want = want.double()
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-300))


def run_bwd(samrs, h, w, bh, hd, dt, dev, impl="auto", **kw):
    q, kt, v, t, dout = inputs(h, w, bh, hd, dt, dev, **kw)
    scale = hd ** -0.5
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, scale)
    got = samrs.attention_relpos_bwd(dout, q, kt, v, t, out, lse, h, w, scale, impl=impl)
    assert samrs.device_status() == 0
    return got, (dout, q, kt, v, t, h, w, scale)


GRIDS = [(1, 5, 3, 8), (5, 1, 2, 33), (2, 3, 5, 1), (7, 11, 3, 80), (14, 14, 7, 64), (14, 14, 5, 80), (13, 17, 2, 20),
         (16, 8, 3, 128), (33, 47, 2, 32), (9, 30, 2, 48), (64, 3, 2, 96), (3, 64, 2, 16), (40, 25, 1, 112), (64, 64, 1, 64),
         (64, 64, 2, 80), (128, 2, 1, 64), (1, 128, 2, 128), (70, 65, 1, 32)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", GRIDS)
def test_attention_bwd_matches_formulas(samrs, cuda, h, w, bh, hd, dt):
    got, args = run_bwd(samrs, h, w, bh, hd, dt, cuda)
    want = ref.attention_bwd_by_heads(*args, heads=1)
    for name, a, b in zip(NAMES, got, want):
        assert a.dtype == DT[dt] and a.shape == b.shape
        assert rel2(a, b) < TOL[dt], name


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_one_token(samrs, cuda, dt):
    """One key: P = 1, so dv = dout, and dq, dk, dtable are 0 up to rounding: dP - D is a difference of two sums of
    hd = 64 products of unit size, equal but for their order (64 x 2^-24 x 64), against keys of unit size."""
    (dq, dkt, dv, dtable), (dout, *_rest) = run_bwd(samrs, 1, 1, 6, 64, dt, cuda)
    assert rel2(dv, dout) < TOL[dt]
    for g in (dq, dkt, dtable):
        assert float(g.float().abs().max()) < (1e-2 if dt == "bf16" else 2e-3)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", [(14, 14, 4, 80), (64, 64, 1, 64), (21, 10, 3, 32)])
def test_peaked_rows(samrs, cuda, h, w, bh, hd, dt):
    """Large tables: most rows put all their weight on one key, and the other probabilities underflow. Logits of a few
    hundred carry f32 errors of 1e-5 each, and the gradients are differences that nearly cancel: f32 bound 1e-3."""
    got, args = run_bwd(samrs, h, w, bh, hd, dt, cuda, table_std=4.0)
    want = ref.attention_bwd_by_heads(*args, heads=1)
    for name, a, b in zip(NAMES, got, want):
        assert bool(torch.isfinite(a).all()), name
        # out's rounding moves D by up to 2^-9 (2^-12) of |dout||out|, which a row of one key does not cancel
        assert rel2(a, b) < {"f32": 1e-3, "f16": 1e-2, "bf16": 5e-2}[dt], name


@pytest.mark.parametrize("std", [1e-4, 1e3])
@pytest.mark.parametrize("h,w,bh,hd", [(14, 14, 4, 64), (64, 64, 1, 80), (11, 19, 3, 48)])
def test_f16_gradients_of_any_size(samrs, cuda, h, w, bh, hd, std):
    """dS = P (dP - D) of small gradients and long rows is far below f16's normal range, that of large ones near its
    end: neither may lose it. Compared where the results themselves are f16 values of full precision."""
    got, args = run_bwd(samrs, h, w, bh, hd, "f16", cuda, dout_std=std)
    want = ref.attention_bwd_by_heads(*args, heads=1)
    for name, a, b in zip(NAMES, got, want):
        ok = (b.abs() > 2.0 ** -14) & (b.abs() < 6e4)
        if int(ok.sum()) > 100:
            assert rel2(a[ok], b[ok]) < 2 * TOL["f16"], name


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_many_heads(samrs, cuda, dt):
    """More heads than one group of the workspace holds."""
    h, w, bh, hd = 14, 14, 9300, 16
    got, args = run_bwd(samrs, h, w, bh, hd, dt, cuda)
    want = ref.attention_bwd_by_heads(*args, heads=500)
    for name, a, b in zip(NAMES, got, want):
        assert rel2(a, b) < TOL[dt], name


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h,w,hd", [(14, 14, 80), (12, 9, 64)])
def test_odd_addresses(samrs, cuda, h, w, hd, dt):
    """Dense tensors that begin one element into their storage."""
    def moved(x):
        buf = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
        buf[1:].copy_(x.flatten())
        return buf[1:].view(x.shape)

    q, kt, v, t, dout = (moved(x) for x in inputs(h, w, 3, hd, dt, cuda))
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, 0.2)
    got = samrs.attention_relpos_bwd(dout, q, kt, v, t, moved(out), lse, h, w, 0.2)
    assert samrs.device_status() == 0
    want = ref.attention_bwd_by_heads(dout, q, kt, v, t, h, w, 0.2)
    for name, a, b in zip(NAMES, got, want):
        assert rel2(a, b) < TOL[dt], name


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", [(14, 14, 50, 80), (64, 64, 3, 80), (33, 47, 2, 32), (10, 10, 2, 20)])
def test_same_inputs_same_bits(samrs, cuda, h, w, bh, hd, dt):
    first, args = run_bwd(samrs, h, w, bh, hd, dt, cuda)
    again, _ = run_bwd(samrs, h, w, bh, hd, dt, cuda)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_empty_batch(samrs, cuda):
    q, kt, t = torch.empty(0, 6, 8, device=cuda), torch.empty(0, 8, 6, device=cuda), torch.ones(8, 8, device=cuda)
    out, lse = samrs.attention_relpos_lse(q, kt, q, t, 2, 3, 0.5)
    assert out.shape == q.shape and lse.shape == (0, 6)
    dq, dkt, dv, dt = samrs.attention_relpos_bwd(q, q, kt, q, t, out, lse, 2, 3, 0.5)
    assert dq.shape == q.shape and dkt.shape == kt.shape and float(dt.abs().max()) == 0


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", [(14, 14, 37, 80), (14, 14, 20, 64), (64, 64, 2, 80), (64, 64, 2, 64), (7, 11, 3, 80),
                                       (1, 1, 2, 8), (30, 41, 2, 33)])
@pytest.mark.parametrize("table_std", [0.3, 4.0])
def test_forward_with_softmax_sums(samrs, cuda, h, w, bh, hd, dt, table_std):
    """out is attention_relpos's, bit for bit. lse: f32 logits of size X carry errors of a few 2^-24 X, and the
    exponentials' 3e-6 of the sum add to that; 16-bit products are exact in f32."""
    q, kt, v, t, _ = inputs(h, w, bh, hd, dt, cuda, table_std=table_std)
    samrs.global_policy(t, reset=True)
    plain = samrs.attention_relpos(q, kt, v, t, h, w, hd ** -0.5)
    samrs.global_policy(t, reset=True)
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, hd ** -0.5)
    assert samrs.device_status() == 0
    assert torch.equal(out, plain)
    for b in range(bh):
        x, _, _ = ref.logits(q[b:b + 1].double(), kt[b:b + 1].double(), t.double(), h, w, hd ** -0.5)
        err = (lse[b].double() - torch.logsumexp(x[0], -1)).abs()
        size = x[0].abs().amax(-1)
        # the f32 tensor-core kernel multiplies in three TF32 products: 2^-20 of the sum of |q||k|
        assert bool((err <= 4e-6 + size * (1e-6 if dt != "f32" else 4e-6)).all()), float((err / (1 + size)).max())


def test_gradient_against_differences(samrs, cuda):
    """Directional derivative of the f32 kernels' own forward pass. A step of 1e-2 in unit directions: truncation
    about 1e-4 of the derivative, rounding 2^-24 sqrt(n) / 1e-2 less than that; bound 2e-3."""
    h, w, bh, hd = 9, 7, 2, 40
    q, kt, v, t, dout = inputs(h, w, bh, hd, "f32", cuda)
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, 0.2)
    grads = samrs.attention_relpos_bwd(dout, q, kt, v, t, out, lse, h, w, 0.2)
    g = torch.Generator(device=cuda).manual_seed(5)
    args = [q, kt, v, t]
    for k in range(4):
        d = torch.randn(args[k].shape, generator=g, device=cuda)
        d = d + grads[k] * (d.norm() / grads[k].norm())  # a direction the loss does change along
        vals = []
        for s in (1e-2, -1e-2):
            moved = list(args)
            moved[k] = args[k] + s * d / d.norm()
            vals.append((samrs.attention_relpos(*moved, h, w, 0.2).double() * dout.double()).sum())
        got, want = float((vals[0] - vals[1]) / 2e-2), float((grads[k].double() * d.double()).sum() / d.norm())
        assert abs(got - want) < 2e-3 * abs(want), NAMES[k]


def test_other_stream_and_graph(samrs, cuda):
    """On a stream of the caller's, and replayed from a captured graph: the same bits as on the default stream."""
    sets = [inputs(h, w, bh, hd, "bf16", cuda) + [h, w] for h, w, bh, hd in ((14, 14, 9, 80), (64, 64, 1, 64), (5, 9, 2, 24))]
    x, dy = torch.randn(300, 96, device=cuda), torch.randn(300, 96, device=cuda)
    wt = torch.randn(96, device=cuda)

    def step():
        res = []
        for q, kt, v, t, dout, h, w in sets:
            out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, 0.1)
            res += [out, lse, *samrs.attention_relpos_bwd(dout, q, kt, v, t, out, lse, h, w, 0.1)]
        res += samrs.layer_norm_bwd(dy, x, wt)
        clipped = [torch.empty_like(x) for x in res[-3:]]
        return res + [samrs.clip_grad_norm(res[-3:], 0.1, out=clipped)] + clipped

    want = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = step()
        s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for o in got:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    assert samrs.device_status() == 0
    del graph


def test_bad_tensors_are_refused(samrs, cuda):
    q, kt, v, t, dout = inputs(3, 4, 2, 16, "f32", cuda)
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, 3, 4, 0.5)
    bad = [(dout[:1], q, kt, v, t, out, lse), (dout.half(), q, kt, v, t, out, lse), (dout, q, v, v, t, out, lse),
           (dout, q, kt, v, t[:-1], out, lse), (dout, q, kt, v, t, out, lse.half()), (dout, q, kt, v, t, out, lse[:, :-1]),
           (dout.transpose(0, 1), q, kt, v, t, out, lse), (dout, q, kt, v, t, out, lse.cpu())]
    for args in bad:
        with pytest.raises(samrs.SamrsError):
            samrs.attention_relpos_bwd(*args, 3, 4, 0.5)
    with pytest.raises(samrs.SamrsError):
        samrs.attention_relpos_bwd(dout, q, kt, v, t, out, lse, 4, 4, 0.5)
    x = torch.zeros(4, 8, device=cuda)
    for args in ((x[:2], x, x[0]), (x, x, x[0, :4]), (x.half(), x, x[0]), (x.t(), x.t(), x[:, 0])):
        with pytest.raises(samrs.SamrsError):
            samrs.layer_norm_bwd(*args)
    for grads, out in (([x, x.cpu()], None), ([x.double()], None), ([x.t()], None), ([x], []), ([x], [x[:2]])):
        with pytest.raises(samrs.SamrsError):
            samrs.clip_grad_norm(grads, 1.0, out=out)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 2), (1, 768), (7, 100), (333, 777), (4096, 1280), (77, 1024), (50, 1536),
                                    (20, 2048), (5, 2056), (33, 5000), (1000, 256), (9, 1000)])
@pytest.mark.parametrize("res", [False, True])
def test_layer_norm_bwd_matches_formulas(samrs, cuda, rows, c, dt, res):
    g = torch.Generator(device=cuda).manual_seed(rows + c)
    x, dy, dres = ((torch.randn(rows, c, generator=g, device=cuda) * s + m).to(DT[dt]) for s, m in ((2, .5), (1, 0), (1, 0)))
    wt = torch.randn(c, generator=g, device=cuda).to(DT[dt])
    got = samrs.layer_norm_bwd(dy, x, wt, 1e-3, dres=dres if res else None)
    want = ref.layer_norm_bwd(dy.double(), x.double(), wt.double(), 1e-3, dres.double() if res else None)
    for a, b in zip(got, want):
        # one rounding of the result; f32 sums of `rows` terms. Rows of one or two channels cancel to 0 (norm < 1).
        err = float((a.double() - b).norm() / b.norm().clamp_min(1.0))
        assert err < {"f32": 1e-5, "f16": 6e-4, "bf16": 4e-3}[dt]
    again = samrs.layer_norm_bwd(dy, x, wt, 1e-3, dres=dres if res else None)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_layer_norm_bwd_shapes(samrs, cuda):
    """Leading dims, no rows, and rows that begin at odd addresses."""
    x = torch.randn(2, 3, 5, 64, device=cuda)
    dy, wt = torch.randn_like(x), torch.randn(64, device=cuda)
    dx, dw, db = samrs.layer_norm_bwd(dy, x, wt)
    want = ref.layer_norm_bwd(dy.double(), x.double(), wt.double(), 1e-6)
    assert dx.shape == x.shape and rel2(dx, want[0]) < 1e-5 and rel2(dw, want[1]) < 1e-5 and rel2(db, want[2]) < 1e-5
    dx, dw, db = samrs.layer_norm_bwd(dy[:0], x[:0], wt)
    assert dx.numel() == 0 and float(dw.abs().max()) == 0 and float(db.abs().max()) == 0
    buf, bufy = torch.randn(641, device=cuda).half(), torch.randn(641, device=cuda).half()
    x, dy = buf[1:].view(10, 64), bufy[1:].view(10, 64)
    got = samrs.layer_norm_bwd(dy, x, wt.half())
    want = ref.layer_norm_bwd(dy.double(), x.double(), wt.half().double(), 1e-6)
    assert all(rel2(a, b) < 6e-4 for a, b in zip(got, want))


def clip_tensors(dt, dev, count=9, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    sizes = [1, 7, 0, 16384, 16385, 40000, 8, 100001, 3]
    return [(torch.randn(sizes[i % 9], generator=g, device=dev) * 0.1).to(DT[dt]) for i in range(count)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", [None, "f32", "f16", "bf16"])
@pytest.mark.parametrize("count", [1, 9, 1100])
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0])
def test_clip_grad_norm(samrs, cuda, dt, out, count, max_norm):
    grads = clip_tensors(dt, cuda, count)
    before = [g.clone() for g in grads]
    outs = None if out is None else [torch.empty_like(g, dtype=DT[out]) for g in grads]
    norm = samrs.clip_grad_norm(grads, max_norm, out=outs)
    want = torch.cat([g.double() for g in before]).norm()
    assert abs(float(norm) - float(want)) <= 1e-6 * float(want)
    f = min(1.0, max_norm / (float(want) + 1e-6))
    to = dt if out is None else out
    # one rounding of g f; what lies below f16's normal range keeps an absolute 2^-25
    tol = {"f32": 1e-6, "f16": 2.0 ** -11 * 1.01, "bf16": 2.0 ** -8 * 1.01}[to]
    for a, b in zip(grads if out is None else outs, before):
        err = (a.double() - b.double() * f).abs()
        assert bool((err <= tol * (b.double() * f).abs() + (2.0 ** -25 if to == "f16" else 0)).all())
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_clip_grad_norm_addresses_and_non_finite(samrs, cuda):
    buf = torch.randn(70001, device=cuda).bfloat16()
    view, whole = buf[1:], torch.randn(33, 5, device=cuda)
    want = torch.cat([view.double(), whole.double().flatten()]).norm()
    first, head = view.clone(), buf[0].clone()
    norm = samrs.clip_grad_norm([view, whole], 1.0)
    assert abs(float(norm) - float(want)) <= 1e-6 * float(want)
    assert float((view.double() - first.double() / float(want)).abs().max()) < 2.0 ** -8 * float(first.abs().max()) / float(want)
    assert torch.equal(buf[0], head)
    empty = torch.empty(0, device=cuda)
    assert float(samrs.clip_grad_norm([empty], 1.0)) == 0
    g = torch.ones(100, device=cuda)
    g[3] = float("inf")
    assert float(samrs.clip_grad_norm([g], 1.0)) == float("inf")
    assert float(g[0]) == 0 and bool(torch.isnan(g[3]))
    g = torch.ones(100, device=cuda)
    g[3] = float("nan")
    assert bool(torch.isnan(samrs.clip_grad_norm([g], 1.0))) and bool(torch.isnan(g).all())


def test_large_tensor(samrs, cuda):
    """More than 2^31 elements in one tensor."""
    n = (1 << 31) + 4099
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    g[-4:] = 3.0
    assert abs(float(samrs.clip_grad_norm([g], 3.0)) - 6.0) < 1e-5
    assert [float(x) for x in g[-5:]] == [0.0, 1.5, 1.5, 1.5, 1.5]


@pytest.mark.parametrize("window", [5, 0])
def test_train_block_matches_plain_autograd(samrs, cuda, window):
    """A block's gradients against torch's own autograd through the same block in 64 bits. f32: matrix products of the
    library on 64-bit-free inputs; the deepest chain is about 10 of them, 1e-6 each; bound 1e-4."""
    from tests.test_gpu_block import block_params
    g = torch.Generator(device=cuda).manual_seed(window)
    heads, dim, side = 3, 48, 8
    span = window or side
    shapes = {"norm1_w": (dim,), "norm1_b": (dim,), "qkv_w": (3 * dim, dim), "qkv_b": (3 * dim,), "proj_w": (dim, dim),
              "proj_b": (dim,), "rel_pos_h": (2 * span - 1, dim // heads), "rel_pos_w": (2 * span - 1, dim // heads),
              "norm2_w": (dim,), "norm2_b": (dim,), "lin1_w": (4 * dim, dim), "lin1_b": (4 * dim,), "lin2_w": (dim, 4 * dim),
              "lin2_b": (dim,)}
    assert set(shapes) == set(block_params(dim, heads, window, g, cuda, "f16"))
    params = {k: torch.randn(*s, generator=g, device=cuda) * 0.2 for k, s in shapes.items()}
    x = torch.randn(2, side, side, dim, generator=g, device=cuda)
    up = torch.randn(2, side, side, dim, generator=g, device=cuda)
    blk = samrs.train.TrainBlock(params, heads, window)
    xg = x.clone().requires_grad_(True)
    y = blk(xg)
    y.backward(up)
    p64 = {k: v.double().requires_grad_(True) for k, v in params.items()}
    x64 = x.double().requires_grad_(True)

    def norm(z, a, b):
        return torch.nn.functional.layer_norm(z, (dim,), a, b, 1e-6)

    z = norm(x64, p64["norm1_w"], p64["norm1_b"])
    hp, wp = side, side
    if window:
        z, hp, wp = samrs.window_partition(z, window)
    nw, n, hd = z.shape[0], span * span, dim // heads
    qkv = (z.reshape(nw, n, dim) @ p64["qkv_w"].T + p64["qkv_b"]).reshape(nw, n, 3, heads, hd).permute(2, 0, 3, 1, 4)
    q, k, v = (t.reshape(nw * heads, n, hd) for t in qkv)
    table = torch.cat([p64["rel_pos_h"], p64["rel_pos_w"]])
    a, _ = ref.attention(q, k.transpose(1, 2), v, table, span, span, hd ** -0.5)
    a = a.reshape(nw, heads, span, span, hd).permute(0, 2, 3, 1, 4).reshape(nw, span, span, dim)
    if window:
        a = samrs.window_unpartition(a, window, hp, wp, (side, side), 2, dim)
    x1 = x64 + a @ p64["proj_w"].T + p64["proj_b"]
    z = norm(x1, p64["norm2_w"], p64["norm2_b"])
    want = x1 + torch.nn.functional.gelu(z @ p64["lin1_w"].T + p64["lin1_b"]) @ p64["lin2_w"].T + p64["lin2_b"]
    want.backward(up.double())
    assert rel2(y, want.detach()) < 1e-4 and rel2(xg.grad, x64.grad) < 1e-4
    for k, p in blk.named_parameters():
        assert rel2(p.grad, p64[k].grad) < 1e-4, k
    norm_got = samrs.clip_grad_norm([p.grad for p in blk.parameters()], 1.0)
    total = torch.cat([p.grad.flatten() for p in p64.values()]).norm()
    assert abs(float(norm_got) - float(total)) < 1e-4 * float(total)
    left = torch.cat([p.grad.flatten() for p in blk.parameters()]).norm()
    assert abs(float(left) - 1.0) < 1e-4


def test_training_lowers_the_loss(samrs, cuda):
    """A windowed bf16 block fitted to a target for a few clipped steps: every step lowers the loss (at first order by
    lr times the squared norm of the gradient, about 0.07, far above the loss's rounding)."""
    from tests.test_gpu_block import block_params
    g = torch.Generator(device=cuda).manual_seed(4)
    blk = samrs.train.TrainBlock(block_params(256, 4, 14, g, cuda, "bf16"), 4, 14)
    x = torch.randn(1, 28, 28, 256, generator=g, device=cuda).bfloat16()
    target = torch.randn(1, 28, 28, 256, generator=g, device=cuda).bfloat16()
    losses = []
    opt = torch.optim.SGD(blk.parameters(), lr=0.5)
    for _ in range(12):
        opt.zero_grad(set_to_none=True)
        loss = (blk(x).float() - target.float()).square().mean()
        loss.backward()
        samrs.clip_grad_norm([p.grad for p in blk.parameters()], 1.0)
        opt.step()
        losses.append(float(loss))
    assert samrs.device_status() == 0
    assert all(b < a for a, b in zip(losses, losses[1:])), losses


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", [(14, 14, 6, 80), (64, 64, 1, 64), (21, 10, 3, 32), (3, 17, 5, 16)])
def test_both_kernels_of_a_shape(samrs, cuda, h, w, bh, hd, dt):
    """The tensor-core and the CUDA-core kernels of a 16-bit shape, each asked for by name."""
    for impl in ("tc", "simt"):
        got, args = run_bwd(samrs, h, w, bh, hd, dt, cuda, impl=impl)
        want = ref.attention_bwd_by_heads(*args, heads=1)
        for name, a, b in zip(NAMES, got, want):
            assert rel2(a, b) < TOL[dt], (impl, name)


@pytest.mark.parametrize("h,w,hd,dt", [(14, 14, 64, "f32"), (14, 14, 20, "bf16"), (65, 3, 64, "f16")])
def test_tensor_core_kernels_refuse_other_shapes(samrs, cuda, h, w, hd, dt):
    q, kt, v, t, dout = inputs(h, w, 1, hd, dt, cuda)
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, 0.2)
    with pytest.raises(samrs.SamrsError):
        samrs.attention_relpos_bwd(dout, q, kt, v, t, out, lse, h, w, 0.2, impl="tc")


def test_offsets_past_32_bits(samrs, cuda):
    """Heads whose elements lie past 2^31: the last ones' gradients are those of the same heads by themselves. (Each head
    is computed the same way wherever it stands; only dtable is a sum over heads.)"""
    h, w, hd = 14, 14, 80
    n, few = h * w, 8
    bh = 2 ** 31 // (n * hd) + 2 * few
    q, kt, v, t, dout = inputs(h, w, few, hd, "bf16", cuda)

    def many(x):
        big = torch.zeros(bh, *x.shape[1:], dtype=x.dtype, device=cuda)
        big[-few:] = x
        return big

    own = samrs.attention_relpos_lse(q, kt, v, t, h, w, 0.1)
    want = samrs.attention_relpos_bwd(dout, q, kt, v, t, *own, h, w, 0.1)
    big = [many(x) for x in (dout, q, kt, v)]
    assert big[0].numel() > 2 ** 31
    out, lse = samrs.attention_relpos_lse(*big[1:], t, h, w, 0.1)
    assert torch.equal(out[-few:], own[0]) and torch.equal(lse[-few:], own[1])
    got = samrs.attention_relpos_bwd(*big, t, out, lse, h, w, 0.1)
    assert samrs.device_status() == 0
    for name, a, b in zip(NAMES[:3], got, want):
        assert torch.equal(a[-few:], b), name
        assert float(a[0].abs().max()) == 0, name  # (a head of zeros has none)
    assert rel2(got[3], want[3].double()) < TOL["bf16"]


def test_residual_norm(samrs, cuda):
    """x + f(norm(x)) through layer_norm_residual: the gradients of plain autograd in 64 bits. f32 sums of 96 and 40
    elements; bound 1e-5."""
    g = torch.Generator(device=cuda).manual_seed(6)
    x, wt, bs = (torch.randn(*s, generator=g, device=cuda).requires_grad_(True) for s in ((5, 8, 96), (96,), (96,)))
    up = torch.randn(5, 8, 96, generator=g, device=cuda)
    y, r = samrs.train.layer_norm_residual(x, wt, bs)
    (r + y.square()).backward(up)
    x64, w64, b64 = (t.detach().double().requires_grad_(True) for t in (x, wt, bs))
    (x64 + torch.nn.functional.layer_norm(x64, (96,), w64, b64, 1e-6).square()).backward(up.double())
    for a, b in ((x, x64), (wt, w64), (bs, b64)):
        assert rel2(a.grad, b.grad) < 1e-5


def test_example(samrs, cuda):
    """The example's losses fall and its norms are those of its gradients (positive and finite)."""
    import examples.train_block as ex
    losses, norms = ex.train(steps=8)
    assert losses[-1] < losses[0] and all(0 < x < float("inf") for x in norms)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", [(14, 14, 75, 64), (40, 7, 20, 48), (17, 23, 20, 96), (3, 3, 200, 20), (60, 60, 2, 128),
                                       (1, 65, 9, 7), (128, 128, 1, 128)])
def test_groups_of_warps(samrs, cuda, h, w, bh, hd, dt):
    """The any-shape kernels with one, two and four groups of warps to a tile (many tiles, some, few)."""
    got, args = run_bwd(samrs, h, w, bh, hd, dt, cuda, impl="simt")
    want = ref.attention_bwd_by_heads(*args, heads=1)
    for name, a, b in zip(NAMES, got, want):
        assert rel2(a, b) < TOL[dt], name
