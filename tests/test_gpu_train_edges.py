"""The training operators on the GPU where they depend on what ran before, or reach the ends of a type's range."""
import pytest

from tests import train_reference as ref
from tests.test_gpu_train import DT, inputs, rel2

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("table_std", [0.3, 4.0])
def test_softmax_sums_do_not_depend_on_earlier_calls(samrs, cuda, table_std):
    """A bf16 64 x 64 layer whose table makes the single-pass kernel hand most blocks on: the library's choice of the
    exact kernel for such a layer, by its table's address, is neither read nor fed by the call with sums."""
    h = w = 64
    hd = 64
    q, kt, v, t, _ = inputs(h, w, 2, hd, "bf16", cuda, table_std=table_std)
    samrs.global_policy(t, reset=True)
    first = samrs.attention_relpos_lse(q, kt, v, t, h, w, hd ** -0.5)
    for _ in range(40):
        again = samrs.attention_relpos_lse(q, kt, v, t, h, w, hd ** -0.5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert samrs.global_policy(t) == (-1.0, False)
    for _ in range(3):  # the layer's own history, of the call without sums
        samrs.attention_relpos(q, kt, v, t, h, w, hd ** -0.5)
        torch.cuda.synchronize()
        again = samrs.attention_relpos_lse(q, kt, v, t, h, w, hd ** -0.5)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert samrs.global_policy(t, reset=False)[0] >= 0


def test_train_block_repeats_itself(samrs, cuda):
    """A global bf16 block with large tables, made anew by every step: equal inputs, equal bits, at any step."""
    g = torch.Generator(device=cuda).manual_seed(3)
    dim, side = 64, 64
    shapes = {"norm1_w": (dim,), "norm1_b": (dim,), "qkv_w": (3 * dim, dim), "qkv_b": (3 * dim,), "proj_w": (dim, dim),
              "proj_b": (dim,), "rel_pos_h": (2 * side - 1, dim), "rel_pos_w": (2 * side - 1, dim), "norm2_w": (dim,),
              "norm2_b": (dim,), "lin1_w": (4 * dim, dim), "lin1_b": (4 * dim,), "lin2_w": (dim, 4 * dim), "lin2_b": (dim,)}
    params = {k: (torch.randn(*s, generator=g, device=cuda) * (4.0 if k.startswith("rel") else 0.2)).bfloat16()
              for k, s in shapes.items()}
    blk = samrs.train.TrainBlock(params, 1, 0)
    x = torch.randn(1, side, side, dim, generator=g, device=cuda).bfloat16()
    up = torch.randn(1, side, side, dim, generator=g, device=cuda).bfloat16()
    samrs.global_policy(x, reset=True)
    steps = []
    for _ in range(6):
        blk.zero_grad(set_to_none=True)
        y = blk(x)
        y.backward(up)
        torch.cuda.synchronize()
        steps.append([y.detach()] + [p.grad for p in blk.parameters()])
    for s in steps[1:]:
        assert all(torch.equal(a, b) for a, b in zip(steps[0], s))


@pytest.mark.parametrize("dt,tol", [("f32", 1e-5), ("bf16", 4e-3)])
@pytest.mark.parametrize("std", [1e-12, 1e-14, 1e-17])
@pytest.mark.parametrize("rows,c", [(5, 768), (4, 777), (9, 100), (3, 2056), (2, 14337)])
def test_layer_norm_bwd_of_rows_of_tiny_deviation(samrs, cuda, rows, c, dt, tol, std):
    """eps = 0 and a rstd of 1e12 to 1e17, whose cube (and at last its square times a mean) f32 does not hold: the gradients
    are finite. Bounds as for ordinary rows: every step's error is relative."""
    g = torch.Generator(device=cuda).manual_seed(rows + c)
    x = (torch.randn(rows, c, generator=g, device=cuda) * std).to(DT[dt])
    dy, wt = torch.randn(rows, c, generator=g, device=cuda).to(DT[dt]), torch.randn(c, generator=g, device=cuda).to(DT[dt])
    got = samrs.layer_norm_bwd(dy, x, wt, 0.0)
    want = ref.layer_norm_bwd(dy.double(), x.double(), wt.double(), 0.0)
    for a, b in zip(got, want):
        assert bool(torch.isfinite(a).all()) and rel2(a, b) < tol


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", [256, 512, 768, 1024, 1280, 1536, 2048, 2056, 5120, 9600, 10240, 14336])
@pytest.mark.parametrize("res", [False, True])
def test_aligned_norm_rows_take_the_vector_kernel(samrs, cuda, c, dt, res):
    """Rows of a multiple of 16 bytes come through the ring of shared memory at every width that the kernel takes, however
    few of them two stages hold; their gradients are the formulas'."""
    rows = 300
    g = torch.Generator(device=cuda).manual_seed(c)
    x, dy, dres = (torch.randn(rows, c, generator=g, device=cuda).to(DT[dt]) for _ in range(3))
    wt = torch.randn(c, generator=g, device=cuda).to(DT[dt])
    call = lambda: samrs.layer_norm_bwd(dy, x, wt, 1e-3, dres=dres if res else None)  # noqa: E731
    call()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        got = call()
        torch.cuda.synchronize()
    names = [e.key for e in p.key_averages() if "ln_bwd_kernel" in e.key]
    assert len(names) == 1 and f", {4 if dt == 'f32' else 8}, " in names[0], names
    want = ref.layer_norm_bwd(dy.double(), x.double(), wt.double(), 1e-3, dres.double() if res else None)
    for a, b in zip(got, want):
        # one rounding of the result; f32 sums of `rows` terms
        assert rel2(a, b) < {"f32": 1e-5, "f16": 6e-4, "bf16": 4e-3}[dt]
    assert all(torch.equal(a, b) for a, b in zip(got, call()))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,c", [(1, 14337), (3, 14337), (40, 20000), (700, 14344), (9, 65536), (2, 100003)])
@pytest.mark.parametrize("res", [False, True])
def test_layer_norm_bwd_of_very_wide_rows(samrs, cuda, rows, c, dt, res):
    """Rows past the widest that a warp group holds: one kernel for dx and the rows' statistics, one for the column sums."""
    g = torch.Generator(device=cuda).manual_seed(rows + c)
    x, dy, dres = ((torch.randn(rows, c, generator=g, device=cuda) * s + m).to(DT[dt]) for s, m in ((2, .5), (1, 0), (1, 0)))
    wt = torch.randn(c, generator=g, device=cuda).to(DT[dt])
    call = lambda: samrs.layer_norm_bwd(dy, x, wt, 1e-3, dres=dres if res else None)  # noqa: E731
    got = call()
    assert samrs.device_status() == 0
    want = ref.layer_norm_bwd(dy.double(), x.double(), wt.double(), 1e-3, dres.double() if res else None)
    for a, b in zip(got, want):
        # one rounding of the result; f32 sums of `rows` terms, and of c terms by 256 threads
        assert a.dtype == DT[dt] and rel2(a, b) < {"f32": 1e-5, "f16": 6e-4, "bf16": 4e-3}[dt]
    assert all(torch.equal(a, b) for a, b in zip(got, call()))


@pytest.mark.parametrize("dt,tol", [("bf16", 2.4e-3), ("f16", 3.0e-4)])
@pytest.mark.parametrize("h,w,bh,hd", [(64, 64, 4, 80), (64, 64, 4, 64), (33, 33, 12, 64), (50, 41, 6, 96)])
def test_the_table_gradient_is_rounded_twice_at_most(samrs, cuda, h, w, bh, hd, dt, tol):
    """dtable on large grids: dS is rounded as an operand and the result once, independent errors of 1.65e-3 (bf16) or
    2.07e-4 (f16) rms each: 2.34e-3 and 2.93e-4 together. The sums of dS between them (the bias gradients) are not rounded
    again, which would make it 2.86e-3 and 3.59e-4."""
    q, kt, v, t, dout = inputs(h, w, bh, hd, dt, cuda, table_std=0.1, dout_std=0.05)
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, hd ** -0.5)
    got = samrs.attention_relpos_bwd(dout, q, kt, v, t, out, lse, h, w, hd ** -0.5, impl="tc")
    want = ref.attention_bwd_by_heads(dout, q, kt, v, t, h, w, hd ** -0.5, heads=1)
    assert rel2(got[3], want[3]) < tol
