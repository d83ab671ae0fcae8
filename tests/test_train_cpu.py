"""The training operators without a GPU: their formulas against differences, and the C entry points' refusals."""
import ctypes

import pytest

from tests import train_reference as ref
from tests.conftest import load_samrs

torch = pytest.importorskip("torch")


def lib():
    return load_samrs()._abi.lib()


@pytest.mark.parametrize("h,w,hd", [(1, 1, 3), (2, 3, 4), (4, 2, 5)])
def test_attention_formulas_match_differences(h, w, hd):
    g = torch.Generator().manual_seed(h * 10 + w)
    n, scale = h * w, 0.7
    shapes = [(2, n, hd), (2, hd, n), (2, n, hd), (2 * h + 2 * w - 2, hd)]
    args = [torch.randn(*s, generator=g, dtype=torch.float64) for s in shapes]
    dout = torch.randn(2, n, hd, generator=g, dtype=torch.float64)
    grads = ref.attention_bwd(dout, *args, h, w, scale)
    eps = 1e-6
    for k, (a, grad) in enumerate(zip(args, grads)):
        flat = a.view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 17)):
            vals = []
            for s in (eps, -eps):
                moved = [t.clone() for t in args]
                moved[k].view(-1)[i] += s
                vals.append(float((ref.attention(*moved, h, w, scale)[0] * dout).sum()))
            # central difference: O(eps^2) = 1e-12 of truncation, 1e-16 / eps = 1e-10 of rounding
            assert abs((vals[0] - vals[1]) / (2 * eps) - float(grad.view(-1)[i])) < 1e-7


@pytest.mark.parametrize("c", [1, 2, 7])
def test_layer_norm_formulas_match_differences(c):
    g = torch.Generator().manual_seed(c)
    x, dy, dres = (torch.randn(3, c, generator=g, dtype=torch.float64) for _ in range(3))
    wt, b = torch.randn(c, generator=g, dtype=torch.float64), torch.randn(c, generator=g, dtype=torch.float64)

    def loss(x, wt, b):
        y = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-3) * wt + b
        return float((y * dy).sum() + (x * dres).sum())

    grads = ref.layer_norm_bwd(dy, x, wt, 1e-3, dres)
    for k, grad in enumerate(grads):
        for i in range(grad.numel()):
            vals = []
            for s in (1e-6, -1e-6):
                moved = [t.clone() for t in (x, wt, b)]
                moved[k].view(-1)[i] += s
                vals.append(loss(*moved))
            assert abs((vals[0] - vals[1]) / 2e-6 - float(grad.view(-1)[i])) < 1e-7


@pytest.mark.parametrize("args,code", [(dict(dtype=9), -1), (dict(bh=-1), -1), (dict(h=0), -2), (dict(w=129), -2),
                                       (dict(hd=0), -2), (dict(hd=129), -2)])
def test_attention_bwd_rejects_bad_shapes(args, code):
    p = dict(bh=1, h=4, w=4, hd=8, dtype=0)
    p.update(args)
    shape = (p["bh"], p["h"], p["w"], p["hd"])
    assert lib().samrs_relpos_attn_bwd_workspace(*shape, p["dtype"]) == code
    assert lib().samrs_last_error()
    assert lib().samrs_relpos_attn_bwd(*[None] * 12, 0, *shape, 0.5, p["dtype"], 0, None) == code


def test_attention_bwd_rejects_bad_pointers_and_workspaces():
    l = lib()
    need = l.samrs_relpos_attn_bwd_workspace(2, 4, 4, 8, 0)
    assert need > 0 and l.samrs_relpos_attn_bwd_workspace(0, 4, 4, 8, 0) == 0
    p = 1 << 20  # an address that is never read: every call below returns before a launch

    def call(ptrs=None, ws=p, ws_bytes=need, impl=0, lse=p):
        a = [p] * 11
        for i, v in (ptrs or {}).items():
            a[i] = v
        a[6] = lse
        return l.samrs_relpos_attn_bwd(*a, ws, ws_bytes, 2, 4, 4, 8, 0.5, 0, impl, None)

    for i in range(11):
        assert call({i: None}, lse=None if i == 6 else p) == -1
        assert call({i: p + 1}, lse=p + 1 if i == 6 else p) == -1
    assert call(ws=None) == -1 and call(ws=p + 128) == -1 and call(ws_bytes=need - 1) == -1
    assert call(impl=7) == -1


def test_workspace_is_bounded_for_large_batches():
    small = lib().samrs_relpos_attn_bwd_workspace(64, 64, 64, 80, 2)
    assert lib().samrs_relpos_attn_bwd_workspace(1 << 20, 64, 64, 80, 2) < 8 * small < 8 << 30


def test_layer_norm_bwd_rejects_bad_arguments():
    l = lib()
    p = 1 << 20
    need = l.samrs_layer_norm_bwd_workspace(5, 8)
    assert need > 0 and l.samrs_layer_norm_bwd_workspace(-1, 8) == -1 and l.samrs_layer_norm_bwd_workspace(5, 0) == -1

    def call(dy=p, x=p, wt=p, dres=p, dx=p, dw=p, db=p, ws=p, n=need, rows=5, c=8, eps=1e-6, dtype=0):
        return l.samrs_layer_norm_bwd(dy, x, wt, dres, dx, dw, db, ws, n, rows, c, eps, dtype, None)

    for bad in (dict(dy=None), dict(x=None), dict(wt=None), dict(dx=None), dict(dw=None), dict(db=None), dict(ws=None),
                dict(dy=p + 2), dict(dres=p + 2), dict(dw=p + 1), dict(ws=p + 8), dict(n=need - 1), dict(rows=-1), dict(c=0),
                dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=3)):
        assert call(**bad) == -1, bad


def test_clip_grad_norm_rejects_bad_arguments():
    l = lib()
    p = 1 << 20
    assert l.samrs_clip_grad_norm_workspace(-1) == -1
    need = l.samrs_clip_grad_norm_workspace(2)

    def call(src=(p, p), dst=(p, p), numel=(4, 0), types=(0, 0), out_types=(0, 0), count=2, most=1.0, norm=p, ws=p, n=need):
        arrays = [(ctypes.c_void_p * 2)(*src), (ctypes.c_void_p * 2)(*dst), (ctypes.c_int64 * 2)(*numel),
                  (ctypes.c_int * 2)(*types), (ctypes.c_int * 2)(*out_types)]
        return l.samrs_clip_grad_norm(*(ctypes.addressof(a) for a in arrays), count, most, norm, ws, n, None)

    for bad in (dict(src=(None, p)), dict(dst=(p + 2, p)), dict(numel=(-1, 0)), dict(types=(3, 0)), dict(out_types=(0, -1)),
                dict(out_types=(2, 0)), dict(count=-1), dict(most=-1.0), dict(most=float("nan")), dict(norm=None),
                dict(norm=p + 2), dict(ws=None), dict(n=need - 1)):
        assert call(**bad) == -1, bad
    assert l.samrs_clip_grad_norm(None, None, None, None, None, 2, 1.0, p, p, need, None) == -1


def test_python_entry_points_refuse_host_tensors_and_mismatches():
    s = load_samrs()
    q, kt, t = torch.zeros(2, 6, 4), torch.zeros(2, 4, 6), torch.zeros(8, 4)
    with pytest.raises(s.SamrsError):
        s.attention_relpos_lse(q, kt, q, t, 2, 3, 0.5)
    with pytest.raises(s.SamrsError):
        s.attention_relpos_bwd(q, q, kt, q, t, q, torch.zeros(2, 6), 2, 3, 0.5)
    with pytest.raises(s.SamrsError):
        s.layer_norm_bwd(q, q, torch.ones(4))
    with pytest.raises(s.SamrsError):
        s.clip_grad_norm([], 1.0)
    with pytest.raises(s.SamrsError):
        s.clip_grad_norm([q], 1.0)
