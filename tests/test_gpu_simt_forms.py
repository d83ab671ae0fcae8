"""The any-shape attention at the edges between its layouts (tiny grids; P over K; P beside K), against the CPU oracle, after
calls that leave NaN in shared memory."""
import pytest

from oracle import oracle
from tests.helpers import F32_TOL, HALF_TOL, make_inputs, parity_err

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TINY = [(1, 1), (1, 9), (9, 1), (2, 3), (3, 3), (4, 6), (5, 5), (7, 3)]
SHAPES = [(h, w, hd) for h, w in TINY for hd in (1, 16, 63, 64, 65, 128)]
SHAPES += [(1, 10, 48), (10, 1, 128), (5, 6, 117), (5, 6, 118), (6, 5, 80),                  # just past them
           (14, 14, 111), (14, 14, 112), (20, 16, 112), (13, 13, 128), (65, 65, 96), (100, 97, 40)]  # P beside / over K


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h,w,hd", SHAPES)
def test_layouts_match_the_oracle(samrs, cuda, h, w, hd, dt):
    tdt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dt]
    bh = 3 if h * w < 2000 else 1
    q, kt, v, t = make_inputs(h, w, bh, hd, seed=100 * h + w + hd, table_std=0.5)
    args = [torch.from_numpy(x).to(cuda).to(tdt) for x in (q, kt, v, t)]
    nan = torch.full((400, 300, 120), float("nan"), device=cuda, dtype=tdt)
    samrs.attention_relpos(nan, nan.transpose(1, 2).contiguous(), nan, torch.ones(78, 120, device=cuda, dtype=tdt), 30, 10, 0.1)
    out, lse = samrs.attention_relpos_lse(*args, h, w, hd ** -0.5)
    plain = samrs.attention_relpos(*args, h, w, hd ** -0.5, impl="simt")
    assert samrs.device_status() == 0
    assert torch.equal(out, plain) and bool(torch.isfinite(lse).all())
    want = oracle.attention_relpos(*(a.float().cpu().numpy() for a in args), h, w, hd ** -0.5)
    assert parity_err(out.float().cpu().numpy(), want, dt) < (F32_TOL if dt == "f32" else HALF_TOL)
