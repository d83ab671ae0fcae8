"""Failure detection of the backward kernels on the GPU, without a fault: a bounded wait that runs out, as in
test_gpu_failure. CTA 0 never loads one step; its waits for it run out, every CTA returns once its own copies have landed,
and the library recovers."""
import time

import pytest

from tests.test_gpu_train import inputs

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("withhold", [0, 3, 1000, 1003])  # a step of the dQ kernel, of the dK / dV kernel
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("h,w,bh,hd", [(64, 64, 6, 80), (14, 14, 200, 64), (33, 47, 8, 32)])
def test_a_wait_that_runs_out_in_the_backward_pass(samrs, cuda, h, w, bh, hd, dt, withhold):
    q, kt, v, t, dout = inputs(h, w, bh, hd, dt, cuda)
    scale = hd ** -0.5
    out, lse = samrs.attention_relpos_lse(q, kt, v, t, h, w, scale)
    args = (dout, q, kt, v, t, out, lse, h, w, scale)
    want = samrs.attention_relpos_bwd(*args, impl="tc")
    assert samrs.device_status() == 0
    lib = samrs._abi.lib()
    try:
        samrs._abi.check(lib.samrs_test_hooks(200_000, withhold))  # about 0.1 ms per wait
        t0 = time.perf_counter()
        samrs.attention_relpos_bwd(*args, impl="tc")
        status = samrs.device_status(clear=False)
        elapsed = time.perf_counter() - t0
    finally:
        samrs._abi.check(lib.samrs_test_hooks(0, -1))
    assert status == 1, status  # kStatusWaitTimeout
    assert elapsed < 1.0, elapsed
    with pytest.raises(samrs.SamrsError) as err:
        samrs.attention_relpos_bwd(*args, impl="tc")
    assert err.value.code == samrs._abi.ERR_DEVICE
    assert samrs.device_status(clear=True) == 1
    got = samrs.attention_relpos_bwd(*args, impl="tc")
    assert samrs.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))
