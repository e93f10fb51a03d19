"""Stream handles that are numbers and no streams: hipStreamLegacy (1) and hipStreamPerThread (2)."""
import numpy as np
import pytest

import decoder_plain as R
import test_decoder_refusals as calls
from ppocr_native_amd import GpuError, decoder as D
from ppocr_native_amd.devmem import synchronize


@pytest.mark.parametrize("call", [calls.norm, calls.product, calls.append, calls.paged, calls.prompt])
def test_the_legacy_handle_is_refused(call):
    with pytest.raises(GpuError, match="handle"):
        call(stream=1)


@pytest.mark.gpu
def test_the_threads_own_stream():
    rng = np.random.default_rng(1)
    x, w = R.stored(rng.normal(0, 1, (40, 96)), D.BF16), R.stored(rng.normal(1, 0.1, 96), D.BF16)
    dx, dw, dy = R.on_gpu(x), R.on_gpu(w), R.on_gpu(np.zeros((40, 96), np.uint16))
    print("the thread's own stream", flush=True)
    D.rms_norm(dx.addr, dw.addr, dy.addr, 40, 96, type=D.BF16, stream=2)
    synchronize()
    _, want = R.norm(R.values(x, D.BF16), None, R.values(w, D.BF16), D.BF16, 1e-6)
    R.close(R.values(R.back(dy, np.uint16, (40, 96)), D.BF16), want,
            R.half_step(want, D.BF16) + np.abs(want) * 12 * R.STEP)
