"""fft_quad_kernel's claimed rounds where the numbers do not divide (cyberether_amd/csrc/kernels/fft_quad.hh): spans whose transform
count is no multiple of the 1024 resident workgroups nor of the eight counters, replayed and launched eagerly in turn on the same
counters.  Every value, index-fed bin and ring slot equals fft_pipe_kernel's."""
import numpy as np
import pytest

from test_gpu_chain import tone_batch
from test_gpu_quad_kernel import _run, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,slots", [(1030, 9), (911, 11), (1, 9001)])
def test_ragged_long_launches(js, oracle, switch, b, slots):
    n, h = 4096, 64
    if b == 1:  # many one-row cycles: the claimed rounds cross a cycle's end at every transform
        base = tone_batch(oracle, 64, n, 5)
        xs = [base[s % 64:s % 64 + 1] * np.float32(0.4 + 0.01 * (s % 50)) for s in range(slots)]
        calls = (1, slots)
    else:
        base = tone_batch(oracle, b, n, 5)
        xs = [np.roll(base, 13 * s, axis=0) * np.float32(0.4 + 0.05 * s) for s in range(slots)]
        calls = (1, slots, 2 * slots + 3, slots)
    pipe = _run(js, xs, h, calls, switch, kernel="pipe")
    quad = _run(js, xs, h, calls, switch)
    _same(pipe, quad, f"claimed rounds, {b} x {slots} transforms")
