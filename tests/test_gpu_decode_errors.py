"""An error that another HIP call of the thread left is not taken for one of a decode-step operator, nor taken away."""
import ctypes as C

import pytest

from test_zzz_gpu_decode_streams import bits, calls, same, spoil

pytestmark = pytest.mark.gpu


def hip():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as maps:
        path = next(line.split()[-1] for line in maps if "libamdhip64" in line)
    return C.CDLL(path)


def test_errors_of_other_calls(torch_gpu):
    torch = torch_gpu
    runtime = hip()
    for name, call, outputs, _ in calls(torch):
        print("case:", name, flush=True)
        spoil(outputs)      # append leaves most pages as they are
        call.enqueue()
        torch.cuda.synchronize()
        want = bits(outputs)
        spoil(outputs)
        torch.cuda.synchronize()
        code = runtime.hipSetDevice(1000)        # no such device: an error and nothing else
        assert code != 0
        try:
            call.enqueue()
        finally:
            left = runtime.hipGetLastError()
        torch.cuda.synchronize()
        assert left == code
        assert same(bits(outputs), want), name
