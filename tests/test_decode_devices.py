"""A call goes to the device of its tensors, whichever is current (CPU: the device calls are replaced)."""
from types import SimpleNamespace

import pytest

from leanstream_amd import _native, decode


@pytest.fixture
def devices(monkeypatch):
    """Two devices, of which `now` is current, and the launches as (device, stream)."""
    torch = pytest.importorskip("torch")
    state = SimpleNamespace(now=0, launches=[])

    class On:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, state.now = state.now, self.index

        def __exit__(self, *_):
            state.now = self.before

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state.now, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 * index, raising=False)
    state.tensor = lambda index: SimpleNamespace(device=torch.device("cuda", index))
    return state


def bound(devices, index, code=0):
    call = decode._Call()
    call._bind("block_norm", _native.BlockNorm(), (devices.tensor(index), None))
    call._enqueue = lambda arg, stream: devices.launches.append((devices.now, stream)) or code
    return call


def test_a_call_is_put_on_its_tensors_device(devices):
    for index in (0, 1):
        call = bound(devices, index)
        for devices.now in (0, 1):
            current = devices.now
            call.enqueue()
            call.enqueue(77)
            assert devices.launches[-2:] == [(index, 1000 * index), (index, 77)]
            assert devices.now == current


def test_an_error_leaves_the_current_device_as_it_was(devices):
    call = bound(devices, 1, code=22)
    with pytest.raises(RuntimeError, match="block_norm failed: 22"):
        call.enqueue()
    assert devices.now == 0


def test_tensors_of_two_devices_are_refused(devices):
    call = decode._Call()
    with pytest.raises(ValueError, match="more than one device"):
        call._bind("block_norm", _native.BlockNorm(), (devices.tensor(0), devices.tensor(1)))
