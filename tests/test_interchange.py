"""Device arrays of other libraries: views over their memory and theirs over
ours, and the order of two streams (torch's arrays stand for the others)."""
import numpy as np
import pytest
import torch

from conftest import assert_bitexact, load_pkg


class _Array:
    def __init__(self, **desc):
        self.__cuda_array_interface__ = dict(dict(shape=(2, 3), typestr="<f4", data=(1 << 20, False), version=2),
                                             **desc)


def test_from_array_describes_the_memory():
    kk = load_pkg()
    a = _Array(strides=(24, 8))
    t = kk.DeviceTensor.from_array(a)
    assert (t.ptr, t.shape, t.strides, t.dtype) == (1 << 20, (2, 3), (6, 2), np.float32)
    assert t.storage.owner is a
    back = t.__cuda_array_interface__
    assert back["strides"] == (24, 8) and back["data"] == (1 << 20, False) and back["typestr"] == "<f4"
    assert kk.DeviceTensor.from_array(_Array()).__cuda_array_interface__["strides"] is None
    assert kk.DeviceTensor.from_array(_Array(shape=(0, 3))).__cuda_array_interface__["data"][0] == 0


@pytest.mark.parametrize("bad,error", [(dict(typestr="<f8"), TypeError), (dict(strides=(12, 2)), ValueError),
                                       (dict(mask=1), TypeError), (dict(shape=(1,) * 9), ValueError)])
def test_from_array_refuses(bad, error):
    with pytest.raises(error):
        load_pkg().DeviceTensor.from_array(_Array(**bad))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.int8, torch.int32, torch.int64, torch.bool])
def test_views_both_ways(gpu, dtype):
    kk = gpu
    x = torch.arange(60, device="cuda").reshape(3, 4, 5).to(dtype)
    y = x.transpose(0, 2)[1:, ::2]
    t = kk.DeviceTensor.from_array(y, stream=torch.cuda.current_stream().cuda_stream)
    assert_bitexact(kk.to_host(t), y.cpu().numpy())
    back = torch.as_tensor(t, device="cuda")
    assert back.data_ptr() == y.data_ptr() and back.stride() == y.stride()
    assert torch.equal(back, y)


@pytest.mark.gpu
def test_streams_are_ordered(gpu):
    """A long chain on a stream of torch's, read by libkk, and back."""
    kk = gpu
    s = torch.cuda.Stream()
    x = torch.zeros(1 << 22, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(200):
            x += 1
    t = kk.DeviceTensor.from_array(x, stream=s.cuda_stream)
    y = t
    one = kk.to_device(np.float32(1))
    for _ in range(50):
        y = kk.ops.binary("Add", y, one)
    kk.signal_stream(s.cuda_stream)
    with torch.cuda.stream(s):
        z = torch.as_tensor(y, device="cuda") + 1
    s.synchronize()
    assert bool((z == 251).all())


@pytest.mark.gpu
def test_streams_are_refused_while_recording(gpu):
    kk = gpu
    kk._lib.call("kk_graph_begin")
    try:
        for fn in (kk.wait_stream, kk.signal_stream):
            with pytest.raises(kk._lib.KKError, match="recorded"):
                fn(0)
    finally:
        kk._lib.call("kk_graph_abort")
