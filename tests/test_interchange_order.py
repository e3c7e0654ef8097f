"""Arrays handed over between torch and libkk without a word about streams:
neither reads what the other has not written yet, nor writes what the other
has still to read (torch's stream is not libkk's, so that only an order
between the two makes these hold)."""
import numpy as np
import pytest
import torch

from conftest import load_pkg

N = 1 << 25  # (each step takes the GPU longer than the host needs to give it out)


class _Array:
    __cuda_array_interface__ = dict(shape=(2, 3), typestr="<f4", data=(1 << 20, False), version=2)


def test_arrays_of_no_library_and_no_stream_need_no_gpu():
    t = load_pkg().DeviceTensor.from_array(_Array())
    del t


def long_work(x, steps=100):
    """Some milliseconds of torch's current stream that end with x + steps in x."""
    for _ in range(steps):
        x += 1


def long_work_kk(kk, steps=100):
    y, one = kk.ops.fill((N,), 0), kk.to_device(np.float32(1))
    for _ in range(steps):
        y = kk.ops.binary("Add", y, one)
    return y


@pytest.fixture
def warm(gpu):
    """The pool holds what the tests ask it for: a new allocation would wait for the whole GPU."""
    y = long_work_kk(gpu, 2)
    spare = [gpu.DeviceTensor.empty((N,)) for _ in range(3)]
    del y, spare
    gpu.sync()
    yield gpu
    gpu.pool_trim(0)


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
def test_what_torch_has_still_to_write_is_waited_for(warm, side):
    kk = warm
    s = torch.cuda.Stream() if side else torch.cuda.current_stream()
    x = torch.zeros(N, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        long_work(x)
        t = kk.DeviceTensor.from_array(x)
        got = kk.to_host(kk.ops.binary("Add", t, kk.to_device(np.float32(1))))
    assert (got == 101).all()


@pytest.mark.gpu
def test_memory_given_back_to_torch_is_read_before_it_is_written(warm):
    kk = warm
    x = torch.full((N,), 7.0, device="cuda")
    torch.cuda.synchronize()
    ptr = x.data_ptr()
    t = kk.DeviceTensor.from_array(x)
    busy = long_work_kk(kk)
    y = kk.ops.binary("Add", busy, t)
    del t, x
    z = torch.full((N,), -1.0, device="cuda")
    assert z.data_ptr() == ptr  # (torch's allocator hands the same memory out)
    assert (kk.to_host(y) == 107).all() and bool((z == -1).all())


@pytest.mark.gpu
def test_arrays_may_be_taken_and_dropped_while_recording(gpu):
    kk = gpu
    x = torch.ones(8, device="cuda")
    kk._lib.call("kk_graph_begin")
    try:
        t = kk.DeviceTensor.from_array(x)
        del t
    finally:
        kk._lib.call("kk_graph_abort")


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
def test_what_libkk_has_still_to_write_is_waited_for(warm, side):
    kk = warm
    s = torch.cuda.Stream() if side else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        z = torch.as_tensor(long_work_kk(kk), device="cuda") + 1
        assert bool((z == 101).all())


@pytest.mark.gpu
def test_memory_lent_to_torch_is_read_before_it_is_written(warm):
    kk = warm
    x = torch.zeros(N, device="cuda")
    t = kk.ops.fill((N,), 7)
    view = torch.as_tensor(t, device="cuda")
    torch.cuda.synchronize()
    long_work(x)
    z = view + x
    ptr = t.ptr
    del t, view
    y = kk.ops.fill((N,), -1)
    assert y.ptr == ptr  # (the pool hands the same memory out)
    assert bool((z == 107).all()) and (kk.to_host(y) == -1).all()


@pytest.mark.gpu
def test_the_interface_names_libkks_stream(gpu):
    kk = gpu
    t = kk.to_device(np.arange(3, dtype=np.float32))
    desc = t.__cuda_array_interface__
    assert desc["version"] == 3 and desc["stream"] > 2
    again = kk.DeviceTensor.from_array(t)  # (a stream does not wait for itself)
    assert kk.to_host(again).tolist() == [0, 1, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
def test_work_on_torchs_stream_is_in_the_order_of_the_calls(warm, side):
    kk = warm
    s = torch.cuda.Stream() if side else torch.cuda.default_stream()
    own = kk.to_device(np.zeros(1, np.float32)).__cuda_array_interface__["stream"]
    one = kk.to_device(np.float32(1))
    x = torch.zeros(N, device="cuda")
    t = kk.DeviceTensor.from_array(x)
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(s):
            kk.use_stream(s.cuda_stream)
            kk.use_stream(s.cuda_stream)
            for i in range(20):
                x += 1
                y = kk.ops.binary("Add", t, one)  # (the same handle: no order but the stream's)
                x.copy_(torch.as_tensor(y, device="cuda"))
            assert t.__cuda_array_interface__["stream"] == (s.cuda_stream or 1)
            assert bool((x == 40).all())
    finally:
        kk.use_stream()
    assert t.__cuda_array_interface__["stream"] == own
    assert (kk.to_host(t) == 40).all()


@pytest.mark.gpu
def test_graphs_on_torchs_default_stream(gpu):
    """Recorded while libkk works on the default stream, which cannot record, and launched there between torch's work."""
    import ctypes
    kk = gpu
    x = torch.zeros(1000, device="cuda")
    t = kk.DeviceTensor.from_array(x)
    y, one = kk.DeviceTensor.empty((1000,)), kk.to_device(np.float32(1))
    g = ctypes.c_int(-1)
    kk.use_stream(torch.cuda.default_stream().cuda_stream)
    try:
        kk._lib.call("kk_graph_begin")
        with pytest.raises(kk._lib.KKError, match="recorded"):
            kk.use_stream()
        kk._lib.call("kk_binary", kk._lib.OP["Add"], y.desc(), t.desc(), one.desc())
        kk._lib.call("kk_graph_end", ctypes.byref(g))
        view = torch.as_tensor(y, device="cuda")
        for i in range(5):
            x += 1
            kk._lib.call("kk_graph_launch", g.value)
            assert bool((view == i + 2).all()), f"replay {i}"
            assert (kk.to_host(kk.ops.binary("Add", y, one)) == i + 3).all()
        kk._lib.call("kk_graph_begin")
        kk._lib.call("kk_graph_abort")
        assert t.__cuda_array_interface__["stream"] == 1
    finally:
        kk.use_stream()
    kk._lib.call("kk_graph_launch", g.value)
    assert (kk.to_host(y) == 6).all()
    kk._lib.call("kk_graph_destroy", g.value)
