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
