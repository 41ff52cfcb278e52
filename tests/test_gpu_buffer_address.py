"""The device address of a buffer: another library sees what the context wrote, and the other way round."""

import numpy as np
import pytest
import torch

from yule_b200 import YuleGpuError
from yule_b200.backend import BufferHandle

pytestmark = pytest.mark.gpu


class View:
    def __init__(self, address, count):
        self.__cuda_array_interface__ = {"data": (address, False), "shape": (count,), "typestr": "<f4", "version": 3}


def test_another_library_sees_the_buffer(backend):
    a, b, out = (backend.upload(np.arange(1000, dtype=np.float32)) for _ in range(3))
    backend.synchronize()
    view = torch.as_tensor(View(backend.buffer_address(b), 1000), device="cuda")
    assert view[10].item() == 10
    view.fill_(2.0)
    torch.cuda.synchronize()
    backend.add(a, b, out, 1000)
    assert (backend.download(out, 1000) == np.arange(1000) + 2).all()
    for h in (a, b, out):
        backend.free(h)


def test_unknown_buffers_have_none(backend):
    with pytest.raises(YuleGpuError):
        backend.buffer_address(BufferHandle(1 << 60))
