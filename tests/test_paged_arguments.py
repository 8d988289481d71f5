"""Arguments of the paged calls that need no GPU: where memory is made, and what is refused."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from test_paged_host import BF16, F32, _Stream, _c, _config, _decode_args


class _Sized:
    """The one entry point that scratch() calls, answering 4096 bytes."""

    @staticmethod
    def x17ai_b200_paged_scratch_bytes(stream, cfg, batch, n_tokens, out):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_size_t))[0] = 4096
        return None


def test_scratch_is_on_the_streams_device(lib, monkeypatch):
    """The device that the bytes were asked for, not the current one."""
    from x17ai_b200 import device as D, kernels as K
    made = []
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: made.append((n, dtype, torch.device(device))))
    kern = K.PagedAttnKernel(_config())
    kern._lib = _Sized
    opened = D.CudaStream.__new__(D.CudaStream)   # as the library opens one on device 3
    opened.handle, opened.device_id, opened._open = 1 << 40, 3, False
    torchs = D.TorchStream(SimpleNamespace(cuda_stream=1 << 40, device=torch.device("cuda", 2)))
    kern.scratch(opened, 16, 4)
    kern.scratch(torchs, 16, 4)
    kern.scratch(torchs, 16, 4, device="cuda:1")   # as asked for
    assert made == [(4096, torch.uint8, torch.device("cuda", i)) for i in (3, 2, 1)]


@pytest.mark.parametrize("window", [-16, -1, 24, (1 << 64) + 16])
def test_decode_refuses_windows(lib, window):
    from x17ai_b200 import X17Error, kernels as K
    kern = K.PagedAttnKernel(_config())
    for call, args in ((kern.decode, _decode_args()),
                       (kern.decode_scaled, _decode_args(q_scale=_c(F32, 6, 8), page_scales=_c(F32, 9, 2, 16, 2), out=_c(BF16, 6, 512)))):
        with pytest.raises(X17Error, match=f"window_size must be zero or divisible by 16, got {window}"):
            call(_Stream(), **args, window_size=window)
