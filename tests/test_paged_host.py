"""Host side of the paged-cache wrappers (no GPU needed)."""

import pytest
import torch

BF, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _aligned(n, dt):
    """A flat buffer of n elements at a 16-byte aligned address."""
    x = torch.arange(n + 16, dtype=torch.float32).to(dt)
    skip = -x.data_ptr() % 16 // x.element_size()
    return x[skip:skip + n]


@pytest.mark.parametrize("dt", [BF, F16, E4M3])
@pytest.mark.parametrize("T,H,D", [(1, 1, 64), (1, 4, 64), (3, 4, 64), (2, 1, 128)])
def test_rows_end_up_aligned(dt, T, H, D):
    from fa4_ring.attn_backend import rows16
    base = _aligned(T * H * D + 16 + 32 * T, dt)
    n = T * H * D
    assert rows16(base[:n].view(T, H, D)).data_ptr() == base.data_ptr()  # taken as it is
    wide = base[:T * (H * D + 32)].view(T, H * D + 32)
    fused = wide[:, 16:16 + H * D].view(T, H, D)
    assert rows16(fused).data_ptr() == fused.data_ptr()
    for x in (base[1:1 + n].view(T, H, D), wide[:, 3:3 + H * D].view(T, H, D),
              base[1:1 + n].view(T, D, H).transpose(1, 2)):
        y = rows16(x)
        assert y.data_ptr() % 16 == 0 and y.is_contiguous()
        assert torch.equal(y.view(torch.uint8), torch.stack(list(x)).contiguous().view(torch.uint8))  # (values may be NaN)


@pytest.mark.parametrize("h_kv", [1, 3])
def test_descales_of_every_form(h_kv):
    from fa4_ring.attn_backend import norm_descale
    dev = torch.device("cpu")
    assert norm_descale(None, h_kv, dev) is None
    for d in (0.3, torch.tensor(0.3), torch.tensor(0.3, dtype=torch.float64, requires_grad=True),
              torch.full((1, h_kv), 0.3), torch.full((h_kv,), 0.3, dtype=torch.float64)):
        got = norm_descale(d, h_kv, dev)
        assert got.dtype == torch.float32 and got.is_contiguous() and not got.requires_grad
        assert got.flatten().tolist() == torch.full((h_kv,), 0.3).tolist()
    for d in (torch.ones(h_kv + 1), torch.ones(1, h_kv + 1)):
        with pytest.raises(AssertionError):
            norm_descale(d, h_kv, dev)
    if h_kv > 1:
        with pytest.raises(AssertionError):  # one entry is not a scalar
            norm_descale(torch.ones(1), h_kv, dev)


def test_launch_stream_and_device_without_the_private_calls(monkeypatch):
    """The stream and the device of a launch come from torch's private calls, which are the cheaper
    ones; a torch without them is served by the public ones."""
    import importlib

    from fa4_ring import _lib

    class Stream:
        def __init__(self, index):
            self.cuda_stream = 1000 + index

    class Tensor:
        def get_device(self):
            return 3

    try:
        with monkeypatch.context() as m:
            m.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
            m.delattr(torch._C, "_cuda_getDevice", raising=False)
            m.setattr(torch.cuda, "current_stream", Stream)
            m.setattr(torch.cuda, "current_device", lambda: 3)
            importlib.reload(_lib)
            assert _lib.stream_of(Tensor()) == 1003
            assert _lib.on_device(torch.device("cuda", 3)) is _lib._no_switch
            assert isinstance(_lib.on_device(torch.device("cuda", 2)), torch.cuda.device)
        with monkeypatch.context() as m:
            m.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 2000 + i, raising=False)
            m.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
            importlib.reload(_lib)
            assert _lib.stream_of(Tensor()) == 2003
            assert _lib.on_device(torch.device("cuda", 1)) is _lib._no_switch
    finally:
        importlib.reload(_lib)
