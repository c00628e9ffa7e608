"""The Python layer of the K/V cache: what it hands to the library, and what it refuses (no GPU needed: nothing here is launched)."""
import pytest


class Factors:
    """Looks like an f32 tensor on a GPU."""

    def __init__(self, n, ptr, device=0):
        import torch

        self.dtype, self.shape, self.ptr, self.device_index = torch.float32, (n,), ptr, device
        self.is_cuda = True

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return self.device_index


def test_a_rotation_is_what_was_last_assigned_to_it(capi):
    rope = capi.Rope(10000.0, factors=Factors(64, 4096))

    def now(head_dim=128):
        s = rope.ref(head_dim)._obj
        return s.base, s.dims, s.style, s.factors

    assert now() == (10000.0, 128, 0, 4096) and now(64) == (10000.0, 64, 0, 4096)
    assert rope.ref(128) is rope.ref(128)  # made once
    rope.base = 5e5
    assert now() == (5e5, 128, 0, 4096)
    rope.factors = Factors(64, 8192)
    assert now() == (5e5, 128, 0, 8192) and now(64) == (5e5, 64, 0, 8192)
    rope.dims, rope.style = 32, "halves"
    assert now() == (5e5, 32, 1, 8192)
    rope.factors = None
    assert now() == (5e5, 32, 1, None)
    rope.factors = Factors(15, 8192)
    with pytest.raises(capi.NhbError):
        rope.ref(128)
    rope.factors, rope.style = None, "spiral"
    with pytest.raises(capi.NhbError):
        rope.ref(128)
