"""What the Python mirror of attention's operators looks at in every call, on stand-ins for device tensors.  No call below reaches a device."""
import pytest
import torch

from hipster_amd import qmm
from hipster_amd._lib import QmmError
from test_attn_edges import Rows, cache
from test_mx_edges import OnDevice, launched  # noqa: F401

I32 = torch.int32


@pytest.mark.parametrize("name", ["kq", "ke", "vq", "ve"])
def test_a_cache_tensor_turned_in_place_is_refused(launched, name):  # noqa: F811
    """A tensor of a cache that a call has checked, transposed in place: the same address and count, other places."""
    kv = cache()
    rows, cu, lens, table = Rows(3, 128), OnDevice(3, I32), OnDevice(2, I32), Rows(2, 4, I32)
    f = lambda: qmm.kv_write_mxfp4(rows, rows, kv, cu, lens, table, 3)       # noqa: E731
    f()
    getattr(kv, name).is_contiguous = lambda: False
    with pytest.raises(QmmError, match="kv." + name):
        f()
    assert len(launched) == 1
    getattr(kv, name).is_contiguous = lambda: True
    f()
    assert len(launched) == 2
