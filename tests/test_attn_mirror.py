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


# ---- host tensors, one argument at a time ----
BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def on_host(n, dtype=BF, rows=None):
    return torch.zeros((n,) if rows is None else (rows, n), dtype=dtype)


def kv_call(f, **kw):
    a = dict(k=Rows(3, 128), v=Rows(3, 128), cu=OnDevice(3, I32), lens=OnDevice(2, I32), table=Rows(2, 4, I32), q=Rows(3, 256), out=Rows(3, 256), ws=None,
             sinks=None) | {x: v for x, v in kw.items() if not x.startswith("kv.")}
    kv = cache(**{x[3:]: v for x, v in kw.items() if x.startswith("kv.")})
    if f == "write":
        qmm.kv_write_mxfp4(a["k"], a["v"], kv, a["cu"], a["lens"], a["table"], 3)
    elif f == "read":
        qmm.kv_read_mxfp4(kv, a["cu"], a["lens"], a["table"], a["k"], a["v"], 3)
    else:
        qmm.attn_kv_mxfp4(a["q"], kv, a["cu"], a["lens"], a["table"], a["out"], 3, 4, 2, 64, a["ws"], sinks=a["sinks"])


SEQ = {"cu": on_host(3, I32), "lens": on_host(2, I32), "table": on_host(4, I32, 2)}
KV = {"kv.kq": on_host(4096, U8), "kv.ke": on_host(256, U8), "kv.vq": on_host(4096, U8), "kv.ve": on_host(256, U8)}
KVROWS = {"k": on_host(128, BF, 3), "v": on_host(128, BF, 3)}


@pytest.mark.parametrize("f,name,t", [(f, n, t) for f, m in (("write", KVROWS), ("read", KVROWS), ("attend", {
    "q": on_host(256, BF, 3), "out": on_host(256, BF, 3), "ws": on_host(64, U8), "sinks": on_host(4, F32)})) for n, t in (SEQ | KV | m).items()])
def test_host_tensors_of_the_cache_calls(launched, f, name, t):  # noqa: F811
    kv_call(f)
    assert len(launched) == 1
    with pytest.raises(QmmError, match=name + " must be a CUDA tensor"):
        kv_call(f, **{name: t})
    assert len(launched) == 1


def prompt_call(**kw):
    a = dict(q=Rows(3, 256), k=Rows(3, 128), v=Rows(3, 128), cu_q=OnDevice(3, I32), cu_k=OnDevice(3, I32), out=Rows(3, 256), sinks=None, ws=False) | kw
    qmm.attn_prompt_bf16(a["q"], a["k"], a["v"], a["cu_q"], a["cu_k"], a["out"], 4, 2, 64, sinks=a["sinks"], ws=a["ws"])


def rope_call(**kw):
    a = dict(x=Rows(3, 256), out=Rows(3, 256), pos=Rows(3, 3, I32), freq=OnDevice(16, F32), axis=OnDevice(16, U8)) | kw
    qmm.rope_axes(a["x"], a["out"], a["pos"], a["freq"], a["axis"], 3, 4, 64)


@pytest.mark.parametrize("f,name,t", [(prompt_call, n, t) for n, t in {
    "q": on_host(256, BF, 3), "k": on_host(128, BF, 3), "v": on_host(128, BF, 3), "out": on_host(256, BF, 3), "cu_q": on_host(3, I32), "cu_k": on_host(3, I32),
    "sinks": on_host(4, F32), "ws": on_host(64, U8)}.items()] + [(rope_call, n, t) for n, t in {
        "x": on_host(256, BF, 3), "out": on_host(256, BF, 3), "pos": on_host(3, I32, 3), "freq": on_host(16, F32), "axis": on_host(16, U8)}.items()])
def test_host_tensors_of_prompt_and_rope(launched, f, name, t):  # noqa: F811
    f()
    assert len(launched) == 1
    with pytest.raises(QmmError, match=name + " must be a CUDA tensor"):
        f(**{name: t})
    assert len(launched) == 1
