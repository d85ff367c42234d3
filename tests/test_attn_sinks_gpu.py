"""Sinks at the ends of f32, on the GPU: the largest takes all the weight, the lowest and minus infinity none."""
import pytest
import torch

from hipster_amd import qmm
from test_attn_gpu import attend, ints, rows

pytestmark = pytest.mark.gpu
MAX = torch.finfo(torch.float32).max


def check(out, none, Hq):
    """Heads in turn: the largest sink, the lowest, minus infinity, plus infinity and NaN."""
    out, none = out.view(-1, Hq, out.shape[-1] // Hq), none.view(-1, Hq, none.shape[-1] // Hq)
    assert (out[:, 0] == 0).all()
    assert torch.equal(out[:, 1:3], none[:, 1:3])                               # the bits of a call without sinks
    assert out[:, 3:].isnan().all()


def sinks():
    return torch.tensor([MAX, -MAX, -float("inf"), float("inf"), float("nan")], device="cuda")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt", ["bf16", "f32"])
@pytest.mark.parametrize("max_len", [300, 3000])
def test_attend(gpu, D, qt, max_len):
    g = torch.Generator().manual_seed(D)
    lens, ms, Hq, Hk = [300, 40], [3, 1], 5, 1
    none, kv, table, q, _ = attend(g, lens, ms, Hq, Hk, D, 32, qt, qt, max_len=max_len, extra=0)
    out, *_ = attend(g, lens, ms, Hq, Hk, D, 32, qt, qt, 0, sinks(), max_len=max_len, kv=kv, table=table, q=q, extra=0)
    check(out, none, Hq)
    lost, *_ = attend(g, [2], [4], Hq, Hk, D, 32, qt, qt, 0, sinks(), max_len=max_len, kv=kv, table=table[:1], q=q, extra=0)
    assert (lost[:2].view(2, Hq, D)[:, :3] == 0).all()                          # rows that see no key


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("m,n", [(70, 70), (40, 5000)])
def test_prompt(gpu, D, m, n):
    g = torch.Generator().manual_seed(D + n)
    q, k, v = rows(g, m, 5, D, "bf16"), rows(g, n, 1, D, "bf16"), rows(g, n, 1, D, "bf16")
    out = [torch.empty((m, 5 * D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for o, s in zip(out, (sinks(), None)):
        qmm.attn_prompt_bf16(q, k, v, ints([0, m]), ints([0, n]), o, 5, 1, D, sinks=s)
    check(*out, 5)
