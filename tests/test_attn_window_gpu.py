"""Attention of prompts with a window behind many keys, on the GPU: small windows stay one part, and what is cut into parts is right."""
import pytest
import torch

from hipster_amd import qmm
from test_attn_gpu import check_prompt, ints, offsets, rows

pytestmark = pytest.mark.gpu


def call(lens, ms, Hq, Hk, D, window, seed, check=True):
    """A call with a workspace of a known filling and one without: (whether it was written, the two results)."""
    g = torch.Generator().manual_seed(seed)
    aq, ak = offsets(ms), offsets(lens)
    q, k, v = rows(g, aq[-1] + 1, Hq, D, "bf16"), rows(g, ak[-1] + 1, Hk, D, "bf16"), rows(g, ak[-1] + 1, Hk, D, "bf16")
    k[-1], v[-1] = float("nan"), float("nan")                                   # rows of no sequence
    size = qmm.attn_prompt_ws_bytes(aq[-1] + 1, ak[-1] + 1, len(lens), Hq, D)
    assert size > 0                                                             # without a window there are parts
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    out = []
    for w in (ws, False):
        out.append(torch.full((aq[-1] + 1, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda"))
        qmm.attn_prompt_bf16(q, k, v, ints(aq), ints(ak), out[-1], Hq, Hk, D, window=window, ws=w)
        if check:
            check_prompt(out[-1], q, k, v, None, lens, ms, Hq, Hk, D, window)
    return bool((ws != 255).any()), out


@pytest.mark.parametrize("D,window", [(64, 1), (64, 128), (64, 511), (128, 1), (128, 128), (128, 511), (256, 1), (256, 128), (256, 255)])
def test_a_small_window_is_one_part(gpu, D, window):
    """The keys that a tile of rows sees are few however many there are: the workspace stays as it was, the bits are those without one."""
    written, out = call([5000], [130], 4, 2, D, window, window + D)
    assert not written and torch.equal(out[0], out[1])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [512, 700, 2500])
@pytest.mark.parametrize("lens,ms", [([5000], [40]), ([9000, 70, 0, 2600], [33, 70, 4, 129])])
def test_a_larger_window_in_parts(gpu, D, window, lens, ms):
    """Parts of the window's keys, in short sequences parts of no keys at all, joined."""
    written, _ = call(lens, ms, 4, 2, D, window, window + D)
    assert written


def test_a_small_window_needs_no_workspace(gpu):
    """A workspace that would be too small for the keys without a window."""
    q, k = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(9000, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(q)
    assert qmm.attn_prompt_ws_bytes(40, 9000, 1, 1, 64) > 16
    qmm.attn_prompt_bf16(q, k, k, ints([0, 40]), ints([0, 9000]), out, 1, 1, 64, window=64, ws=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert (out == 1).all()
