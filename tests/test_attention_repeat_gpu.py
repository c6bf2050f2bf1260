"""The load-balanced flash attention gives the same bits whatever the timing of its CTAs (GPU).

A query block cut between CTAs is merged by the one that finishes last, from the workspace or, for the
block's first piece, partly from tensor memory: both ways are the same arithmetic."""
import ctypes

import pytest
import torch

from dollama_b200 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,Sq,Sk", [(2, 10, 1024, 1024), (2, 20, 256, 256), (1, 5, 700, 900)])
def test_stream_k_attention_repeats_to_the_bit(B, H, Sq, Sk):
    g = torch.Generator(device="cuda").manual_seed(B + H + Sq)
    q, k, v = (torch.randn(B, H, n, 64, generator=g, device="cuda").half() for n in (Sq, Sk, Sk))
    n = int(L.lib().dlm_attention_workspace_bytes(B, H, Sq))
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    outs = torch.empty(16, B, H, Sq, 64, device="cuda", dtype=torch.half)
    busy = torch.randn(3000, 3000, device="cuda").half()
    side = torch.cuda.Stream()
    s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    first = None
    for i in range(60):
        # alone first; then beside products that hold some of the SMs for some of the time
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for j in range(6 if i else 0):
                busy[:200 + 350 * ((i + j) % 8)] @ busy
        for o in outs:
            L.call("dlm_launch_attention_ws", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B, H, Sq, Sk, 64,
                   0.125, ws.data_ptr(), n, s)
        if first is None:
            first = outs[0].clone()
        differ += (outs != first).flatten(1).any(1).sum()
    torch.cuda.synchronize()
    assert int(differ) == 0
