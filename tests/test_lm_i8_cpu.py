"""Refusals of the int8 language-model operators: every rejected call returns its status and a
message before anything is launched, so no GPU is needed; and the oracle's own rounding rule."""
import ctypes

import numpy as np
import pytest
import torch

from dollama_b200 import _lib as L
from tests import lm_i8_oracle as O

INVALID, UNSUPPORTED = -1, -4
_buf = np.zeros(4096, np.uint8)
A = (_buf.ctypes.data + 255) // 256 * 256  # an aligned address that no refused call reads


def rc(fn, *args):
    return getattr(L.lib(), fn)(*args)


def norm(x=A, ldx=64, r=A, ldr=64, w=A, h=A, ldh=64, q=A, s=A, M=4, K=64, eps=1e-5, t=0):
    return rc("dlm_add_rms_norm_i8", x, ldx, r, ldr, w, h, ldh, q, s, M, K, eps, t, None)


def gemm(xq=A, ldx=64, xs=A, w=A, ws=A, b=None, y=A, ldy=32, M=4, N=32, K=64, t=0):
    return rc("dlm_gemm_i8", xq, ldx, xs, w, ws, b, y, ldy, M, N, K, t, None)


def append(k=A, ldk=128, v=A, ldv=128, kq=A, ks=A, vq=A, vs=A, B=2, S=3, H=2, Dh=64, Lm=16, pos=A, n=None, t=0):
    return rc("dlm_kv_i8_append", k, ldk, v, ldv, kq, ks, vq, vs, B, S, H, Dh, Lm, pos, n, t, None)


def read(k=A, ldk=128, v=A, ldv=128, kq=A, ks=A, vq=A, vs=A, B=2, S=3, H=2, Dh=64, Lm=16, pos=A, n=None, t=0):
    return rc("dlm_kv_i8_read", kq, ks, vq, vs, k, ldk, v, ldv, B, S, H, Dh, Lm, pos, n, t, None)


def attn(q=A, ldq=256, kq=A, ks=A, vq=A, vs=A, o=A, ldo=256, B=2, Hq=4, Hkv=2, Sq=1, Dh=64, Lm=16, n=A, m=None,
         causal=1, scale=0.125, t=0):
    return rc("dlm_attention_kv_i8", q, ldq, kq, ks, vq, vs, o, ldo, B, Hq, Hkv, Sq, Dh, Lm, n, m, causal, scale,
              t, None)


CASES = [
    (norm, dict(x=None), INVALID), (norm, dict(w=None), INVALID), (norm, dict(q=None), INVALID),
    (norm, dict(s=None), INVALID), (norm, dict(M=-1), INVALID), (norm, dict(K=-1), INVALID),
    (norm, dict(t=3), INVALID), (norm, dict(t=-1), INVALID), (norm, dict(ldx=63), INVALID),
    (norm, dict(ldr=63), INVALID), (norm, dict(ldh=63), INVALID), (norm, dict(eps=0.0), INVALID),
    (norm, dict(eps=float("nan")), INVALID), (norm, dict(eps=float("inf")), INVALID),
    (norm, dict(K=32769, ldx=40000, ldr=40000, ldh=40000), UNSUPPORTED), (norm, dict(x=A + 2), INVALID),
    (norm, dict(r=A + 1, t=1), INVALID), (norm, dict(s=A + 2), INVALID),
    (gemm, dict(xq=None), INVALID), (gemm, dict(xs=None), INVALID), (gemm, dict(w=None), INVALID),
    (gemm, dict(ws=None), INVALID), (gemm, dict(y=None), INVALID), (gemm, dict(K=40), INVALID),
    (gemm, dict(ldx=72), INVALID), (gemm, dict(ldx=48), INVALID), (gemm, dict(ldy=31), INVALID),
    (gemm, dict(K=1 << 17, ldx=1 << 17), UNSUPPORTED), (gemm, dict(xq=A + 8), INVALID),
    (gemm, dict(w=A + 1), INVALID), (gemm, dict(y=A + 2), INVALID), (gemm, dict(b=A + 1, t=1), INVALID),
    (gemm, dict(N=-1), INVALID), (gemm, dict(t=7), INVALID),
    *[(f, c, e) for f in (append, read) for c, e in (
        (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(kq=None), INVALID), (dict(ks=None), INVALID),
        (dict(vq=None), INVALID), (dict(vs=None), INVALID), (dict(pos=None), INVALID), (dict(ldk=127), INVALID),
        (dict(ldv=64), INVALID), (dict(ldk=130), INVALID), (dict(k=A + 8), INVALID), (dict(vq=A + 8), INVALID),
        (dict(Dh=96, ldk=256, ldv=256), UNSUPPORTED), (dict(B=-1), INVALID), (dict(S=-2), INVALID),
        (dict(Lm=-1), INVALID), (dict(t=5), INVALID), (dict(ks=A + 2), INVALID), (dict(pos=A + 1), INVALID),
        (dict(n=A + 2), INVALID), (dict(vs=A + 1), INVALID))],
    (attn, dict(q=None), INVALID), (attn, dict(o=None), INVALID), (attn, dict(kq=None), INVALID),
    (attn, dict(vs=None), INVALID), (attn, dict(n=None), INVALID), (attn, dict(Hkv=3), INVALID),
    (attn, dict(Hkv=0), INVALID), (attn, dict(ldq=255), INVALID), (attn, dict(ldo=252, Hq=4), INVALID),
    (attn, dict(Dh=80), UNSUPPORTED), (attn, dict(scale=float("nan")), INVALID),
    (attn, dict(scale=float("inf")), INVALID), (attn, dict(q=A + 4), INVALID), (attn, dict(t=1, ldq=260), INVALID),
    (attn, dict(B=-1), INVALID), (attn, dict(t=9), INVALID), (attn, dict(Lm=(1 << 30) + 1), UNSUPPORTED),
    (attn, dict(Sq=1 << 30), UNSUPPORTED),
    (attn, dict(n=A + 2), INVALID), (attn, dict(m=A + 1), INVALID), (attn, dict(ks=A + 2), INVALID),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_refused(i):
    f, bad, want = CASES[i]
    assert f(**bad) == want
    assert L.last_error()


@pytest.mark.parametrize("f,empty", [(norm, dict(M=0)), (norm, dict(K=0)), (gemm, dict(M=0)), (gemm, dict(N=0)),
                                     (gemm, dict(K=0)), (append, dict(B=0)), (append, dict(S=0)),
                                     (append, dict(H=0)), (read, dict(B=0)), (read, dict(S=0)),
                                     (attn, dict(B=0)), (attn, dict(Sq=0)), (attn, dict(Hq=0, Hkv=2))])
def test_empty_problem_is_ok(f, empty):
    assert f(**empty) == 0


def test_call_raises_with_the_message():
    with pytest.raises(L.DlmError, match="ldy"):
        L.call("dlm_gemm_i8", A, 64, A, A, A, None, A, 8, 4, 32, 64, 0, None)


def test_oracle_codes_round_halves_away_from_zero():
    # 127 x / 2 with x = k / 127 + 1 / 127: quotients k + 0.5 come out exactly for powers of two
    x = torch.tensor([[127.0, 0.5, -0.5, 1.5, -1.5, 0.49, 126.5, -126.5]])
    q, s = O.quant_rows(x)
    assert q.tolist() == [[127, 1, -1, 2, -2, 0, 127, -127]] and s.tolist() == [1.0]
    q, s = O.quant_rows(torch.tensor([[0.0, 0.0], [1.0, float("nan")], [float("inf"), 1.0]]))
    assert q.abs().sum() == 0 and s[0] == 0 and torch.isnan(s[1:]).all()
