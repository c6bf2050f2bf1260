"""The int8 language-model operators on the GPU against 64-bit forms of their formulas.

Tolerances count roundings: half a step of a type is eps / 2 relative (fp32 2^-24, fp16 2^-11,
bf16 2^-8).  Codes are compared exactly."""
import ctypes
import math

import pytest
import torch

from dollama_b200 import _lib as L
from tests import lm_i8_oracle as O

pytestmark = pytest.mark.gpu

F32, F16, BF16 = L.F32, L.F16, L.BF16
ALL = [F32, F16, BF16]


def _p(t):
    return None if t is None else t.data_ptr()


def _s():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def device_status():
    c = ctypes.c_int(-1)
    L.call("dlm_get_device_status", ctypes.byref(c), 1, _s())
    return c.value


@pytest.fixture(autouse=True)
def clean_status():
    yield
    torch.cuda.synchronize()
    assert device_status() == 0  # no kernel gave up a wait, no position was out of range


def same(a, b):
    """Equal values, NaN equal to NaN."""
    return a.dtype == b.dtype and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


# ------------------------------------------------------------------ norm

def run_norm(x, r, w, eps=1e-5, h=None, store=True):
    M, K = x.shape
    q = torch.full((M, K), 99, dtype=torch.int8, device="cuda")
    s = torch.full((M,), 7.0, device="cuda")
    if h is None and store:
        h = torch.empty(M, K, dtype=x.dtype, device="cuda")
    t = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[x.dtype]
    L.call("dlm_add_rms_norm_i8", _p(x), x.stride(0), _p(r), r.stride(0) if r is not None else 0, _p(w), _p(h),
           h.stride(0) if h is not None else 0, _p(q), _p(s), M, K, eps, t, _s())
    return h, q, s


def check_norm(x, r, w, got, eps=1e-5):
    h, q, s = got
    hr, qr, sr = O.add_rms_norm(x, r, w, eps)
    if h is not None:
        assert same(h, hr)
    assert torch.equal(q, qr)
    # sum of squares: chains of at most 64 (wide rows) + 37 fp32 additions, halved by the square root;
    # mean, + eps, root, two products and the quotient: 6 more
    assert torch.equal(torch.isnan(s), torch.isnan(sr))
    ok = ~torch.isnan(sr)
    assert ((s.double() - sr).abs() <= sr * (101 / 2 + 6) * O.U24 + 2.0 ** -150)[ok].all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 512), (8, 512), (3, 31), (5, 64), (70, 1000), (33, 1531), (2, 4096),
                                 (3, 8192), (2, 16384), (1, 32768), (2, 32767), (300, 8), (9, 2056)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm(t, M, K, residual):
    g, ty = gen(M * 7 + K), O.TYPES[t]
    x = (3 * torch.randn(M, K, generator=g, device="cuda")).to(ty)
    r = torch.randn(M, K, generator=g, device="cuda").to(ty) if residual else None
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(ty)
    check_norm(x, r, w, run_norm(x, r, w))


@pytest.mark.parametrize("t", ALL)
def test_norm_rows_of_special_values(t):
    ty, K = O.TYPES[t], 520
    x = torch.randn(9, K, generator=gen(5), device="cuda").to(ty)
    x[0] = 0                      # scale 0, codes 0
    x[1, 7] = float("nan")
    x[2, 100] = float("inf")
    x[3, 3] = -float("inf")
    x[4] = 0.5                    # equal values, all codes +-127
    x[5] = x[5] * (1e-4 if t == F16 else 1e-30)   # squares below fp32's range
    x[6] = x[6] * (1e4 if t == F16 else 1e30)     # squares above it
    x[7] = 0
    x[7, 511] = 2.0 ** -24        # one tiny value (a subnormal of fp16)
    x[8, ::2] = 127
    x[8, 1::2] = 0.5              # ties: code 1 (halves away from zero)
    w = torch.ones(K, device="cuda").to(ty)
    w[9] = 0
    check_norm(x, None, w, run_norm(x, None, w))
    w[500] = float("nan")         # every row has a NaN product
    h, q, s = run_norm(x, None, w)
    assert torch.isnan(s).all() and (q == 0).all() and same(h, x)


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("off,ld", [(0, 1024), (1, 1024), (0, 1003), (8, 1032)])
def test_norm_strides_in_place_and_neighbours(t, off, ld):
    """Row strides, unaligned starts, h over x and over the residual; nothing beyond the rows changes."""
    ty, M, K = O.TYPES[t], 6, 1000
    for where in ("x", "r"):
        g = gen(ld + off)
        bx = torch.randn(off + M * ld + 5, generator=g, device="cuda").to(ty)
        br = torch.randn(off + M * ld + 5, generator=g, device="cuda").to(ty)
        w = torch.randn(K, generator=g, device="cuda").to(ty)
        x = bx[off:off + M * ld].view(M, ld)[:, :K]
        r = br[off:off + M * ld].view(M, ld)[:, :K]
        x0, r0, bx0, br0 = x.clone(), r.clone(), bx.clone(), br.clone()
        got = run_norm(x, r, w, h=x if where == "x" else r)
        check_norm(x0, r0, w, (got[0].clone(), *got[1:]))
        (x if where == "x" else r).copy_(x0 if where == "x" else r0)
        assert torch.equal(bx, bx0) and torch.equal(br, br0)


def test_norm_without_h_and_matches_quantize_act():
    """With unit weights and no residual, the codes are dlm_quantize_act_i8's of the rows."""
    x = torch.randn(50, 768, generator=gen(3), device="cuda")
    w = torch.ones(768, device="cuda")
    h, q, s = run_norm(x, None, w, store=False)
    assert h is None
    qa = torch.empty_like(q)
    sa = torch.empty_like(s)
    L.call("dlm_quantize_act_i8", _p(x), 50, 768, _p(qa), _p(sa), _s())
    assert torch.equal(q, qa)


# ------------------------------------------------------------------ product

def make_gemm(M, N, K, t, bias, seed=1, ldx=None, ldy=None, full=False):
    g, ty = gen(seed + M + 3 * N + 5 * K), O.TYPES[t]
    ldx, ldy = ldx or K, ldy or N
    xq = torch.randint(-128 if full else -127, 128, (M, ldx), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.randint(-128 if full else -127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(M, generator=g, device="cuda") * 0.01
    ws = torch.rand(N, generator=g, device="cuda") * 0.001
    b = torch.randn(N, generator=g, device="cuda").to(ty) if bias else None
    y = torch.full((M, ldy), -77.0, device="cuda", dtype=ty)
    return xq, xs, wq, ws, b, y


def run_gemm(xq, xs, wq, ws, b, y, t, M, N, K):
    L.call("dlm_gemm_i8", _p(xq), xq.stride(0), _p(xs), _p(wq), _p(ws), _p(b), _p(y), y.stride(0), M, N, K, t, _s())


def check_gemm(xq, xs, wq, ws, b, y, t, M, N, K):
    ty = O.TYPES[t]
    want, prod = O.gemm(xq[:, :K], xs, wq, ws, b)
    # the sum's conversion and its product with xscale: one rounding each; the product with wscale
    # joins the bias in one; then the rounding to T
    tol = prod * 2.1 * O.U24 + want.abs() * (O.U24 + O.half_eps(ty)) * 1.01 + O.half_tiny(ty)
    assert ((y[:, :N].double() - want).abs() <= tol).all()
    assert (y[:, N:] == -77).all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 1536, 512), (8, 1536, 512), (16, 4096, 4096), (17, 130, 144),
                                   (32, 4096, 4096), (33, 257, 1040), (64, 512, 1536), (65, 640, 640), (100, 96, 48),
                                   (128, 128, 128), (129, 127, 272), (200, 5, 4096), (256, 512, 512),
                                   (1003, 2111, 1360), (300, 16000, 512), (2048, 1536, 512), (1, 16000, 512),
                                   (2050, 4100, 2064), (3, 40, 16384), (3000, 2111, 272)])
@pytest.mark.parametrize("bias", [False, True])
def test_gemm(t, M, N, K, bias):
    a = make_gemm(M, N, K, t, bias)
    run_gemm(*a, t, M, N, K)
    check_gemm(*a, t, M, N, K)


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("M", [3, 40, 100, 600, 3000])
def test_gemm_strides(t, M):
    """Row strides of both sides, odd output rows, a shifted output; the elements between stay."""
    N, K = 389, 208
    for ldx, ldy in ((224, 389), (1040, 400), (208, 391)):
        a = make_gemm(M, N, K, t, True, ldx=ldx, ldy=ldy)
        run_gemm(*a, t, M, N, K)
        check_gemm(*a, t, M, N, K)
        big = torch.full((M * ldy + 1,), -77.0, device="cuda", dtype=O.TYPES[t])
        y = big[1:].view(M, ldy)
        run_gemm(*a[:5], y, t, M, N, K)
        check_gemm(*a[:5], y, t, M, N, K)
        assert big[0] == -77


@pytest.mark.parametrize("M", [4, 50, 128, 2048])
def test_gemm_sum_is_exact_at_the_largest_codes(M):
    """All codes -128: the sum is 2^14 K, exact in int32 up to the largest K."""
    K, N = 131056, 48
    xq = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(max(M, N), device="cuda")
    y = torch.empty(M, N, device="cuda")
    run_gemm(xq, one, wq, one, None, y, F32, M, N, K)
    assert (y == float(torch.tensor(16384.0 * K))).all()


@pytest.mark.parametrize("M", [5, 64, 200, 1500])
def test_gemm_rows_with_nan_scale(M):
    """A token whose scale is NaN gives a row of NaN and touches no other."""
    a = make_gemm(M, 256, 512, F16, False)
    a[1][2] = float("nan")
    run_gemm(*a, F16, M, 256, 512)
    y = a[5]
    assert torch.isnan(y[2]).all() and not torch.isnan(y[:2]).any() and not torch.isnan(y[3:]).any()


# ------------------------------------------------------------------ cache

def ld(x):
    """Elements between the tokens of [B, S, heads, Dh] (a size-1 dimension's stride says nothing)."""
    return x.stride(1) if x.shape[1] > 1 else x.stride(0) if x.shape[0] > 1 else x.shape[2] * x.shape[3]


def empty_cache(B, H, Lm, Dh):
    kq = torch.full((B, H, Lm, Dh), 55, dtype=torch.int8, device="cuda")
    ks = torch.full((B, H, Lm), 9.0, device="cuda")
    return kq, ks, kq.clone(), ks.clone()


def append(k, v, cache, pos, n, t, Lm):
    B, S, H, Dh = k.shape
    L.call("dlm_kv_i8_append", _p(k), ld(k), _p(v), ld(v), *map(_p, cache), B, S, H, Dh, Lm, _p(pos),
           _p(n), t, _s())


def read(k, v, cache, pos, n, t, Lm):
    B, S, H, Dh = k.shape
    L.call("dlm_kv_i8_read", *map(_p, cache), _p(k), ld(k), _p(v), ld(v), B, S, H, Dh, Lm, _p(pos),
           _p(n), t, _s())


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("B,S,H,Dh,Lm,ragged", [(1, 1, 1, 64, 1, False), (3, 1, 8, 64, 128, False),
                                                (2, 5, 3, 128, 37, True), (4, 130, 2, 64, 300, True),
                                                (1, 257, 1, 128, 257, False), (5, 2, 16, 128, 9, True)])
def test_cache_write_and_read(t, B, S, H, Dh, Lm, ragged):
    g, ty = gen(B + 10 * S), O.TYPES[t]
    qkv = torch.randn(B, S, 3 * H * Dh, generator=g, device="cuda").to(ty)  # columns of a projection
    k = qkv[..., H * Dh:2 * H * Dh].unflatten(-1, (H, Dh))
    v = qkv[..., 2 * H * Dh:].unflatten(-1, (H, Dh))
    if S * H > 2:
        k[0, 0, 0] = 0
        v[0, 0, H - 1, 5] = float("inf")
        k[0, S - 1, H - 1, 3] = float("nan")
        v[B - 1, 0, 0] = v[B - 1, 0, 0] * (6e-8 if t == F16 else 1e-37)
        k[B - 1, 0, 0, ::2] = 0.5
        k[B - 1, 0, 0, 1] = 127.0
    pos = torch.randint(0, Lm - S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n = torch.randint(0, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if ragged else None
    cache = empty_cache(B, H, Lm, Dh)
    ko, vo = (torch.full((B, S, H, Dh), 3.0, device="cuda", dtype=ty) for _ in range(2))
    append(k, v, cache, pos, n, t, Lm)
    read(ko, vo, cache, pos, n, t, Lm)
    for x, out, cq, cs in ((k, ko, cache[0], cache[1]), (v, vo, cache[2], cache[3])):
        wq, wsc = torch.full_like(cq, 55), torch.full_like(cs, 9.0)
        wo = torch.full_like(out, 3.0)
        q, s = O.quant_rows(x)
        # a / 127 rounded to fp32: a quotient of 24 bits by 127 is further than 2^-32 (relative)
        # from any rounding border, so its value to 52 bits rounds to the same
        s32 = s.float()
        for b in range(B):
            m, p0 = (S if n is None else int(n[b])), int(pos[b])
            wq[b, :, p0:p0 + m] = q[b, :m].transpose(0, 1)
            wsc[b, :, p0:p0 + m] = s32[b, :m].transpose(0, 1)
            wo[b, :m] = (q[b, :m].float() * s32[b, :m, :, None]).to(ty)
        assert torch.equal(cq, wq)
        assert torch.equal(cs.nan_to_num(nan=-5.0), wsc.nan_to_num(nan=-5.0))
        assert torch.equal(out.nan_to_num(nan=-5.0), wo.nan_to_num(nan=-5.0))


@pytest.mark.parametrize("t", [F16, BF16])
def test_cache_codes_of_every_pair_of_mantissas(t):
    """Every mantissa against every largest one, at exponent distances 0 to 8: codes exact, halves away
    from zero."""
    bits = 10 if t == F16 else 7
    n = 1 << bits
    m = (torch.arange(n, device="cuda", dtype=torch.float64) + n) / n  # [1, 2)
    for d in range(9):
        x = (m * 2.0 ** -d).repeat(n, 1)  # row: all mantissas, under one largest value
        x = torch.where(x > m[:, None], -x / 2, x)
        pad = -x.numel() // n % 60 if n % 60 == 0 else 60 - n % 60
        x = torch.cat([x, x[:, :pad]], 1).view(n, -1, 60)
        top = m[:, None, None].expand(-1, x.shape[1], 4)
        k = torch.cat([x, top], 2).to(O.TYPES[t]).view(1, -1, 1, 64)
        L_ = k.shape[1]
        cache = empty_cache(1, 1, L_, 64)
        append(k, k, cache, torch.zeros(1, dtype=torch.int32, device="cuda"), None, t, L_)
        q, s = O.quant_rows(k)
        assert torch.equal(cache[0].view(-1, 64), q.view(-1, 64)) and torch.equal(cache[1].view(-1), s.float().view(-1))


def test_cache_positions_outside_are_skipped_and_reported():
    B, S, H, Dh, Lm = 4, 3, 2, 64, 8
    k = torch.randn(B, S, H, Dh, device="cuda")
    cache = empty_cache(B, H, Lm, Dh)
    pos = torch.tensor([0, 6, -2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    append(k, k, cache, pos, None, F32, Lm)
    assert device_status() == 6
    q, _ = O.quant_rows(k)
    want = torch.full_like(cache[0], 55)
    want[0, :, 0:3] = q[0].transpose(0, 1)
    want[1, :, 6:8] = q[1, :2].transpose(0, 1)
    want[2, :, 0:1] = q[2, 2:].transpose(0, 1)
    assert torch.equal(cache[0], want) and torch.equal(cache[2], want)
    out = torch.full_like(k, 4.0)
    read(out, out.clone(), cache, pos, None, F32, Lm)
    assert device_status() == 6
    assert (out[1, 2] == 4).all() and (out[2, :2] == 4).all() and (out[3] == 4).all() and (out[1, :2] != 4).any()
    # counts below zero and above S: none, and all of S
    cache = empty_cache(B, H, Lm, Dh)
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    append(k, k, cache, pos, torch.tensor([-3, 9, 0, 1], dtype=torch.int32, device="cuda"), F32, Lm)
    rows = (cache[1] != 9).sum((1, 2)).tolist()
    assert rows == [0, S * H, 0, H]


# ------------------------------------------------------------------ attention

def make_cache(B, H, Lm, Dh, g):
    kq = torch.randint(-127, 128, (B, H, Lm, Dh), generator=g, device="cuda", dtype=torch.int8)
    vq = torch.randint(-127, 128, (B, H, Lm, Dh), generator=g, device="cuda", dtype=torch.int8)
    ks = (0.2 + torch.rand(B, H, Lm, generator=g, device="cuda")) / 64
    vs = (0.2 + torch.rand(B, H, Lm, generator=g, device="cuda")) / 64
    return kq, ks, vq, vs


def run_attn(q, cache, kv, ql, causal, t, out=None, scale=None):
    B, Sq, Hq, Dh = q.shape
    Hkv, Lm = cache[0].shape[1:3]
    if out is None:
        out = torch.full_like(q, -3.0)
    L.call("dlm_attention_kv_i8", _p(q), ld(q), *map(_p, cache), _p(out), ld(out), B, Hq, Hkv, Sq, Dh, Lm,
           _p(kv), _p(ql), int(causal), 1 / math.sqrt(Dh) if scale is None else scale, t, _s())
    return out


def check_attn(q, cache, kv, ql, causal, t, out, scale=None):
    ty = q.dtype
    Sq, Dh = q.shape[1], q.shape[3]
    want, bound = O.attention(q, *cache, kv, ql, causal, 1 / math.sqrt(Dh) if scale is None else scale)
    # weights: one rounding to fp16 (fp32: two terms, 2^-22)
    tol = bound(2.0 ** -22 if t == F32 else 2.0 ** -11) + want.abs() * O.half_eps(ty) * 1.01 + O.half_tiny(ty) + 1e-30
    for b in range(q.shape[0]):
        m = Sq if ql is None else min(max(int(ql[b]), 0), Sq)
        err = (out[b, :m].double() - want[b, :m]).abs()
        assert (err <= tol[b, :m]).all(), (b, (err / tol[b, :m]).max())
        assert (out[b, m:] == -3).all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Lm", [(1, 1, 1, 1, 1), (3, 8, 8, 1, 40), (2, 8, 2, 1, 130), (1, 4, 1, 1, 3000),
                                            (2, 6, 2, 3, 65), (2, 32, 2, 1, 257), (1, 2, 2, 70, 100),
                                            (1, 2, 1, 33, 200), (2, 1, 1, 17, 17), (1, 20, 1, 2, 513)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(t, Dh, B, Hq, Hkv, Sq, Lm, causal):
    g, ty = gen(B + Hq * 3 + Sq * 5 + Lm), O.TYPES[t]
    q = (1.5 * torch.randn(B, Sq, Hq, Dh, generator=g, device="cuda")).to(ty)
    cache = make_cache(B, Hkv, Lm, Dh, g)
    kv = torch.randint(Sq, Lm + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    for b in range(B):  # what lies behind the last token must not matter
        for c in (cache[1], cache[3]):
            c[b, :, int(kv[b]):] = float("nan")
    out = run_attn(q, cache, kv, None, causal, t)
    check_attn(q, cache, kv, None, causal, t, out)


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Sq", [1, 4, 40, 150])
def test_attention_ragged_and_empty(t, Sq):
    """Lengths of zero and one, queries without a key, fewer queries than Sq."""
    B, Hq, Hkv, Dh, Lm = 7, 4, 2, 64, 200
    g, ty = gen(Sq), O.TYPES[t]
    q = torch.randn(B, Sq, Hq, Dh, generator=g, device="cuda").to(ty)
    cache = make_cache(B, Hkv, Lm, Dh, g)
    kv = torch.tensor([0, 1, Lm, 2, 33, 64, Lm - 1], dtype=torch.int32, device="cuda")
    ql = torch.tensor([Sq, 1, 0, Sq, max(1, Sq // 2), 1, Sq], dtype=torch.int32, device="cuda")
    for causal in (True, False):
        for m in (None, ql):
            out = run_attn(q, cache, kv, m, causal, t)
            check_attn(q, cache, kv, m, causal, t, out)
            assert (out[0, :Sq] == 0).all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Sq", [2, 150])
def test_attention_masked_keys_may_hold_anything(t, Sq):
    """NaN and infinite scales of keys that only later queries see leave the earlier ones alone."""
    g, ty = gen(8), O.TYPES[t]
    q = torch.randn(1, Sq, 2, 64, generator=g, device="cuda").to(ty)
    cache = make_cache(1, 1, 300, 64, g)
    kv = torch.tensor([290], dtype=torch.int32, device="cuda")
    clean = run_attn(q, cache, kv, None, True, t)
    cache[1][0, 0, 289] = float("nan")
    cache[3][0, 0, 288] = float("inf") if Sq > 2 else float("nan")
    cache[3][0, 0, 289] = float("nan")
    out = run_attn(q, cache, kv, None, True, t)
    n = Sq - 2 if Sq > 2 else 0
    assert torch.equal(out[:, :n], clean[:, :n])
    assert torch.isnan(out[:, Sq - 1]).all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Sq", [3, 12, 40, 200])
def test_attention_rows_are_independent(t, Sq):
    """Infinite, NaN, huge and tiny queries leave the other rows' results as they are."""
    g, ty = gen(21), O.TYPES[t]
    q = torch.randn(1, Sq, 2, 64, generator=g, device="cuda").to(ty)
    cache = make_cache(1, 1, 300, 64, g)
    kv = torch.tensor([280], dtype=torch.int32, device="cuda")
    clean = run_attn(q, cache, kv, None, True, t)
    bad = q.clone()
    bad[0, 0, 0, 3] = float("inf")
    bad[0, 1, 1, 5] = float("nan")
    bad[0, 2, 0] *= 1e4 if t == F16 else 1e30
    bad[0, 2, 1] *= 1e-4 if t == F16 else 1e-30
    out = run_attn(bad, cache, kv, None, True, t)
    same_rows = [(i, h) for i in range(Sq) for h in range(2) if (i, h) not in ((0, 0), (1, 1), (2, 0), (2, 1))]
    for i, h in same_rows:
        assert torch.equal(out[0, i, h], clean[0, i, h]), (i, h)
    assert torch.isnan(out[0, 0, 0]).all() and torch.isnan(out[0, 1, 1]).all()
    check_attn(bad[:, 2:3, 1:], cache, torch.tensor([280 - Sq + 3], device="cuda"), None, True, t, out[:, 2:3, 1:])


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Sq,at", [(40, 291), (200, 200), (200, 270)])
@pytest.mark.parametrize("Dh", [64, 128])
def test_attention_tile_weighed_three_times(t, Sq, at, Dh):
    """An infinite value scale late in the cache never fits: the rows that do not see its key keep their
    results, whatever passes the tile takes for the others."""
    g, ty = gen(23), O.TYPES[t]
    q = torch.randn(1, Sq, 2, Dh, generator=g, device="cuda").to(ty)
    cache = make_cache(1, 1, 300, Dh, g)
    kv = torch.tensor([300], dtype=torch.int32, device="cuda")
    clean = run_attn(q, cache, kv, None, True, t)
    cache[3][0, 0, at] = float("inf")
    out = run_attn(q, cache, kv, None, True, t)
    n = at - (300 - Sq)  # query i sees keys 0 .. 300 - Sq + i
    assert 0 < n < Sq
    assert torch.equal(out[:, :n], clean[:, :n])
    assert not torch.isfinite(out[:, n:]).any()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Sq", [1, 20, 140])
def test_attention_scales_of_all_sizes(t, Sq):
    """Loud and silent rows: q, key and value scales over many orders of magnitude, sharp softmaxes."""
    g, ty = gen(4), O.TYPES[t]
    B, Hq, Hkv, Dh, Lm = 2, 4, 2, 64, 333
    q = torch.randn(B, Sq, Hq, Dh, generator=g, device="cuda")
    q = (q * torch.logspace(-3, 1, Hq, device="cuda")[:, None]).to(ty)
    cache = make_cache(B, Hkv, Lm, Dh, g)
    e = torch.rand(B, Hkv, Lm, generator=g, device="cuda")
    cache[3].mul_(10 ** (8 * e - 6))
    cache[1].mul_(10 ** (-2 * e))
    cache[3][0, 0] *= 1e-12
    cache[3][:, :, ::5] = 0
    kv = torch.tensor([Lm, 300], dtype=torch.int32, device="cuda")
    if t == F16:
        cache[3].mul_(1e-3).clamp_max_(100)
    out = run_attn(q, cache, kv, None, True, t)
    check_attn(q, cache, kv, None, True, t, out)
    z = run_attn(torch.zeros_like(q), cache, kv, None, True, t)  # equal weights
    check_attn(torch.zeros_like(q), cache, kv, None, True, t, z)


@pytest.mark.parametrize("t", ALL)
def test_attention_strides(t):
    ty, B, Sq, Hq, Dh = O.TYPES[t], 2, 3, 4, 64
    g = gen(2)
    qkv = torch.randn(B, Sq, 3 * Hq * Dh, generator=g, device="cuda").to(ty)
    q = qkv[..., :Hq * Dh].unflatten(-1, (Hq, Dh))
    cache = make_cache(B, Hq, 50, Dh, g)
    kv = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    wide = torch.full((B, Sq, Hq * Dh + 16), -3.0, device="cuda", dtype=ty)
    out = wide[..., :Hq * Dh].unflatten(-1, (Hq, Dh))
    run_attn(q, cache, kv, None, True, t, out=out)
    check_attn(q, cache, kv, None, True, t, out)
    assert (wide[..., Hq * Dh:] == -3).all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("g,Dh", [(1, 64), (4, 128), (12, 64)])
def test_attention_many_sequences(t, g, Dh):
    """More (sequence, kv head) pairs than the SMs hold CTAs: one warp for each, ragged lengths."""
    B, Hkv, Lm = 900, 3, 70
    gn, ty = gen(g), O.TYPES[t]
    q = torch.randn(B, 1, Hkv * g, Dh, generator=gn, device="cuda").to(ty)
    cache = make_cache(B, Hkv, Lm, Dh, gn)
    kv = torch.randint(0, Lm + 1, (B,), generator=gn, device="cuda", dtype=torch.int32)
    out = run_attn(q, cache, kv, None, True, t)
    pick = torch.arange(0, B, 47, device="cuda")
    check_attn(q[pick], [c[pick] for c in cache], kv[pick], None, True, t, out[pick])
    # a sequence's result does not depend on the batch around it beyond the order of its sums
    one = run_attn(q[3:4].contiguous(), [c[3:4].contiguous() for c in cache], kv[3:4], None, True, t)
    check_attn(q[3:4], [c[3:4] for c in cache], kv[3:4], None, True, t, one)


@pytest.mark.parametrize("Sq,Hq,Hkv", [(127, 1, 1), (129, 1, 1), (43, 6, 2), (300, 5, 1), (17, 16, 16)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_attention_row_tiles(t, Sq, Hq, Hkv):
    """Rows that end inside a tile, groups of heads that no tile divides, keys split over clusters."""
    g, ty = gen(Sq), O.TYPES[t]
    q = torch.randn(1, Sq, Hq, 128, generator=g, device="cuda").to(ty)
    cache = make_cache(1, Hkv, 700, 128, g)
    kv = torch.tensor([691], dtype=torch.int32, device="cuda")
    out = run_attn(q, cache, kv, None, True, t)
    pick = [0, 1, Sq // 2, Sq - 2, Sq - 1]
    for i in pick:  # query i alone is the last of a shorter sequence
        n = torch.tensor([691 - Sq + i + 1], dtype=torch.int32, device="cuda")
        check_attn(q[:, i:i + 1].contiguous(), cache, n, None, True, t, out[:, i:i + 1])


def test_attention_without_a_cache_is_zero():
    q = torch.randn(2, 3, 4, 64, device="cuda")
    out = torch.full_like(q, 5.0)
    kv = torch.zeros(2, dtype=torch.int32, device="cuda")
    L.call("dlm_attention_kv_i8", _p(q), 256, None, None, None, None, _p(out), 256, 2, 4, 2, 3, 64, 0, _p(kv), None, 1,
           0.125, F32, _s())
    assert (out == 0).all()


def test_attention_length_outside_is_clamped_and_reported():
    g = gen(6)
    q = torch.randn(2, 1, 2, 64, generator=g, device="cuda")
    cache = make_cache(2, 2, 30, 64, g)
    kv = torch.tensor([-1, 31], dtype=torch.int32, device="cuda")
    out = run_attn(q, cache, kv, None, True, F32)
    assert device_status() == 6
    ok = torch.tensor([0, 30], dtype=torch.int32, device="cuda")
    assert torch.equal(out, run_attn(q, cache, ok, None, True, F32))


def test_attention_offsets_beyond_32_bits():
    """A cache of more than 2^32 code bytes: the last head of the last sequence."""
    B, H, Dh, Lm = 3, 8, 128, 1 << 21
    kq = torch.zeros(B, H, Lm, Dh, dtype=torch.int8, device="cuda")
    ks = torch.zeros(B, H, Lm, device="cuda")
    vq, vs = torch.zeros_like(kq), torch.zeros_like(ks)
    assert kq.numel() > 2 ** 32
    g = gen(12)
    k = torch.randn(B, 2, H, Dh, generator=g, device="cuda").half()
    v = torch.randn(B, 2, H, Dh, generator=g, device="cuda").half()
    pos = torch.tensor([0, 5, Lm - 2], dtype=torch.int32, device="cuda")
    append(k, v, (kq, ks, vq, vs), pos, None, F16, Lm)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    read(ko, vo, (kq, ks, vq, vs), pos, None, F16, Lm)
    q, s = O.quant_rows(v)
    assert torch.equal(vo, (q.float() * s.float()[..., None]).half())
    # every other key has scale 0 (score 0): make the two written ones of the last sequence dominate
    qy = (ko[:, 1:2] * 40).contiguous()
    kv = torch.tensor([2, 7, Lm], dtype=torch.int32, device="cuda")
    out = run_attn(qy, (kq, ks, vq, vs), kv, None, True, F16)
    assert ((out[2, 0].float() - vo[2, 1].float()).abs() <= 2.0 ** -9 * vo[2, 1].float().abs() + 1e-3).all()


def test_repeated_calls_are_bit_identical():
    g = gen(31)
    q = torch.randn(2, 1, 8, 64, generator=g, device="cuda")
    cache = make_cache(2, 2, 2500, 64, g)
    kv = torch.tensor([2500, 1999], dtype=torch.int32, device="cuda")
    first = run_attn(q, cache, kv, None, True, F32)
    a = make_gemm(16, 512, 2048, F16, False)
    run_gemm(*a, F16, 16, 512, 2048)
    y0 = a[5].clone()
    for _ in range(5):
        assert torch.equal(first, run_attn(q, cache, kv, None, True, F32))
        run_gemm(*a, F16, 16, 512, 2048)
        assert torch.equal(y0, a[5])


def test_calls_on_two_streams_at_once():
    """The same operators on two streams, in turn, each with its own outputs."""
    work = []
    for k in range(2):
        g = gen(50 + k)
        q = torch.randn(4, 30, 4, 64, generator=g, device="cuda").half()
        cache = make_cache(4, 2, 900, 64, g)
        kv = torch.full((4,), 880, dtype=torch.int32, device="cuda")
        work.append((q, cache, kv, make_gemm(300, 700, 1040, F16, True, seed=k)))
    want = []
    for q, cache, kv, a in work:
        run_gemm(*a, F16, 300, 700, 1040)
        want.append((run_attn(q, cache, kv, None, True, F16), a[5].clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    outs = [torch.zeros_like(w[0]) for w in work]
    for _ in range(10):
        for s, o, (q, cache, kv, a) in zip(streams, outs, work):
            with torch.cuda.stream(s):
                run_gemm(*a, F16, 300, 700, 1040)
                run_attn(q, cache, kv, None, True, F16, out=o)
    torch.cuda.synchronize()
    for (o, (w, y), (_, _, _, a)) in zip(outs, want, work):
        assert torch.equal(o, w) and torch.equal(a[5], y)


@pytest.mark.parametrize("M", [20, 33, 64])
def test_split_product_beside_clusters_of_attention(M):
    """Both kinds of clusters hold tensor memory: on two streams neither may keep the other's waiting."""
    g = gen(60 + M)
    q = torch.randn(4, 30, 4, 64, generator=g, device="cuda").half()
    cache = make_cache(4, 2, 900, 64, g)
    kv = torch.full((4,), 880, dtype=torch.int32, device="cuda")
    a = make_gemm(M, 2048, 2048, F16, False, seed=M)
    run_gemm(*a, F16, M, 2048, 2048)
    want, y = run_attn(q, cache, kv, None, True, F16), a[5].clone()
    a[5].fill_(-77)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    s = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(50):
        with torch.cuda.stream(s[0]):
            run_attn(q, cache, kv, None, True, F16, out=out)
        with torch.cuda.stream(s[1]):
            run_gemm(*a, F16, M, 2048, 2048)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(a[5], y)


_FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from tests import test_lm_i8_gpu as G
torch.zeros(1, device="cuda")
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(40, 256, generator=g, device="cuda").half()
w = torch.ones(256, device="cuda").half()
h, q, s = torch.empty_like(x), torch.empty(40, 256, dtype=torch.int8, device="cuda"), torch.empty(40, device="cuda")
wq = torch.randint(-127, 128, (256, 256), device="cuda", dtype=torch.int8)
ws = torch.rand(256, device="cuda")
y = torch.empty(40, 256, device="cuda").half()
cache = [torch.zeros(2, 2, 64, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, 64, device="cuda")]
cache += [c.clone() for c in cache]
pos = torch.zeros(2, dtype=torch.int32, device="cuda")
kv = torch.full((2,), 20, dtype=torch.int32, device="cuda")
qq = torch.randn(2, 20, 4, 64, device="cuda").half()
o, one = torch.empty_like(qq), torch.empty(2, 1, 4, 64, device="cuda").half()
def all_of_them():
    G.L.call("dlm_add_rms_norm_i8", x.data_ptr(), 256, None, 0, w.data_ptr(), h.data_ptr(), 256, q.data_ptr(),
             s.data_ptr(), 40, 256, 1e-5, 1, G._s())
    G.run_gemm(q, s, wq, ws, None, y, 1, 40, 256, 256)
    G.L.call("dlm_kv_i8_append", y.data_ptr(), 256, y.data_ptr() + 256, 256, *[c.data_ptr() for c in cache], 2, 20, 2, 64,
             64, pos.data_ptr(), None, 1, G._s())
    G.run_attn(qq, cache, kv, None, True, 1, out=o)
    G.run_attn(qq[:, :1].contiguous(), cache, kv, None, True, 1, out=one)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    all_of_them()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (q, s, y, *cache, o)]
all_of_them()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (q, s, y, *cache, o)))
print("captured first")
"""


def test_first_calls_inside_a_capture():
    """A process whose first call of each operator is captured (no warm-up)."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", _FIRST, root], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------ together

class Layer:
    """One attention block of a decoder layer: norm -> q|k|v -> cache -> attention -> quantize ->
    out projection, with the residual stream in `dtype`."""

    def __init__(self, D, Hq, Hkv, Dh, B, Lm, t, seed):
        g, ty = gen(seed), O.TYPES[t]
        self.D, self.Hq, self.Hkv, self.Dh, self.B, self.Lm, self.t, self.ty = D, Hq, Hkv, Dh, B, Lm, t, ty
        self.nw = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(ty)
        self.N = (Hq + 2 * Hkv) * Dh
        self.w = {}
        for name, n, k in (("qkv", self.N, D), ("out", D, Hq * Dh)):
            w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
            q = torch.empty(n, k, dtype=torch.int8, device="cuda")
            s = torch.empty(n, device="cuda")
            L.call("dlm_quantize_act_i8", _p(w), n, k, _p(q), _p(s), _s())
            self.w[name] = (q, s)
        self.cache = [torch.zeros(B, Hkv, Lm, Dh, dtype=torch.int8, device="cuda"),
                      torch.zeros(B, Hkv, Lm, device="cuda")]
        self.cache += [c.clone() for c in self.cache]

    def buffers(self, S):
        M, z = self.B * S, dict(device="cuda")
        return dict(h=torch.empty(M, self.D, dtype=self.ty, **z), xq=torch.empty(M, self.D, dtype=torch.int8, **z),
                    xs=torch.empty(M, **z), qkv=torch.empty(M, self.N, dtype=self.ty, **z),
                    ao=torch.empty(M, self.Hq * self.Dh, dtype=self.ty, **z),
                    af=torch.empty(M, self.Hq * self.Dh, **z),
                    aq=torch.empty(M, self.Hq * self.Dh, dtype=torch.int8, **z), as_=torch.empty(M, **z),
                    y=torch.empty(M, self.D, dtype=self.ty, **z))

    def step(self, x, r, pos, kv, S, b):
        M, W, e = self.B * S, self.Hq * self.Dh, self.nw.element_size()
        L.call("dlm_add_rms_norm_i8", _p(x), self.D, _p(r), self.D, _p(self.nw), _p(b["h"]), self.D, _p(b["xq"]),
               _p(b["xs"]), M, self.D, 1e-5, self.t, _s())
        run_gemm(b["xq"], b["xs"], *self.w["qkv"], None, b["qkv"], self.t, M, self.N, self.D)
        at = _p(b["qkv"])
        k, v = at + W * e, at + (W + self.Hkv * self.Dh) * e
        L.call("dlm_kv_i8_append", k, self.N, v, self.N, *map(_p, self.cache), self.B, S, self.Hkv, self.Dh, self.Lm,
               _p(pos), None, self.t, _s())
        L.call("dlm_attention_kv_i8", at, self.N, *map(_p, self.cache), _p(b["ao"]), W, self.B, self.Hq, self.Hkv, S,
               self.Dh, self.Lm, _p(kv), None, 1, 1 / math.sqrt(self.Dh), self.t, _s())
        b["af"].copy_(b["ao"])
        L.call("dlm_quantize_act_i8", _p(b["af"]), M, W, _p(b["aq"]), _p(b["as_"]), _s())
        run_gemm(b["aq"], b["as_"], *self.w["out"], None, b["y"], self.t, M, self.D, W)
        return b["h"], b["y"]

    def check(self, x, r, pos, kv, S, b, before):
        """Each stage against its 64-bit form, on the stage's own inputs."""
        W, H, Dh = self.Hq * self.Dh, self.Hkv, self.Dh
        check_norm(x, r, self.nw, (b["h"], b["xq"], b["xs"]))
        check_gemm(b["xq"], b["xs"], *self.w["qkv"], None, b["qkv"], self.t, self.B * S, self.N, self.D)
        qkv = b["qkv"].view(self.B, S, self.N)
        for x2, cq, cs, c0 in ((qkv[..., W:W + H * Dh], self.cache[0], self.cache[1], before[0]),
                               (qkv[..., W + H * Dh:], self.cache[2], self.cache[3], before[2])):
            q, _ = O.quant_rows(x2.unflatten(-1, (H, Dh)))
            want = c0.clone()
            for i in range(self.B):
                want[i, :, int(pos[i]):int(pos[i]) + S] = q[i].transpose(0, 1)
            assert torch.equal(cq, want)
        check_attn(qkv[..., :W].unflatten(-1, (self.Hq, Dh)), self.cache, kv, None, True, self.t,
                   b["ao"].view(self.B, S, self.Hq, Dh))
        check_gemm(b["aq"], b["as_"], *self.w["out"], None, b["y"], self.t, self.B * S, self.D, W)


@pytest.mark.parametrize("t", ALL)
def test_layer_prefill_and_decode(t):
    B, S = 3, 40
    ly = Layer(512, 8, 4, 64, B, 64, t, 5)
    g = gen(9)
    x, r = (torch.randn(B * S, 512, generator=g, device="cuda").to(ly.ty) for _ in range(2))
    pos = torch.tensor([0, 4, 20], dtype=torch.int32, device="cuda")
    b = ly.buffers(S)
    c0 = [c.clone() for c in ly.cache]
    ly.step(x, r, pos, pos + S, S, b)
    ly.check(x, r, pos, pos + S, S, b, c0)
    pos = pos + S
    one = ly.buffers(1)
    for _ in range(3):
        x, r = (torch.randn(B, 512, generator=g, device="cuda").to(ly.ty) for _ in range(2))
        c0 = [c.clone() for c in ly.cache]
        ly.step(x, r, pos, pos + 1, 1, one)
        ly.check(x, r, pos, pos + 1, 1, one, c0)
        pos = pos + 1


def test_layer_in_a_graph_on_another_stream():
    """The decode step captured and replayed with new inputs and positions equals the eager call."""
    B, t = 4, F16
    ly = Layer(256, 4, 2, 64, B, 32, t, 6)
    g = gen(3)
    x, r = (torch.randn(B, 256, generator=g, device="cuda").to(ly.ty) for _ in range(2))
    pos = torch.tensor([3, 0, 9, 1], dtype=torch.int32, device="cuda")
    kv = pos + 1
    b = ly.buffers(1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ly.step(x, r, pos, kv, 1, b)  # warm-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ly.step(x, r, pos, kv, 1, b)
    torch.cuda.synchronize()
    for k in range(4):
        x.copy_(torch.randn(B, 256, generator=g, device="cuda"))
        pos.add_(1)
        kv.add_(1)
        before = [c.clone() for c in ly.cache]
        graph.replay()
        torch.cuda.synchronize()
        got = {n: v.clone() for n, v in b.items()}
        after = [c.clone() for c in ly.cache]
        for c, c0 in zip(ly.cache, before):
            c.copy_(c0)
        ly.step(x, r, pos, kv, 1, b)
        assert all(torch.equal(got[n], b[n]) for n in b)
        assert all(torch.equal(p, q) for p, q in zip(after, ly.cache))
