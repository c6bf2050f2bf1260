"""The int8 language-model operators where their launch rules and main loops change form: rows just
below a kernel's shared-memory limit, rings used many times over, references that move late, keys and
rows that must not touch one another.  Tolerances and 64-bit forms are those of test_lm_i8_gpu."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from dollama_b200 import _lib as L
from dollama_b200.build import nvcc
from tests import lm_i8_oracle as O
from tests import test_lm_i8_gpu as G
from tests.test_lm_i8_gpu import ALL, F32, clean_status, gen  # noqa: F401 (clean_status: autouse)

pytestmark = pytest.mark.gpu
ROOT = str(Path(__file__).resolve().parent.parent)


def fresh_process(code):
    """Runs `code` in a process of its own, in which it makes the first calls of the library."""
    r = subprocess.run([sys.executable, "-c", code, ROOT], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------ norm

_LONG_ROWS = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from tests import test_lm_i8_gpu as G
ty = torch.%s
for K in %s:
    g = G.gen(K)
    x, r = ((torch.randn(2, K, generator=g, device="cuda")).to(ty) for _ in range(2))
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(ty)
    G.check_norm(x, r, w, G.run_norm(x, r, w))
print("done")
"""


@pytest.mark.parametrize("ty,Ks", [("float32", (10244, 12288)), ("float32", (11777, 12287)),
                                   ("float16", (20488, 24576)), ("float16", (24065, 24575)),
                                   ("bfloat16", (20488, 24576)), ("bfloat16", (24065, 24575))])
def test_norm_rows_of_48_kilobytes_first(ty, Ks):
    """Rows that take 48 KB of dynamic shared memory (beside the kernel's static arrays) as a process's
    first: no longer row has raised the kernel's limit before."""
    fresh_process(_LONG_ROWS % (ty, Ks))


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("K", [8200, 12288, 24575, 32768])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_norm_long_rows_in_place(t, K, over):
    """Rows in shared memory whose sum replaces an input."""
    g, ty = gen(K), O.TYPES[t]
    x, r = (torch.randn(3, K, generator=g, device="cuda").to(ty) for _ in range(2))
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(ty)
    x0, r0 = x.clone(), r.clone()
    got = G.run_norm(x, r, w, h=x if over == "x" else r)
    G.check_norm(x0, r0, w, got)
    assert torch.equal(r, r0) if over == "x" else torch.equal(x, x0)


def test_norm_and_product_beyond_32_bit_offsets():
    """More than 2^31 elements in rows and results: the last rows."""
    M, K = 70000, 32768
    g = gen(77)
    x = torch.empty(M, K, device="cuda", dtype=torch.half)
    x.normal_(generator=g)
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).half()
    h, q, s = G.run_norm(x, None, w)
    for rows in (slice(0, 2), slice(65535, 65538), slice(M - 2, M)):
        G.check_norm(x[rows], None, w, (h[rows], q[rows], s[rows]))
    del x, h
    N = 32768
    a = q[:, :256].contiguous()
    wq = torch.randint(-127, 128, (N, 256), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(N, generator=g, device="cuda") / 64
    for t, ldy in ((L.F16, N), (L.BF16, N + 1)):  # tensor stores, element stores
        y = torch.full((M, ldy), -77.0, device="cuda", dtype=O.TYPES[t])
        G.run_gemm(a, s, wq, ws, None, y, t, M, N, 256)
        for rows in (slice(0, 2), slice(65534, 65538), slice(M - 2, M)):
            G.check_gemm(a[rows], s[rows], wq, ws, None, y[rows], t, len(a[rows]), N, 256)
        del y


# ------------------------------------------------------------------ empty problems

@pytest.mark.parametrize("t", ALL)
def test_a_size_of_zero_writes_nothing(t):
    """Any size of 0 is an empty problem: no output changes, a product's bias with K = 0 included."""
    ty = O.TYPES[t]
    p, s = G._p, G._s()
    x, w = torch.ones(4, 64, device="cuda", dtype=ty), torch.ones(64, device="cuda", dtype=ty)
    h, xq, xs = (torch.full((4, 64), 9, device="cuda", dtype=d) for d in (ty, torch.int8, torch.float32))
    for M, K in ((0, 64), (4, 0), (0, 0)):
        L.call("dlm_add_rms_norm_i8", p(x), 64, None, 0, p(w), p(h), 64, p(xq), p(xs), M, K, 1e-5, t, s)
    wq, y = torch.ones(32, 64, device="cuda", dtype=torch.int8), torch.full((4, 32), 9, device="cuda", dtype=ty)
    for M, N, K in ((4, 32, 0), (0, 32, 64), (4, 0, 64)):
        L.call("dlm_gemm_i8", p(xq), 64, p(xs), p(wq), p(xs), p(w), p(y), 32, M, N, K, t, s)
    cache = G.empty_cache(2, 2, 16, 64)
    k = torch.full((2, 3, 2, 64), 9, device="cuda", dtype=ty)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    for B, S, H, Lm in ((0, 3, 2, 16), (2, 0, 2, 16), (2, 3, 0, 16), (2, 3, 2, 0)):
        shape = (B, S, H, 64, Lm, p(pos), None, t, s)
        L.call("dlm_kv_i8_append", p(k), 128, p(k), 128, *map(p, cache), *shape)
        L.call("dlm_kv_i8_read", *map(p, cache), p(k), 128, p(k), 128, *shape)
    o = torch.full((2, 3, 4, 64), 9, device="cuda", dtype=ty)
    for B, Hq, Hkv, Sq in ((0, 4, 2, 3), (2, 0, 2, 3), (2, 4, 2, 0)):
        L.call("dlm_attention_kv_i8", p(k), 256, *map(p, cache), p(o), 256, B, Hq, Hkv, Sq, 64, 16, p(pos), None, 1,
               0.125, t, s)
    assert all((z == 9).all() for z in (h, xq, xs, y, k, o))
    assert all((c == v).all() for c, v in zip(cache, (55, 9, 55, 9)))


# ------------------------------------------------------------------ attention: rows and keys apart

@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("Sq,Lm,B", [(2, 4096, 1), (4, 4096, 1), (8, 4096, 1), (4, 100, 900), (8, 100, 900)])
def test_few_rows_keep_their_bits_when_a_neighbour_moves(t, Dh, Sq, Lm, B):
    """A loud key that the last query alone sees, in a unit of keys that is not its warp's first (one
    sequence: four units of a warp, clusters; 900: a warp each): the last query's reference moves, the
    other rows' results stay to the bit."""
    g, ty = gen(Sq + Dh), O.TYPES[t]
    q = (1.5 * torch.randn(B, Sq, 2, Dh, generator=g, device="cuda")).to(ty)
    cache = G.make_cache(B, 1, Lm, Dh, g)
    n = Lm - 6  # the last unit holds keys that all see, too
    kv = torch.full((B,), n, dtype=torch.int32, device="cuda")
    clean = G.run_attn(q, cache, kv, None, True, t)
    cache[3][:, :, n - 1] *= 1e6
    out = G.run_attn(q, cache, kv, None, True, t)
    assert torch.equal(out[:, :Sq - 1], clean[:, :Sq - 1])
    assert not torch.equal(out[:, Sq - 1], clean[:, Sq - 1])


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("loud", [1e5, 1e36])
def test_many_rows_keep_their_bits_when_a_neighbour_searches(t, Dh, loud):
    """Keys late in the cache (ten tiles, one CTA for all of them): one whose weight overshoots every
    row's reference by a known factor, one that only the last query sees and that sends its row back for
    the tile's maxima.  The other rows move as they do alone, to the bit."""
    g, ty = gen(Dh), O.TYPES[t]
    B, Hkv, Sq, Lm = 37, 4, 20, 640  # 148 row tiles
    q = (1.5 * torch.randn(B, Sq, Hkv, Dh, generator=g, device="cuda")).to(ty)
    cache = G.make_cache(B, Hkv, Lm, Dh, g)
    cache[3][:, :, Lm - 30] *= 1e5
    kv = torch.full((B,), Lm, dtype=torch.int32, device="cuda")
    clean = G.run_attn(q, cache, kv, None, True, t)
    cache[3][:, :, Lm - 1] *= loud
    out = G.run_attn(q, cache, kv, None, True, t)
    assert torch.equal(out[:, :Sq - 1], clean[:, :Sq - 1])
    assert not torch.equal(out[:, Sq - 1], clean[:, Sq - 1])


# ------------------------------------------------------------------ attention: long runs of the main loops

def shaped_cache(B, Hkv, Lm, Dh, shape, q, g):
    """smooth: random codes; rising: keys turn towards the queries along the cache, so that the scores'
    maximum moves again and again; leaps: a few keys far above (2^100 and more) all before them; values:
    value scales grow along the cache by 2^36; falling: the first keys are the loudest."""
    cache = G.make_cache(B, Hkv, Lm, Dh, g)
    j = torch.arange(Lm, device="cuda") / Lm
    if shape in ("rising", "falling"):
        to = q.float().mean((1, 2))  # [B, Dh], shared by all queries (see base below)
        to = 90 * to / to.abs().amax(-1, keepdim=True)
        a = j if shape == "rising" else 1 - j
        k = a[:, None] * to[:, None, None] + (1 - a[:, None]) * cache[0].float() * 0.4
        cache[0].copy_(k.round().clamp(-127, 127))
        cache[1].mul_(5)
    elif shape == "leaps":
        cache[1][:, :, Lm * 2 // 5::97] *= 40
    elif shape == "values":
        cache[3].mul_(torch.exp2(36 * j - 30))
    return cache


def check_some(q, cache, kv, causal, t, out, seqs, queries):
    """Query i alone is the last of a shorter sequence."""
    Sq = q.shape[1]
    s = torch.tensor(seqs, device="cuda")
    for i in queries:
        n = kv[s] - (Sq - 1 - i if causal else 0)
        G.check_attn(q[s, i:i + 1].contiguous(), [c[s] for c in cache], n, None, causal, t,
                     out[s, i:i + 1])


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("shape", ["smooth", "rising", "falling", "leaps", "values"])
@pytest.mark.parametrize("B,Hkv,g,Sq,Lm", [(37, 4, 2, 20, 700), (19, 4, 2, 70, 460), (1, 4, 1, 20, 8000)])
def test_many_rows_over_many_tiles(t, Dh, shape, B, Hkv, g, Sq, Lm):
    """The many-row kernel with 8 to 16 tiles of 64 keys a CTA (row tiles for every SM, two waves of them,
    and a cluster of eight), so that stages, score buffers and phases are used again and O is rescaled
    between tiles: rising and values move a row's reference 1.7 to 3.6 times after a stream's first tile,
    leaps half of them, some beyond what an overshoot can say (counted on the inputs in 64 bits)."""
    gn, ty = gen(B + Sq + Dh), O.TYPES[t]
    base = torch.randn(B, 1, 1, Dh, generator=gn, device="cuda")
    noise = torch.randn(B, Sq, Hkv * g, Dh, generator=gn, device="cuda")
    q = (base + 0.5 * noise if shape in ("rising", "falling") else 1.5 * noise).to(ty)
    cache = shaped_cache(B, Hkv, Lm, Dh, shape, q, gn)
    kv = torch.randint(Lm - 100, Lm + 1, (B,), generator=gn, device="cuda", dtype=torch.int32)
    for c in (cache[1], cache[3]):
        for b in range(B):
            c[b, :, int(kv[b]):] = float("nan")
    for causal in (True, False):
        out = G.run_attn(q, cache, kv, None, causal, t)
        check_some(q, cache, kv, causal, t, out, sorted({0, B // 2, B - 1}), (0, Sq // 2, Sq - 1))
        assert torch.equal(out, G.run_attn(q, cache, kv, None, causal, t))


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("shape", ["smooth", "rising", "falling", "leaps", "values"])
@pytest.mark.parametrize("B,Hkv,g,Sq,Lm", [(1, 1, 8, 1, 16000), (1, 2, 4, 4, 16000), (150, 2, 4, 1, 900),
                                           (600, 2, 2, 2, 500)])
def test_few_rows_over_many_units(t, Dh, shape, B, Hkv, g, Sq, Lm):
    """The few-row kernel with 7 to 16 units of 32 keys a warp: clusters with the deep ring, one or two CTAs
    a tile with the shallow one, a warp a tile."""
    gn, ty = gen(B + Sq + Dh), O.TYPES[t]
    base = torch.randn(B, 1, 1, Dh, generator=gn, device="cuda")
    noise = torch.randn(B, Sq, Hkv * g, Dh, generator=gn, device="cuda")
    q = (base + 0.5 * noise if shape in ("rising", "falling") else 1.5 * noise).to(ty)
    cache = shaped_cache(B, Hkv, Lm, Dh, shape, q, gn)
    kv = torch.randint(Lm - 100, Lm + 1, (B,), generator=gn, device="cuda", dtype=torch.int32)
    out = G.run_attn(q, cache, kv, None, True, t)
    check_some(q, cache, kv, True, t, out, sorted({0, B // 2, B - 1}), (0, Sq - 1) if Sq > 1 else (0,))
    assert torch.equal(out, G.run_attn(q, cache, kv, None, True, t))


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("Sq", [4, 8, 150])
@pytest.mark.parametrize("Lm,B", [(300, 1), (4096, 1), (300, 500)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_keys_of_later_queries_may_hold_anything(t, Dh, Sq, Lm, B, what):
    """NaN and infinite key and value scales of keys that the last two queries alone see: 8 and 16 rows of
    the few-row kernel (clusters of one and of four units a warp, a warp a tile) and 300 rows."""
    if B > 1 and Sq > 8:
        B = 60  # row tiles beyond a wave
    g, ty = gen(Sq + Lm), O.TYPES[t]
    q = torch.randn(B, Sq, 2, Dh, generator=g, device="cuda").to(ty)
    cache = G.make_cache(B, 1, Lm, Dh, g)
    n = Lm - 3
    kv = torch.full((B,), n, dtype=torch.int32, device="cuda")
    clean = G.run_attn(q, cache, kv, None, True, t)
    before = Sq - 2
    assert before > 0
    for ks, vs in ((what, None), (None, what), (what, what)):
        bad = [c.clone() for c in cache]
        for at in (n - 2, n - 1):
            if ks is not None:
                bad[1][:, :, at] = ks
            if vs is not None:
                bad[3][:, :, at] = vs
        out = G.run_attn(q, bad, kv, None, True, t)
        assert torch.equal(out[:, :before], clean[:, :before])
        # a key's NaN is its row's; an infinite key scale is a score of +-inf (a weight of NaN or 0), an
        # infinite value scale a result that is not finite
        if what != what or vs is not None:
            assert not torch.isfinite(out[:, Sq - 1]).any()


# ------------------------------------------------------------------ first calls captured

_CAPTURED = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from tests import test_lm_i8_gpu as G
dev = dict(device="cuda")
g = G.gen(1)
K = %d
x = torch.randn(40, K, generator=g, **dev).half()
w = torch.ones(K, **dev).half()
wq = torch.randint(-127, 128, (256, 256), generator=g, device="cuda", dtype=torch.int8)
ws = torch.rand(256, generator=g, **dev)
xq = torch.randint(-127, 128, (40, 256), generator=g, device="cuda", dtype=torch.int8)
xs = torch.rand(40, generator=g, **dev) / 64  # sums of 256 products of 73 x 73, about 9e4, inside fp16
pos = torch.zeros(2, dtype=torch.int32, **dev)
kv = torch.full((2,), 20, dtype=torch.int32, **dev)
qq = torch.randn(2, 20, 4, 64, generator=g, **dev).half()
q1 = qq[:, :1].contiguous()
out = dict(h=torch.empty_like(x), q=torch.empty(40, K, dtype=torch.int8, **dev), s=torch.empty(40, **dev),
           y=torch.empty(40, 256, **dev).half(), kq=torch.empty(2, 2, 64, 64, dtype=torch.int8, **dev),
           ks=torch.empty(2, 2, 64, **dev), vq=torch.empty(2, 2, 64, 64, dtype=torch.int8, **dev),
           vs=torch.empty(2, 2, 64, **dev), k=torch.empty(2, 20, 2, 64, **dev).half(),
           v=torch.empty(2, 20, 2, 64, **dev).half(), many=torch.empty_like(qq), one=torch.empty_like(q1))
cache = [out[n] for n in ("kq", "ks", "vq", "vs")]
def fill():
    for o in out.values():
        o.fill_(99)
def all_of_them():
    G.L.call("dlm_add_rms_norm_i8", x.data_ptr(), K, None, 0, w.data_ptr(), out["h"].data_ptr(), K,
             out["q"].data_ptr(), out["s"].data_ptr(), 40, K, 1e-5, 1, G._s())
    G.run_gemm(xq, xs, wq, ws, None, out["y"], 1, 40, 256, 256)
    G.L.call("dlm_kv_i8_append", out["y"].data_ptr(), 256, out["y"].data_ptr() + 256, 256,
             *[c.data_ptr() for c in cache], 2, 20, 2, 64, 64, pos.data_ptr(), None, 1, G._s())
    G.read(out["k"], out["v"], cache, pos, None, 1, 64)
    G.run_attn(qq, cache, kv, None, True, 1, out=out["many"])
    G.run_attn(q1, cache, kv, None, True, 1, out=out["one"])
fill()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    all_of_them()
torch.cuda.synchronize()
assert all((o == 99).all() for o in out.values())  # captured, not run
graph.replay()
torch.cuda.synchronize()
got = {n: o.clone() for n, o in out.items()}
fill()
all_of_them()
torch.cuda.synchronize()
for n, o in out.items():
    assert torch.equal(got[n], o) and torch.isfinite(o).all(), n
    assert (o != 99).any(), n
G.check_norm(x, None, w, (got["h"], got["q"], got["s"]))
G.check_attn(q1, cache, kv, None, True, 1, got["one"])
print("done")
"""


@pytest.mark.parametrize("K", [256, 24575])
def test_every_first_call_captured(K):
    """Each operator's first call of a process in a capture (norm rows in registers and in shared memory,
    many and few rows of attention): what the replay writes is what the eager calls write."""
    fresh_process(_CAPTURED % K)


# ------------------------------------------------------------------ device status

_STATUS = r"""
#include "dollama_b200/csrc/common.cu"
#include "dollama_b200/csrc/attention_kv.cuh"
using namespace dlm;
// a barrier that nothing arrives on: the wait gives up after its two seconds
__global__ void give_up(int* status) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  abort_flag = 0;
  mbar_init(&bar, 1);
  fence_mbar_init();
  mbar_wait(&bar, 0, &abort_flag, status, kDevTimeoutMma);
}
// the attention's own check of a length outside its cache
__global__ void bad_length(const AttnKvParams p) { AttnKvTile(p, 0, 8, true); }
int read(int clear) {
  int c = -1;
  return dlm_get_device_status(&c, clear, nullptr) == DLM_OK ? c : -2;
}
int main() {
  const int five = 5;
  int* n = nullptr;
  if (cudaMalloc(&n, 4) != cudaSuccess || cudaMemcpy(n, &five, 4, cudaMemcpyHostToDevice) != cudaSuccess) return 1;
  AttnKvParams p{};
  p.kv_len = n;
  p.Lmax = 4;
  p.Sq = p.Hkv = p.Hq = p.g = p.B = p.row_tiles = p.tiles = 1;
  p.status = device_status_ptr();
  p.bad_position = device_position_ptr();
  printf("%d ", read(1));
  bad_length<<<1, 1>>>(p);
  printf("%d ", read(0));
  printf("%d ", read(1));
  printf("%d ", read(1));
  bad_length<<<1, 1>>>(p);
  give_up<<<1, 1>>>(p.status);
  bad_length<<<1, 1>>>(p);
  printf("%d ", read(0));
  printf("%d ", read(1));
  printf("%d ", read(1));
  printf("%d\n", read(1));
  return cudaDeviceSynchronize() == cudaSuccess ? 0 : 1;
}
"""


def test_a_bad_length_does_not_hide_a_timeout(tmp_path):
    """A kernel that gave up a wait is reported whatever bad positions came before it; they are reported
    after it."""
    src, exe = tmp_path / "status.cu", tmp_path / "status"
    src.write_text(_STATUS.replace("\n#include \"", "\n#include \"" + ROOT + "/"))
    r = subprocess.run([nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17",
                        "--expt-relaxed-constexpr", "-I", ROOT + "/include", "-o", str(exe), str(src)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.split() == "0 6 6 0 2 2 6 0".split(), r.stdout + r.stderr


# ------------------------------------------------------------------ attention: any finite scale

@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-6, 4.0])
@pytest.mark.parametrize("Sq", [1, 8, 40])
def test_attention_scale(t, scale, Sq):
    """No weight but equal ones, the lowest scores first, and rows that one key takes."""
    g, ty = gen(Sq), O.TYPES[t]
    q = torch.randn(2, Sq, 4, 64, generator=g, device="cuda").to(ty)
    cache = G.make_cache(2, 2, 200, 64, g)
    kv = torch.tensor([200, 77], dtype=torch.int32, device="cuda")
    out = G.run_attn(q, cache, kv, None, True, t, scale=scale)
    G.check_attn(q, cache, kv, None, True, t, out, scale=scale)
