"""The int8 language-model operators where their launch rules and main loops change form: rows just
below a kernel's shared-memory limit, rings used many times over, references that move late, keys and
rows that must not touch one another.  Tolerances and 64-bit forms are those of test_lm_i8_gpu."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from dollama_b200 import _lib as L
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
