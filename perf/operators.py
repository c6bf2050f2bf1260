"""The int8 language-model operators as cases to be measured: RMS norm with residual and int8 output,
int8 matrix product with token and channel scales, int8 K/V cache write and read-back, and attention
over that cache.  `run` computes them in elementary torch operations, or, with `own` set, through the
library's entry points.  `exact` gives the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"f32": 0, "f16": 1, "bf16": 2}  # dlm_dtype
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of the tag LM (d_model 512) for a handful of sequences: launch latency
        dict(name="norm_decode_8x512", op="norm", M=8, K=512, dtype="f32", residual=True),
        # a ragged batch of prompts, rows of an odd length that no vector width divides
        dict(name="norm_ragged_1003x1531", op="norm", M=1003, K=1531, dtype="bf16", residual=True),
        # a long prefill of a wide model
        dict(name="norm_prefill_16384x4096", op="norm", M=16384, K=4096, dtype="f16", residual=True),
        # the tag LM's q|k|v projection for a few sequences: launch latency
        dict(name="gemm_decode_8x1536x512", op="gemm", M=8, N=1536, K=512, dtype="f32", bias=False),
        # a batch of 32 single tokens against a 4096 x 4096 weight: the weight's bytes count
        dict(name="gemm_decode_32x4096x4096", op="gemm", M=32, N=4096, K=4096, dtype="f16", bias=False),
        # a ragged prompt batch, odd numbers of tokens and channels, with a bias
        dict(name="gemm_ragged_1003x2111x1360", op="gemm", M=1003, N=2111, K=1360, dtype="bf16", bias=True),
        # a long prefill: the tensor cores' rate counts
        dict(name="gemm_prefill_8192x8192x4096", op="gemm", M=8192, N=8192, K=4096, dtype="f16", bias=False),
        # 256 sequences of the tag LM (8 heads of 64, 128 positions) store one token each and read it back
        dict(name="kv_decode_256x8x64", op="kv", B=256, S=1, H=8, Dh=64, L=128, dtype="f32", ragged=False),
        # ragged prompts stored and read back
        dict(name="kv_prefill_16x2048x8x128", op="kv", B=16, S=2048, H=8, Dh=128, L=2304, dtype="f16", ragged=True),
        # one decode step of 256 tag LM sequences at up to 128 positions
        dict(name="attn_decode_256x8x64_L128", op="attn", B=256, Sq=1, Hq=8, Hkv=8, Dh=64, L=128, dtype="f32"),
        # one decode step over long caches with heads that share keys
        dict(name="attn_decode_8x32x128_L16384", op="attn", B=8, Sq=1, Hq=32, Hkv=8, Dh=128, L=16384, dtype="f16"),
        # a chunk of a prompt against the cache of what came before it
        dict(name="attn_chunk_2x500x16x64_L4096", op="attn", B=2, Sq=500, Hq=16, Hkv=4, Dh=64, L=4096, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "gemm", "kv", "attn"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        K = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            K = (K + 7) // 8 * 8
        M = _log(rng, 1, min(16384, 16384 * 2048 // K))
        return dict(op=op, M=M, K=K, dtype=dtype, residual=rng.random() < 0.8)
    if op == "gemm":
        K = 16 * _log(rng, 4, 512)
        N = _log(rng, 32, 8192)
        M = _log(rng, 1, min(8192, (1 << 36) // (N * K)) or 1)
        return dict(op=op, M=M, N=N, K=K, dtype=dtype, bias=rng.random() < 0.5)
    Dh = rng.choice([64, 128])
    if op == "kv":
        H = rng.choice([1, 2, 4, 8, 16])
        if rng.random() < 0.5:
            B, S = _log(rng, 1, 512), rng.randint(1, 4)
        else:
            B, S = _log(rng, 1, 16), _log(rng, 16, 2048)
        return dict(op=op, B=B, S=S, H=H, Dh=Dh, L=S + _log(rng, 1, 512), dtype=dtype, ragged=rng.random() < 0.5)
    Hkv, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8])
    L = _log(rng, 16, 16384)
    if rng.random() < 0.6:
        Sq = rng.randint(1, 4)
        B = _log(rng, 1, max(1, min(256, (1 << 20) // (L * Hkv))))
    else:
        L = max(32, L // 4)
        Sq = min(_log(rng, 5, 1000), L)
        B = _log(rng, 1, max(1, min(16, (1 << 25) // (L * Sq * Hkv * g))))
    return dict(op=op, B=B, Sq=min(Sq, L), Hq=Hkv * g, Hkv=Hkv, Dh=Dh, L=L, dtype=dtype)


def _lengths(c, seed):
    """Cache lengths and query counts of an attention case, from the seed (host integers)."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    B, L, Sq = c["B"], c["L"], c["Sq"]
    kv = torch.randint(max(Sq, L // 2), L + 1, (B,), generator=g)
    return kv


def work(c):
    e = _BYTES[c["dtype"]]
    if c["op"] == "norm":
        n = c["M"] * c["K"]
        # x, residual and the weight in; the sum, the values the codes stand for and the scales out
        return {"bytes": n * e * (4 if c["residual"] else 3) + c["K"] * e + 4 * c["M"], "flops": 6 * n}
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": M * K + N * K + e * M * N + 4 * (M + N) + (e * N if c["bias"] else 0),
                "flops": 2 * M * N * K}
    if c["op"] == "kv":
        rows = c["B"] * c["S"] * c["H"]
        if c["ragged"]:
            rows = rows * 3 // 4
        # k, v in; codes and scales written and read; the values out
        return {"bytes": 2 * rows * (2 * c["Dh"] * e + 2 * c["Dh"] + 8), "flops": 2 * rows * 4 * c["Dh"]}
    keys = c["B"] * max(c["Sq"], c["L"] * 3 // 4)
    seen = c["B"] * c["Sq"] * (max(c["Sq"], c["L"] * 3 // 4) - (c["Sq"] - 1) / 2)
    return {"bytes": 2 * keys * c["Hkv"] * (c["Dh"] + 4) + 2 * c["B"] * c["Sq"] * c["Hq"] * c["Dh"] * e,
            "flops": 4 * c["Dh"] * c["Hq"] * seen}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _quant_rows(x):
    """Codes and scales of a user's stored int8 weights or cache rows (made once, outside the call)."""
    a = x.abs().amax(-1, keepdim=True).clamp_min(1e-20)
    return torch.round(x * (127.0 / a)).clamp_(-127, 127).to(torch.int8), (a[..., 0] / 127.0)


def prepare(case, seed):
    c, g, dev = dict(case), _gen(seed), "cuda"
    t = _TYPES[c["dtype"]]
    if c["op"] == "norm":
        M, K = c["M"], c["K"]
        big = 1 + 12 * (torch.rand(K, generator=g, device=dev) < 0.01).float()  # a few loud channels
        x = (torch.randn(M, K, generator=g, device=dev) * big).to(t)
        r = (2 * torch.randn(M, K, generator=g, device=dev) * big).to(t) if c["residual"] else None
        w = (1 + 0.1 * torch.randn(K, generator=g, device=dev)).to(t)
        return dict(c, x=x, r=r, w=w, h=torch.empty_like(x), y=torch.empty_like(x),
                    q=torch.empty(M, K, dtype=torch.int8, device=dev), s=torch.empty(M, device=dev))
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        xq, xs = _quant_rows(torch.randn(M, K, generator=g, device=dev))
        wq, ws = _quant_rows(torch.randn(N, K, generator=g, device=dev) / math.sqrt(K))
        b = (0.1 * torch.randn(N, generator=g, device=dev)).to(t) if c["bias"] else None
        return dict(c, xq=xq, xs=xs, wq=wq, ws=ws, b=b, y=torch.empty(M, N, dtype=t, device=dev))
    if c["op"] == "kv":
        B, S, H, Dh, L = c["B"], c["S"], c["H"], c["Dh"], c["L"]
        k = (2 * torch.randn(B, S, H, Dh, generator=g, device=dev)).to(t)
        v = torch.randn(B, S, H, Dh, generator=g, device=dev).to(t)
        pos = torch.randint(0, L - S + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        n = torch.randint(S // 2, S + 1, (B,), generator=g, device=dev, dtype=torch.int32) if c["ragged"] else None
        kq, vq = (torch.zeros(B, H, L, Dh, dtype=torch.int8, device=dev) for _ in range(2))
        ks, vs = (torch.zeros(B, H, L, device=dev) for _ in range(2))
        return dict(c, k=k, v=v, pos=pos, n=n, kq=kq, vq=vq, ks=ks, vs=vs, ko=torch.zeros_like(k),
                    vo=torch.zeros_like(v))
    B, Sq, Hq, Hkv, Dh, L = (c[n] for n in ("B", "Sq", "Hq", "Hkv", "Dh", "L"))
    q = (1.5 * torch.randn(B, Sq, Hq, Dh, generator=g, device=dev)).to(t)
    kq, ks = _quant_rows(torch.randn(B, Hkv, L, Dh, generator=g, device=dev))
    vq, vs = _quant_rows(torch.randn(B, Hkv, L, Dh, generator=g, device=dev))
    n = _lengths(c, seed).to(dev, torch.int32)
    return dict(c, q=q, kq=kq, ks=ks, vq=vq, vs=vs, n=n, o=torch.empty_like(q))


# ------------------------------------------------------------------ the library's calls

def _p(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    from dollama_b200 import _lib as L
    stream = torch.cuda.current_stream().cuda_stream
    t = _CODES[s["dtype"]]
    if s["op"] == "norm":
        M, K = s["M"], s["K"]
        L.call("dlm_add_rms_norm_i8", _p(s["x"]), K, _p(s["r"]), K, _p(s["w"]), _p(s["h"]), K, _p(s["q"]),
               _p(s["s"]), M, K, 1e-5, t, stream)
        torch.mul(s["q"], s["s"][:, None], out=s["y"])
        return {"h": s["h"], "y": s["y"], "scale": s["s"]}
    if s["op"] == "gemm":
        M, N, K = s["M"], s["N"], s["K"]
        L.call("dlm_gemm_i8", _p(s["xq"]), K, _p(s["xs"]), _p(s["wq"]), _p(s["ws"]), _p(s["b"]), _p(s["y"]), N,
               M, N, K, t, stream)
        return s["y"]
    if s["op"] == "kv":
        B, S, H, Dh, Lm = (s[n] for n in ("B", "S", "H", "Dh", "L"))
        cache = (_p(s["kq"]), _p(s["ks"]), _p(s["vq"]), _p(s["vs"]))
        shape = (B, S, H, Dh, Lm, _p(s["pos"]), _p(s["n"]), t, stream)
        L.call("dlm_kv_i8_append", _p(s["k"]), H * Dh, _p(s["v"]), H * Dh, *cache, *shape)
        L.call("dlm_kv_i8_read", *cache, _p(s["ko"]), H * Dh, _p(s["vo"]), H * Dh, *shape)
        return {"k": s["ko"], "v": s["vo"], "ks": s["ks"], "vs": s["vs"]}
    B, Sq, Hq, Hkv, Dh, Lm = (s[n] for n in ("B", "Sq", "Hq", "Hkv", "Dh", "L"))
    L.call("dlm_attention_kv_i8", _p(s["q"]), Hq * Dh, _p(s["kq"]), _p(s["ks"]), _p(s["vq"]), _p(s["vs"]),
           _p(s["o"]), Hq * Dh, B, Hq, Hkv, Sq, Dh, Lm, _p(s["n"]), None, 1, 1 / math.sqrt(Dh), t, stream)
    return s["o"]


# ------------------------------------------------------------------ the plain forms

def _half_away(v):
    return torch.trunc(v + torch.copysign(torch.full_like(v, 0.5), v))


def _plain_norm(s):
    t = s["x"].dtype
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(t)
    f = h.float()
    inv = torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-5)
    # codes lie next to a border now and then: the quotient in 64 bits
    p = h.double() * s["w"].double()
    a = p.abs().amax(-1, keepdim=True)
    q = _half_away(127.0 * p / a).clamp(-127, 127).float()
    scale = a.float() * inv / 127.0
    return {"h": h, "y": (q * scale).to(t), "scale": scale[:, 0]}


def _plain_gemm(s):
    y = s["xq"].float() @ s["wq"].float().t() * s["xs"][:, None] * s["ws"]
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(s["y"].dtype)


def _plain_rows(x):
    a = x.abs().amax(-1, keepdim=True)
    q = _half_away(127.0 * x.double() / a.double()).clamp(-127, 127)
    return q.to(torch.int8), (a.float() / 127.0)[..., 0]


def _plain_kv(s):
    B, S, L = s["B"], s["S"], s["L"]
    dev = s["k"].device
    b = torch.arange(B, device=dev)[:, None]
    at = s["pos"].long()[:, None] + torch.arange(S, device=dev)
    live = torch.ones(B, S, dtype=torch.bool, device=dev)
    if s["n"] is not None:
        live = torch.arange(S, device=dev) < s["n"][:, None]
    out = {}
    for x, cq, cs, o, name in ((s["k"], s["kq"], s["ks"], s["ko"], "k"), (s["v"], s["vq"], s["vs"], s["vo"], "v")):
        q, sc = _plain_rows(x)  # [B, S, H, Dh], [B, S, H]
        cq[b, :, at] = torch.where(live[..., None, None], q, cq[b, :, at])
        cs[b, :, at] = torch.where(live[..., None], sc, cs[b, :, at])
        back = cq[b, :, at].float() * cs[b, :, at][..., None]
        o.copy_(torch.where(live[..., None, None], back.to(o.dtype), o))
        out[name], out[name + "s"] = o, cs
    return out


def _plain_attn(s):
    B, Sq, Hq, Hkv, Dh, L = (s[n] for n in ("B", "Sq", "Hq", "Hkv", "Dh", "L"))
    g = Hq // Hkv
    k = s["kq"].float() * s["ks"][..., None]
    v = s["vq"].float() * s["vs"][..., None]
    q = s["q"].float().view(B, Sq, Hkv, g, Dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * Sq, Dh)
    w = (q @ k.transpose(-1, -2) * (1 / math.sqrt(Dh))).view(B, Hkv, g, Sq, L)
    n = s["n"].long()[:, None, None]
    i = torch.arange(Sq, device=q.device)[:, None]
    j = torch.arange(L, device=q.device)
    hidden = j > n - Sq + i  # [B, Sq, L]
    w = w.masked_fill(hidden[:, None, None], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = w.view(B, Hkv, g * Sq, L) @ v
    return o.view(B, Hkv, g, Sq, Dh).permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, Dh).to(s["q"].dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "gemm": _plain_gemm, "kv": _plain_kv, "attn": _plain_attn}[state["op"]](state)


# ------------------------------------------------------------------ 64 bits

def _away64(v):
    return torch.sign(v) * torch.floor(v.abs() + 0.5)


def exact(case, seed):
    s = prepare(case, seed)
    t = _TYPES[s["dtype"]]
    if s["op"] == "norm":
        # the sum is held in the inputs' type: what is stored is what is normed
        total = s["x"].double()
        if s["r"] is not None:
            total = total + s["r"].double()
        h = total.to(t).double()
        y = h / torch.sqrt(h.pow(2).sum(1) / s["K"] + 1e-5)[:, None] * s["w"].double()
        top = y.abs().max(1).values[:, None]
        return {"h": h, "y": _away64(y * 127 / top) * top / 127, "scale": top[:, 0] / 127}
    if s["op"] == "gemm":
        y = torch.mm(s["xq"].double(), s["wq"].double().T)
        y = torch.einsum("mn,m,n->mn", y, s["xs"].double(), s["ws"].double())
        return y if s["b"] is None else y + s["b"].double()
    if s["op"] == "kv":
        out = {n: torch.zeros_like(s["k"], dtype=torch.float64) for n in ("k", "v")}
        out |= {n: torch.zeros_like(s["ks"], dtype=torch.float64) for n in ("ks", "vs")}
        pos = s["pos"].tolist()
        num = s["n"].tolist() if s["n"] is not None else [s["S"]] * s["B"]
        for b in range(s["B"]):
            for n in ("k", "v"):
                x = s[n][b, :num[b]].double()
                top = x.abs().max(-1).values
                out[n][b, :num[b]] = _away64(x / top[..., None] * 127) * top[..., None] / 127
                out[n + "s"][b, :, pos[b]:pos[b] + num[b]] = top.T / 127
        return out
    B, Sq, Hq, Hkv, Dh = (s[n] for n in ("B", "Sq", "Hq", "Hkv", "Dh"))
    if 4.0 * Dh * Hq * B * Sq * s["L"] > 1e13:
        return None
    out = torch.empty(B, Sq, Hq, Dh, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["n"].tolist()):
        see = torch.ones(Sq, n, dtype=torch.bool, device="cuda").tril(n - Sq)
        for m in range(Hkv):
            keys = s["kq"][b, m, :n].double() * s["ks"][b, m, :n, None].double()
            vals = s["vq"][b, m, :n].double() * s["vs"][b, m, :n, None].double()
            for h in range(m * Hq // Hkv, (m + 1) * Hq // Hkv):
                z = s["q"][b, :, h].double() @ keys.T / math.sqrt(Dh)
                e = torch.where(see, torch.exp(z - torch.where(see, z, -math.inf).max(1, keepdim=True).values), 0.0)
                out[b, :, h] = (e @ vals) / e.sum(1, keepdim=True)
    return out
