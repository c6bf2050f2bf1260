"""Plain 64-bit forms of the int8 language-model operators (the formulas of
include/dollama_b200.h), for the parity tests."""
import torch

TYPES = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}  # dlm_dtype
U24 = 2.0 ** -24  # half a step of fp32, relative


def half_eps(t):
    return torch.finfo(t).eps / 2


def half_tiny(t):
    """Half a step of the type's subnormals."""
    f = torch.finfo(t)
    return f.tiny * f.eps / 2


def half_away(v):
    return torch.sign(v) * torch.floor(v.abs() + 0.5)


def quant_rows(x):
    """Codes (int8) and scales (64 bits) of the last dimension's rows.  127 x / a in double is the
    quotient correctly rounded, exact ties included, for x of up to 46 bits."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(a) | torch.isnan(x).any(-1, keepdim=True)
    q = half_away(127.0 * x / a)
    q = torch.where((a == 0) | bad, torch.zeros_like(q), q)
    scale = torch.where(bad, torch.full_like(a, float("nan")), a / 127.0)
    return q.to(torch.int8), scale[..., 0]


def add_rms_norm(x, r, w, eps):
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    p = h.double() * w.double()
    q, s = quant_rows(p)
    rms = torch.sqrt(h.double().pow(2).mean(-1) + eps)
    return h, q, s / rms


def gemm(xq, xs, wq, ws, bias):
    """y and the magnitude of its scaled product."""
    y = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    return (y if bias is None else y + bias.double()), y.abs()


def attention(q, kq, ks, vq, vs, kv_len, q_len, causal, scale):
    """out [B, Sq, Hq, Dh] in 64 bits (zeros for queries from q_len on) and the bound of a
    kernel's absolute error before the rounding of its output, for weights rounded with relative
    error `w_eps` (the second result is a function of it)."""
    B, Sq, Hq, Dh = q.shape
    Hkv, L = kq.shape[1], kq.shape[2]
    g = Hq // Hkv
    out = torch.zeros(B, Sq, Hq, Dh, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)                       # sum p |v|
    eps_s = torch.zeros(B, Sq, Hq, 1, dtype=torch.float64, device=q.device)
    terms = torch.zeros(B, 1, 1, 1, dtype=torch.float64, device=q.device)
    floor = torch.zeros_like(eps_s)
    for b in range(B):
        n, m = min(max(int(kv_len[b]), 0), L), Sq if q_len is None else min(int(q_len[b]), Sq)
        terms[b] = n
        for i in range(m):
            seen = min(n, n - m + i + 1) if causal else n
            if seen <= 0:
                continue
            for h in range(Hq):
                k = kq[b, h // g, :seen].double() * ks[b, h // g, :seen, None].double()
                v = vq[b, h // g, :seen].double() * vs[b, h // g, :seen, None].double()
                s = (k @ q[b, i, h].double()) * scale
                p = torch.softmax(s, 0)
                out[b, i, h] = p @ v
                mass[b, i, h] = p @ v.abs()
                # weights p vscale are held in fp16 terms scaled so that the row's largest is 2^10 or
                # more: one below 2^-14 is off by half a subnormal step, 2^-25, which is 2^-35 of the
                # largest (fp32: 2^12, 2^-37), times a code of at most 127, for each of n keys
                floor[b, i, h] = seen * 127 * 2.0 ** (-37 if q.dtype == torch.float32 else -35) * (p * vs[b, h // g, :seen].double().abs()).max()
                big = (k.abs() @ q[b, i, h].double().abs()).max() * abs(scale)
                # score error: Dh products summed in fp32 (each partial sum rounded or cut: 2^-23), q
                # held to 2^-22, three fp32 factors and the subtraction of the maximum (2^-23 each of
                # at most 2 |s|); exp2 itself 2^-22, summed weights 2^-22
                eps_s[b, i, h] = big * (Dh + 16) * 2.0 ** -23 + 2.0 ** -20
    def bound(w_eps):
        # numerator and denominator both move by eps_s; sums over n keys: 16 at a time, then one
        # addition for every 16 keys and the joins of warps and blocks
        return mass * (2 * eps_s + w_eps + (terms / 16 + 96) * 2.0 ** -23) + floor
    return out, bound
