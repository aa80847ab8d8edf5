"""Plain 64-bit forms of the 4-bit KV cache and of what runs around it (livecc_amd/csrc/kv4.hip), for its tests: written from the definitions in
include/livecc_amd.h, on the CPU, without the product's code."""
import math

import torch

D = 128
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def b16(x):
    """the nearest bf16, as a 64-bit value (fp32 values and 64-bit ones that fp32 holds)"""
    return x.float().to(torch.bfloat16).double()


def quantise(x):
    """(codes, exponents, values) of bf16-valued rows [..., 128]: nearest of +-VALUES (ties to the even code) under the smallest 2^(e - 127), 2 <= e <= 252, with
    seven of it no less than the group's largest magnitude; a group that is not finite: 255 and NaN."""
    g = x.double().unflatten(-1, (4, 32))
    a = g.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(g).all(-1, keepdim=True)
    e = torch.full_like(a, 2.0)
    for k in range(2, 252):                        # the definition, step by step: while seven of the scale are too few, the next
        e = torch.where((e == k) & (7 * 2.0 ** (k - 127) < a), float(k + 1), e)
    v = torch.where(fine, g, torch.zeros_like(g)) / torch.pow(2.0, e - 127)
    far = (v.abs().unsqueeze(-1) - VALUES).abs()
    even = torch.arange(8, dtype=torch.float64) % 2 * 1e-12
    code = (far + even).argmin(-1)
    sign = torch.signbit(v)
    val = torch.where(sign, -VALUES[code], VALUES[code]) * torch.pow(2.0, e - 127)
    val = torch.where(fine, val, torch.full_like(val, math.nan))
    codes = torch.where(fine, code + 8 * sign, torch.zeros_like(code))
    return codes.flatten(-2), torch.where(fine, e, torch.full_like(e, 255.0)).squeeze(-1), val.flatten(-2)


def norm_rope(x, w, cos, sin, eps=1e-6):
    """heads [S, H, 128] (bf16 values) -> the same normed (w None: not) and rotated, with the model's rounding points; tables [S, 64]"""
    x = x.double()
    if w is not None:
        r = (1.0 / (x.pow(2).mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))).sqrt()).float().double()
        x = b16(w.double() * b16((x * r).float()))
    c, s = cos.double()[:, None], sin.double()[:, None]
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat((b16(b16(lo * c) - b16(hi * s)), b16(b16(hi * c) + b16(lo * s))), -1)


def attention(q, k, v, lim):
    """(out, tolerance) of q [S, Hq, 128] over k, v [Hkv, L, 128], row s seeing keys 0 .. lim[s] (none below 0: zeros), all in 64 bits.

    Tolerance of a kernel that multiplies bf16 with fp32 sums and rounds its probabilities and its result to bf16 (half a step: 2^-8 of the value):
    2^-8 |out| for the result, 2^-8 A with A = sum p |v| / sum p for the probabilities; a score is off by at most 128 half steps of fp32 of sum |q k| / sqrt(128)
    and twice its own size in half steps (scaling, subtraction), which the exponential turns into a relative error of p, in numerator and denominator;
    the exponential itself, the sums over keys (they are joined pairwise within tiles) and the merges: 2^-16 A covers 256 half steps."""
    S, Hq, _ = q.shape
    Hkv, L, _ = k.shape
    G = Hq // Hkv
    out, tol = torch.zeros(S, Hq, D, dtype=torch.float64), torch.zeros(S, Hq, D, dtype=torch.float64)
    for h in range(Hq):
        kk, vv = k[h // G].double(), v[h // G].double()
        for s in range(S):
            n = int(min(lim[s] + 1, L))
            if n <= 0:
                continue
            qs = q[s, h].double()
            sc = kk[:n] @ qs / math.sqrt(D)
            p = torch.softmax(sc, 0)
            out[s, h] = p @ vv[:n]
            A = p @ vv[:n].abs()
            d = 2.0 ** -24 * (128 * (kk[:n].abs() @ qs.abs()).max() / math.sqrt(D) + 4 * sc.abs().max())
            tol[s, h] = 2.0 ** -8 * out[s, h].abs() + (2.0 ** -8 + 2.0 ** -16 + 2 * d) * A
    return out, tol


def assert_within(got, want, tol, what=""):
    got, want = got.double().cpu().reshape(want.shape), want
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = torch.isnan(want) | ((got - want).abs() <= tol + 1e-30)
    worst = ((got - want).abs() / (tol + 1e-30)).nan_to_num(0.0).max().item()
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} beyond the tolerance, worst {worst:.3g} of it"
