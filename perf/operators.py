"""A layer's attention with its keys and values held in 4 bits, as cases that can be timed and checked: the pass between the q|k|v projection and the
cache (norms per head, rotation, append -- into the bf16 cache and into the 4-bit one), the attention of single tokens and of chunks over the 4-bit
cache.  `listed()` are fixed cases, `draw` gives others of the same ranges.  A case is a dict of plain values; `prepare` makes what a program holds
before the call (rows, tables, filled caches, the launch plan), `run` is one pass, `work` what it cannot do without, `exact` the outputs in 64 bits.

The 4-bit cache: groups of 32 channels of one token and KV head, 16 values of 4 bits (sign, 0 .5 1 1.5 2 3 4 6) and one power of two, 2^(e - 127).
A slot is [layer][K codes | V codes | K scales | V scales] bytes:
  K codes  [head][position][64]                byte b: channels 2 b (low half) and 2 b + 1
  V codes  [head][position / 32][4][16][4][8]  byte (g, i, t, e): position 8 g + e of the block, channels 32 t + i (low half) and 32 t + 16 + i
  K scales [head][position][4]                 e of channels 32 t .. 32 t + 31
  V scales [head][position / 32][4][4][8]      byte (g, t, e)
"""
import math

import torch

own = False
DEVICE = "cuda"
D = 128
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_PAIRS = 8 * 340 * 5000 * 28          # (row, key, head) products of the largest listed chunk
MOST_KEYS = 64 * 4000 * 4                 # (key, KV head) pairs of the largest listed decode step
MOST_ROWS = 9048 * 36                     # (row, head) pairs of the largest listed append


def listed():
    return [
        # the token of one stream between projection and attention: every layer of every decode step; latency alone
        dict(name="append_1", kind="append", bits=16, heads=28, kv_heads=4, streams=1, rows=1, spread=0, past=6501, idle=0),
        # one tick of live commentary (two new frames and their text) on a stream that has run for a while
        dict(name="append_386", kind="append", bits=16, heads=28, kv_heads=4, streams=1, rows=386, spread=0, past=2003, idle=0),
        # the first turns of eight streams in one call
        dict(name="append_8x1131", kind="append", bits=16, heads=28, kv_heads=4, streams=8, rows=1131, spread=0, past=0, idle=0),
        # a decode step of eight streams of the smaller model, three of its rows idle, into the 4-bit cache; what was written is read back
        dict(name="append4_8", kind="append", bits=4, heads=12, kv_heads=2, streams=8, rows=1, spread=0, past=1777, idle=3),
        # a tick into the 4-bit cache
        dict(name="append4_386", kind="append", bits=4, heads=28, kv_heads=4, streams=1, rows=386, spread=0, past=6501, idle=0),
        # first turns of unequal length, the large model's heads
        dict(name="append4_4x1131", kind="append", bits=4, heads=64, kv_heads=8, streams=4, rows=1131, spread=300, past=0, idle=0),
        # a token of a young stream
        dict(name="decode4_517", kind="decode", heads=28, kv_heads=4, streams=1, keys=517, spread=0),
        # a token of a stream at the end of its window, the large model's heads
        dict(name="decode4_32k", kind="decode", heads=64, kv_heads=8, streams=1, keys=32767, spread=0),
        # the widest decode batch, histories of unequal length
        dict(name="decode4_64x6k", kind="decode", heads=28, kv_heads=4, streams=64, keys=6000, spread=4000),
        # a short question asked late in a stream
        dict(name="chunk4_17", kind="chunk", heads=28, kv_heads=4, streams=1, rows=17, spread=0, past=26800, past_spread=0),
        # one tick
        dict(name="chunk4_386", kind="chunk", heads=28, kv_heads=4, streams=1, rows=386, spread=0, past=6120, past_spread=0),
        # the ticks of eight streams together, chunks and histories of unequal length
        dict(name="chunk4_8x386", kind="chunk", heads=28, kv_heads=4, streams=8, rows=386, spread=100, past=6400, past_spread=3000),
    ]


def between(rng, lo, hi):
    """Whole number, spread over the logarithm of the range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((28, 4), (12, 2), (64, 8), (2, 1), (7, 1), (8, 8), (32, 2))


def draw(rng):
    heads, kv_heads = rng.choice(HEADS)
    case = dict(kind=rng.choice(("append", "append", "decode", "decode", "chunk", "chunk")), heads=heads, kv_heads=kv_heads)
    if case["kind"] == "append":
        streams, rows = between(rng, 1, 64), between(rng, 1, 1131)
        while streams * rows * (heads + 2 * kv_heads) > MOST_ROWS:
            streams = max(1, streams // 2)
        return dict(case, bits=rng.choice((16, 4)), streams=streams, rows=rows, spread=rng.randrange(0, max(1, rows // 2)), past=rng.choice((0, between(rng, 1, 8000))),
                    idle=rng.randrange(0, streams * rows // 4 + 1))
    if case["kind"] == "decode":
        streams, keys = between(rng, 1, 64), between(rng, 1, 32767)
        while streams * keys * kv_heads > MOST_KEYS:
            keys = max(1, keys * 2 // 3)
        return dict(case, streams=streams, keys=keys, spread=rng.randrange(0, keys))
    streams, rows, past = between(rng, 1, 16), between(rng, 2, 1131), rng.choice((0, between(rng, 1, 26800)))
    while streams * rows * (rows + past) * heads > MOST_PAIRS:
        streams, rows, past = max(1, streams * 2 // 3), max(2, rows * 5 // 6), past * 5 // 6
    return dict(case, streams=streams, rows=rows, spread=rng.randrange(0, max(1, rows // 2)), past=past, past_spread=rng.randrange(0, past + 1))


def up(n, m):
    return (n + m - 1) // m * m


def sizes(case):
    """New rows, history and capacity: of each stream, of each stream, of every slot.  The first stream has the longest of both."""
    n = case["streams"]
    less = [(k * 7919) % n / n for k in range(n)]
    if case["kind"] == "decode":
        rows, past = [1] * n, [case["keys"] - 1 - int(u * case["spread"]) for u in less]
    else:
        rows = [case["rows"] - int(u * case["spread"]) for u in less]
        past = [case["past"] - int(u * case.get("past_spread", case["past"] // 2)) for u in less]
    return rows, past, up(max(r + p for r, p in zip(rows, past)), 32)


# ---- the 4-bit format in elementary operations
def encode(x):
    """bf16 rows [..., 128] -> (halves [..., 128] uint8, exponents [..., 4] uint8)."""
    g = x.float().unflatten(-1, (4, 32))
    a = g.abs().amax(-1)
    bits = a.to(torch.bfloat16).view(torch.int16).int()
    e = (((bits + 31) >> 7) - 2).clamp(2, 252)
    fine = torch.isfinite(a)
    v = torch.where(fine.unsqueeze(-1), torch.ldexp(g, (127 - e).unsqueeze(-1)), 0.0)
    m = v.abs()
    code = (m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0) + 8 * torch.signbit(v)
    return code.to(torch.uint8).flatten(-2), torch.where(fine, e, 255).to(torch.uint8)


def decode(halves, e):
    """The values of halves [..., 128] under exponents [..., 4], fp32."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=halves.device)
    s = torch.where(e == 255, math.nan, torch.ldexp(torch.ones((), device=e.device), e.int() - 127))
    return (table[halves.int()].unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten(-2)


def parts(buf, kv_heads, lmax):
    """K codes, V codes, K scales, V scales of slots [n, bytes] (one layer), as views."""
    n, c, s = buf.shape[0], kv_heads * lmax * 64, kv_heads * lmax * 4
    k, v, ks, vs = buf.split((c, c, s, s), dim=1)
    return (k.view(n, kv_heads, lmax, 64), v.view(n, kv_heads, lmax // 32, 4, 16, 4, 8), ks.view(n, kv_heads, lmax, 4), vs.view(n, kv_heads, lmax // 32, 4, 4, 8))


def fill(buf, kv_heads, lmax, k, v):
    """Slots that hold keys and values [n, kv_heads, lmax, 128]."""
    kc, vc, ks, vs = parts(buf, kv_heads, lmax)
    h, e = encode(k)
    kc.copy_(h[..., 0::2] | h[..., 1::2] << 4)
    ks.copy_(e)
    h, e = encode(v)
    h = h.unflatten(-1, (4, 2, 16)).unflatten(2, (lmax // 32, 4, 8))                   # n, head, block, g, e, t, half, i
    vc.copy_((h[..., 0, :] | h[..., 1, :] << 4).permute(0, 1, 2, 3, 6, 5, 4))
    vs.copy_(e.unflatten(2, (lmax // 32, 4, 8)).permute(0, 1, 2, 3, 5, 4))


def codes_k(kc):
    return torch.stack((kc & 15, kc >> 4), -1).flatten(-2)


def codes_v(vc):
    """[n, head, block, g, i, t, e] bytes -> [n, head, position, 128] halves."""
    return torch.stack((vc & 15, vc >> 4), -1).permute(0, 1, 2, 3, 6, 5, 7, 4).flatten(5).flatten(2, 4)


def unpack(buf, kv_heads, lmax, keys):
    """Keys and values [n, kv_heads, keys, 128] of the slots' first positions, fp32."""
    kc, vc, ks, vs = parts(buf, kv_heads, lmax)
    b = up(keys, 32) // 32
    k = decode(codes_k(kc[:, :, :keys]), ks[:, :, :keys])
    v = decode(codes_v(vc[:, :, :b]), vs[:, :, :b].permute(0, 1, 2, 3, 5, 4).flatten(2, 4))
    return k, v[:, :, :keys]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    rows, past, lmax = sizes(case)
    n, heads, kv_heads = case["streams"], case["heads"], case["kv_heads"]
    f = lambda *s: torch.randn(*s, generator=g, device=DEVICE)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    stream = [s for s in range(n) for _ in range(rows[s])]
    pos = [past[s] + r for s in range(n) for r in range(rows[s])]
    st = dict(kind=case["kind"], heads=heads, kv_heads=kv_heads, lmax=lmax, rows=len(stream), n=n)
    # channels of keys differ in size by a factor of a few, as they do in trained models; a stream's first token has a key and a value of its own kind
    size = torch.exp(0.5 * f(kv_heads, 1, D))
    if case["kind"] == "append":
        st.update(bits=case["bits"])
        st["qkv"] = torch.cat((f(len(stream), heads * D), f(len(stream), kv_heads * D) * size.view(-1), f(len(stream), kv_heads * D)), 1).to(torch.bfloat16)
        st["q_norm"], st["k_norm"] = ((1.0 + 0.2 * f(D)).to(torch.bfloat16) for _ in range(2))
        at = torch.tensor(pos, device=DEVICE, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(64, device=DEVICE, dtype=torch.float64) / 64)
        st["cos"], st["sin"] = at.cos().to(torch.bfloat16), at.sin().to(torch.bfloat16)
        for k in range(case["idle"]):                # rows of no stream, among the others
            stream[(k * 4 + 1) % len(stream)] = -1
        st["stream"], st["pos"], st["kv_len"] = i32(stream), i32(pos), i32(past)
        st["by_len"] = case["rows"] == 1
        if case["bits"] == 16:
            st["buf"] = torch.zeros(n, 2 * kv_heads * lmax * D, dtype=torch.bfloat16, device=DEVICE)
        else:
            st["buf"] = torch.zeros(n, kv_heads * lmax * 136, dtype=torch.uint8, device=DEVICE)
    else:
        k = (f(n, kv_heads, lmax, D) * size).to(torch.bfloat16)
        v = f(n, kv_heads, lmax, D).to(torch.bfloat16)
        k[:, :, 0], v[:, :, 0] = k[:, :, 0] * 2, v[:, :, 0] / 8
        st["buf"] = torch.empty(n, kv_heads * lmax * 136, dtype=torch.uint8, device=DEVICE)
        fill(st["buf"], kv_heads, lmax, k, v)
        del k, v
        st["q"] = f(len(stream), heads * D).to(torch.bfloat16)
        st["slots"], st["kv_len"], st["stream"], st["pos"] = i32(list(range(n))), i32(past), i32(stream), i32(pos)
        st["most"], st["most_rows"] = max(r + p for r, p in zip(rows, past)), max(rows)
        st["row"] = i32([r for s in range(n) for r in range(rows[s])])
    if own:
        from livecc_amd import ops
        if case["kind"] == "append" and case["bits"] == 16:
            st["kv"] = ops.KvArena(n, 1, kv_heads, lmax, torch.device(DEVICE))
            st["buf"] = st["kv"].buf
        else:
            st["kv"] = ops.Kv4Arena(n, 1, kv_heads, lmax, torch.device(DEVICE))
            st["kv"].buf.copy_(st["buf"])
            st["buf"] = st["kv"].buf
        if case["kind"] == "decode":
            st["splits"] = ops.kv4_decode_splits([p + 1 for p in past], kv_heads)
        if case["kind"] == "chunk":
            st["plan"] = ops.kv4_prefill_plan([(s, rows[s], past[s]) for s in range(n)], heads, kv_heads, torch.device(DEVICE))
    return st


def run(st):
    if own:
        return run_own(st)
    return append_plain(st) if st["kind"] == "append" else attention_plain(st)


def run_own(st):
    from livecc_amd import ops
    if st["kind"] == "decode":
        return ops.attn_decode4(st["q"], st["kv"], 0, st["slots"], st["kv_len"], st["heads"], st["splits"])
    if st["kind"] == "chunk":
        return ops.attn_prefill4(st["q"], st["kv"], 0, st["plan"], st["heads"])
    q = ops.qk_norm_rope_kv_append(st["qkv"], st["cos"], st["sin"], st["stream"], None if st["by_len"] else st["pos"], st["kv"], 0, st["heads"],
                                   q_norm=st["q_norm"], k_norm=st["k_norm"], eps=1e-6, kv_len=st["kv_len"])
    if st["bits"] == 16:
        return q, st["buf"]
    return (q,) + tuple(ops.kv4_read(st["kv"], 0, st["stream"], st["pos"]))


def normed(x, w):
    """Rows' heads [S, heads, 128] fp32: RMS norm with the model's rounding points.  The statistic is formed in 64 bits and its root rounded once: what
    follows is quantised, and a sum's order must not decide a rounding."""
    r = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt().float()
    return (w.float() * (x * r).to(torch.bfloat16).float()).to(torch.bfloat16).float()


def rotated(x, cos, sin):
    b = lambda t: t.to(torch.bfloat16).float()  # noqa: E731
    c, s = cos.float().unsqueeze(1), sin.float().unsqueeze(1)
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat((b(lo * c) + b(-hi * s), b(hi * c) + b(lo * s)), -1).to(torch.bfloat16)


def append_plain(st):
    heads, kv_heads, lmax, buf = st["heads"], st["kv_heads"], st["lmax"], st["buf"]
    x = st["qkv"].float().unflatten(-1, (heads + 2 * kv_heads, D))
    q = rotated(normed(x[:, :heads], st["q_norm"]), st["cos"], st["sin"])
    k = rotated(normed(x[:, heads:heads + kv_heads], st["k_norm"]), st["cos"], st["sin"])
    v = x[:, heads + kv_heads:].to(torch.bfloat16)
    live = st["stream"] >= 0
    s, p = st["stream"].long()[live], st["pos"].long()[live]
    if st["bits"] == 16:
        half = kv_heads * lmax * D
        buf[:, :half].view(-1, kv_heads, lmax, D)[s, :, p] = k[live]
        buf[:, half:].view(-1, kv_heads, lmax // 32, D, 32)[s, :, p // 32, :, p % 32] = v[live]
        return q.flatten(1), buf
    kc, vc, ks, vs = parts(buf, kv_heads, lmax)
    h, e = encode(k[live])
    kc[s, :, p] = h[..., 0::2] | h[..., 1::2] << 4
    ks[s, :, p] = e
    h, e = encode(v[live])
    h = h.unflatten(-1, (4, 2, 16))
    vc[s, :, p // 32, p % 32 // 8, :, :, p % 8] = (h[..., 0, :] | h[..., 1, :] << 4).transpose(-1, -2)
    vs[s, :, p // 32, p % 32 // 8, :, p % 8] = e
    got_k, got_v = (torch.zeros(st["rows"], kv_heads, D, dtype=torch.bfloat16, device=buf.device) for _ in range(2))
    got_k[live] = decode(codes_k(kc[s, :, p]), ks[s, :, p]).to(torch.bfloat16)
    b = vc[s, :, p // 32, p % 32 // 8, :, :, p % 8]                                     # row, head, i, t
    got_v[live] = decode(torch.stack((b & 15, b >> 4), -1).permute(0, 1, 3, 4, 2).flatten(2), vs[s, :, p // 32, p % 32 // 8, :, p % 8]).to(torch.bfloat16)
    return q.flatten(1), got_k, got_v


def attention_plain(st):
    heads, kv_heads, keys, n, most = st["heads"], st["kv_heads"], st["most"], st["n"], st["most_rows"]
    k, v = unpack(st["buf"], kv_heads, st["lmax"], keys)
    s, r = st["stream"].long(), st["row"].long()
    q = torch.zeros(n, most, kv_heads, heads // kv_heads, D, device=k.device)
    at = torch.full((n, most), -1, device=k.device)
    q[s, r] = st["q"].float().view(-1, kv_heads, heads // kv_heads, D)
    at[s, r] = st["pos"].long()
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)                                          # n, kv_heads, rows * group, 128
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5)
    seen = torch.arange(keys, device=k.device) <= at.repeat_interleave(heads // kv_heads, 1)[:, None, :, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = out.unflatten(2, (most, heads // kv_heads)).permute(0, 2, 1, 3, 4)[s, r]
    return out.reshape(-1, heads * D).to(torch.bfloat16)


def work(case):
    rows, past, _ = sizes(case)
    heads, kv_heads, s = case["heads"], case["kv_heads"], sum(rows)
    if case["kind"] == "append":
        b = s * ((heads + 2 * kv_heads) * 256 + 256 + heads * 256)
        # the 4-bit cache: written, read, and the values of it written
        b += s * kv_heads * 512 if case["bits"] == 16 else s * kv_heads * (2 * 136 + 512)
        return {"bytes": b, "flops": 0}
    pairs = sum(p * r + r * (r + 1) // 2 for r, p in zip(rows, past))
    return {"bytes": sum(r + p for r, p in zip(rows, past)) * kv_heads * 136 + s * heads * 512, "flops": 4 * D * heads * pairs}


# ---- 64 bits
def value64(half, e):
    """Values of halves [...] under exponents of the same shape: sign, two bits of exponent, one of mantissa."""
    m, x = (half & 1).double(), (half >> 1 & 3).int()
    mag = torch.where(x == 0, m / 2, (1 + m / 2) * torch.pow(2.0, (x - 1).double()))
    scale = torch.pow(2.0, e.double() - 127)
    return torch.where(half >= 8, -mag, mag) * torch.where(e == 255, math.nan, scale)


def quantised64(x):
    """What bf16-valued rows [..., 128] stand for once held in 4 bits: the nearest of the fifteen values, under the smallest scale with seven of it no less
    than the group's largest magnitude."""
    g = x.double().unflatten(-1, (4, 32))
    a = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a / 7)).nan_to_num(0.0, 0.0, -125.0)
    e = e + (7 * torch.pow(2.0, e) < a).double()                                        # the logarithm next to a whole number
    e = e - (7 * torch.pow(2.0, e - 1) >= a).double()
    v = g / torch.pow(2.0, e.clamp(-125, 125))
    m = v.abs().unsqueeze(-1)
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    even = torch.arange(8, device=x.device) % 2 * 1e-9                                  # a tie goes to the even code
    near = table[((m - table).abs() + even).argmin(-1)]
    return (torch.copysign(near, v) * torch.pow(2.0, e.clamp(-125, 125))).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    heads, kv_heads, lmax = st["heads"], st["kv_heads"], st["lmax"]
    if case["kind"] == "append":
        x = st["qkv"].double().unflatten(-1, (heads + 2 * kv_heads, D))
        cos, sin = st["cos"].double()[:, None], st["sin"].double()[:, None]

        def turned(x, w, at=lambda t: t):
            y = at(w.double() * at(x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()))
            a, b = y.chunk(2, -1)
            return at(torch.cat((at(a * cos) - at(b * sin), at(b * cos) + at(a * sin)), -1))

        q, k, v = turned(x[:, :heads], st["q_norm"]), x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
        if case["bits"] == 16:
            k = turned(k, st["k_norm"])
            cache_k = torch.zeros(case["streams"], kv_heads, lmax, D, dtype=torch.float64, device=k.device)
            cache_v = cache_k.clone()
            live = (st["stream"] >= 0).nonzero().flatten()
            s, p = st["stream"][live].long(), st["pos"][live].long()
            cache_k[s, :, p], cache_v[s, :, p] = k[live], v[live]
            cache_v = cache_v.view(case["streams"], kv_heads, lmax // 32, 32, D).transpose(-1, -2)
            return q.flatten(1), torch.cat((cache_k.flatten(1), cache_v.flatten(1)), 1)
        # the cache holds what the bf16 keys are rounded to, so those have their rounding points
        k = turned(k, st["k_norm"], lambda t: t.float().to(torch.bfloat16).double())
        live = (st["stream"] >= 0).double()[:, None, None]
        return q.flatten(1), quantised64(k) * live, quantised64(v) * live
    rows, past, _ = sizes(case)
    kc, vc, ks, vs = parts(st["buf"], kv_heads, lmax)
    out, row = [], 0
    for s in range(case["streams"]):
        total, group = rows[s] + past[s], heads // kv_heads
        at = torch.arange(total, device=DEVICE)
        c = torch.arange(D, device=DEVICE)
        k = value64(kc[s][:, :total, c // 2] >> (c % 2 * 4).to(torch.uint8) & 15, ks[s][:, :total, c // 32])
        blk, unit, e = (at // 32)[:, None], (at % 32 // 8)[:, None], (at % 8)[:, None]
        v = value64(vc[s][:, blk, unit, c % 16, c // 32, e] >> (c // 16 % 2 * 4).to(torch.uint8) & 15, vs[s][:, blk, unit, c // 32, e])
        q = st["q"][row:row + rows[s]].double().view(rows[s], kv_heads, group, D)
        for h in range(kv_heads):
            sc = (q[:, h].reshape(-1, D) @ k[h].T / math.sqrt(D)).view(rows[s], group, total)
            sc = sc + torch.where(at[None, None, :] > past[s] + torch.arange(rows[s], device=DEVICE)[:, None, None], -math.inf, 0.0)
            out.append((torch.softmax(sc, -1).view(-1, total) @ v[h]).view(rows[s], group * D))
        out[-kv_heads:] = [torch.cat(out[-kv_heads:], 1)]
        row += rows[s]
    return torch.cat(out)
