"""GPU tests of the 4-bit KV cache (livecc_amd/csrc/kv4.hip): norm + rotation + append into both caches, read-back, attention of tokens and of chunks,
each against plain 64-bit forms (tests/kv4_util.py), and a run of them as a decoder layer would use them."""
import math

import pytest
import torch

from tests import kv4_util as U

pytestmark = pytest.mark.gpu


def rand(shape, dev, seed, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16).to(dev)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def tables(pos, dev):
    at = torch.tensor(pos, dtype=torch.float64).clamp(min=0)[:, None] * 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return at.cos().to(torch.bfloat16).to(dev), at.sin().to(torch.bfloat16).to(dev)


def filled(dev, k, v, layers=1, layer=0):
    """a Kv4Arena whose slots hold k, v [n, Hkv, L, 128] (through the append kernel: it has tests of its own), and the values held"""
    from livecc_amd import ops
    n, hkv, L, _ = k.shape
    kv = ops.Kv4Arena(n, layers, hkv, (L + 31) // 32 * 32, dev)
    rows = torch.cat((k.permute(0, 2, 1, 3).reshape(n * L, hkv * 128), v.permute(0, 2, 1, 3).reshape(n * L, hkv * 128)), 1).contiguous()
    one = torch.ones(n * L, 64, dtype=torch.bfloat16, device=dev)
    stream = torch.arange(n, device=dev, dtype=torch.int32).repeat_interleave(L)
    pos = torch.arange(L, device=dev, dtype=torch.int32).repeat(n)
    ops.qk_norm_rope_kv_append(rows, one, torch.zeros_like(one), stream, pos, kv, layer, 0)
    return kv


def values(kv, slot, layer=0):
    return kv.k_view(slot, layer).double().cpu(), kv.v_view(slot, layer).double().cpu()


# ---- append
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (28, 4), (8, 8), (32, 2)])
@pytest.mark.parametrize("rows,past", [(1, 0), (1, 31), (7, 30), (33, 1), (70, 29)])
@pytest.mark.parametrize("norm", ["both", "q", "k", "none"])
@pytest.mark.parametrize("bits", [16, 4])
def test_norm_rope_append(dev, heads, kv_heads, rows, past, norm, bits):
    """Every value and every code equals the definition's: the one step that is not exact, the root of a 64-bit mean rounded once to fp32, differs only where the
    mean's last bits decide (2^-28 of the cases).  Untouched positions and other layers stay as they were."""
    from livecc_amd import ops
    n, lmax, layers, layer = 3, 128, 2, 1
    S = n * rows
    qkv = rand((S, (heads + 2 * kv_heads) * 128), dev, 1, 2.0)
    qkv[0, :128] = 0
    qn, kn = rand((128,), dev, 2) if norm in ("both", "q") else None, rand((128,), dev, 3) if norm in ("both", "k") else None
    pos = [past + s + r for s in range(n) for r in range(rows)]
    stream = [s for s in (2, 0, 1) for _ in range(rows)]
    pos = [min(p, lmax - 1 - (S - i)) if p >= lmax else p for i, p in enumerate(pos)]
    cos, sin = tables(pos, dev)
    kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(n, layers, kv_heads, lmax, dev)
    kv.buf.view(torch.uint8).fill_(0x3B)
    before = kv.buf.clone()
    q = ops.qk_norm_rope_kv_append(qkv, cos, sin, i32(stream, dev), i32(pos, dev), kv, layer, heads, q_norm=qn, k_norm=kn)
    x = qkv.cpu().view(S, heads + 2 * kv_heads, 128)
    c, s = cos.cpu(), sin.cpu()
    want_q = U.norm_rope(x[:, :heads], None if qn is None else qn.cpu(), c, s)
    want_k = U.norm_rope(x[:, heads:heads + kv_heads], None if kn is None else kn.cpu(), c, s)
    want_v = x[:, heads + kv_heads:].double()
    assert torch.equal(q.double().cpu().view_as(want_q), want_q)
    if bits == 4:
        want_k, want_v = U.quantise(want_k)[2], U.quantise(want_v)[2]
    for i, (sl, p) in enumerate(zip(stream, pos)):
        assert torch.equal(kv.k_view(sl, layer)[:, p].double().cpu(), want_k[i]), (sl, p)
        assert torch.equal(kv.v_view(sl, layer)[:, p].double().cpu(), want_v[i]), (sl, p)
    # nothing else changed: put back what was written and compare all bytes
    same = kv.buf.clone()
    per = kv.buf.shape[1] // layers
    assert torch.equal(same[:, :per], before[:, :per])
    changed = (kv.buf != before).sum().item()
    most = S * kv_heads * (136 if bits == 4 else 256)
    assert changed <= most


def test_append_without_norms_equals_the_existing_append(dev):
    from livecc_amd import ops
    heads, kv_heads, rows = 28, 4, 45
    qkv = rand((rows, 36 * 128), dev, 5)
    pos = list(range(9, 9 + rows))
    cos, sin = tables(pos, dev)
    a, b = ops.KvArena(1, 1, kv_heads, 64, dev), ops.KvArena(1, 1, kv_heads, 64, dev)
    st = i32([0] * rows, dev)
    qa = ops.rope_kv_append(qkv, cos, sin, st, i32(pos, dev), a, 0, heads)
    qb = ops.qk_norm_rope_kv_append(qkv, cos, sin, st, i32(pos, dev), b, 0, heads)
    assert torch.equal(qa, qb) and torch.equal(a.buf, b.buf)


@pytest.mark.parametrize("nsplit", [1, 3, 8])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("with_bias", [True, False])
def test_append_from_slabs(dev, nsplit, bits, with_bias):
    """fp32 slabs, summed in order, plus the bias, rounded: as the bf16 rows with that value."""
    from livecc_amd import ops
    heads, kv_heads, S = 7, 1, 5
    g = torch.Generator().manual_seed(nsplit)
    part = torch.randn(nsplit, S, 9 * 128, generator=g).to(dev)
    bias = rand((9 * 128,), dev, 4) if with_bias else None
    acc = torch.zeros_like(part[0])
    for p in part:
        acc = acc + p
    qkv = (acc + bias.float() if with_bias else acc).to(torch.bfloat16)
    cos, sin = tables(range(S), dev)
    kn = rand((128,), dev, 8)
    out = []
    for src in ("rows", "slabs"):
        kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(2, 1, kv_heads, 32, dev)
        q = ops.qk_norm_rope_kv_append(qkv if src == "rows" else None, cos, sin, i32([1, 0, 1, 1, 0], dev), i32([3, 4, 5, 6, 31], dev), kv, 0, heads,
                                       q_norm=kn, k_norm=kn, partial=None if src == "rows" else part, bias=None if src == "rows" else bias)
        out.append((q, kv.buf))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


@pytest.mark.parametrize("bits", [16, 4])
def test_append_at_kv_len_and_rows_of_no_stream(dev, bits):
    """tok_pos None: positions are the slots' lengths.  Rows of stream -1, of a stream that does not exist, and streams whose position is out of range: queries come, the
    cache stays."""
    from livecc_amd import ops
    heads, kv_heads, S, n = 4, 2, 7, 4
    qkv = rand((S, 8 * 128), dev, 6)
    cos, sin = tables([1] * S, dev)
    stream, lens = [2, -1, 0, 9, 1, 3, -5], [31, 64, 17, -1]
    kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(n, 1, kv_heads, 64, dev)
    q = ops.qk_norm_rope_kv_append(qkv, cos, sin, i32(stream, dev), None, kv, 0, heads, kv_len=i32(lens, dev))
    x = qkv.cpu().view(S, 8, 128)
    want = U.norm_rope(x[:, :heads], None, cos.cpu(), sin.cpu())
    assert torch.equal(q.double().cpu().view_as(want), want)
    k = U.norm_rope(x[:, heads:heads + kv_heads], None, cos.cpu(), sin.cpu())
    k = U.quantise(k)[2] if bits == 4 else k
    for slot in range(n):
        held = kv.k_view(slot, 0).double().cpu()
        for row, p in {2: ((0, 17),), 0: ((2, 31),)}.get(slot, ()):
            assert torch.equal(held[:, p], k[row])
            held[:, p] = 0
        assert not held.any() and (slot in (0, 2) or not kv.buf[slot].any())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows", [130, 600])
@pytest.mark.parametrize("how", ["tokens of many streams", "a chunk with gaps", "one chunk", "two chunks", "a chunk that leaves the arena"])
def test_append_of_many_rows(dev, bits, rows, how):
    """V by windows of 32 rows: whole octets of positions where the rows are consecutive, rows one by one where they are not"""
    from livecc_amd import ops
    heads, kv_heads, lmax = 2, 2, 640
    if how == "tokens of many streams":
        n, lmax, lens = rows, 32, [(37 * s) % 32 for s in range(rows)]
        stream = list(reversed(range(rows)))
        pos = [lens[s] for s in stream]
    else:
        n, lens = 2, [0, 0]
        first = {"a chunk with gaps": 21, "a chunk that leaves the arena": lmax - rows + 3}.get(how, 5)
        stream, pos = [1] * rows, [first + r for r in range(rows)]
        if how == "a chunk with gaps":
            stream[40], pos[75], pos[76] = -1, lmax - 1, -2
        if how == "two chunks":
            stream[77:], pos[77:] = [0] * (rows - 77), list(range(rows - 77))
    S = rows
    qkv = rand((S, 6 * 128), dev, 6)
    cos, sin = tables(pos, dev)
    kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(n, 2, kv_heads, lmax, dev)
    by_len = how == "tokens of many streams"
    ops.qk_norm_rope_kv_append(qkv, cos, sin, i32(stream, dev), None if by_len else i32(pos, dev), kv, 1, heads, kv_len=i32(lens, dev) if by_len else None)
    x = qkv.cpu().view(S, 6, 128)
    want = [U.norm_rope(x[:, 2:4], None, cos.cpu(), sin.cpu()), x[:, 4:].double()]
    want = [U.quantise(w)[2] for w in want] if bits == 4 else want
    for view, w in ((kv.k_view, want[0]), (kv.v_view, want[1])):
        held = torch.stack([view(s, 1) for s in range(n)]).double().cpu()
        for i, (s, p) in enumerate(zip(stream, pos)):
            if s >= 0 and 0 <= p < lmax:
                assert torch.equal(held[s, :, p], w[i]), (s, p)
                held[s, :, p] = 0
        assert not held.any()
    assert not kv.buf[:, :kv.buf.shape[1] // 2].any()


def test_codes_of_every_bf16(dev):
    """Groups whose largest magnitude is each of the finite bf16 magnitudes in turn, beside values spread over its binades, zeros, and both signs; infinities and NaN."""
    from livecc_amd import ops
    bits = torch.arange(0, 0x7F80, 61, dtype=torch.int32)
    a = bits.to(torch.int16).view(torch.bfloat16).double()
    rows = len(a)
    g = torch.Generator().manual_seed(0)
    frac = torch.rand(rows, 256, generator=g, dtype=torch.float64) * 2 - 1
    frac[:, ::7] = torch.round(frac[:, ::7] * 16) / 16                       # many ties
    frac[:, 0::32] = 1.0
    frac[:, 5::32] = 0.0
    x = (a[:, None] * frac).to(torch.bfloat16)
    x = torch.where(x.double().abs() > a[:, None], x.sign() * a[:, None].to(torch.bfloat16), x)
    x[3, 40], x[5, 200], x[9, 130] = math.inf, -math.inf, math.nan
    kv = ops.Kv4Arena(1, 1, 1, (rows + 31) // 32 * 32, dev)
    one = torch.ones(rows, 64, dtype=torch.bfloat16, device=dev)
    # keys through the identity rotation x * 1 - y * 0: an infinity beside it would become a NaN there, which the group is in any case
    ops.qk_norm_rope_kv_append(x.to(dev), one, torch.zeros_like(one), torch.zeros(rows, dtype=torch.int32, device=dev), torch.arange(rows, dtype=torch.int32, device=dev), kv, 0, 0)
    rot = x[:, :128].double()
    rot = torch.cat((rot[:, :64] - rot[:, 64:] * 0, rot[:, 64:] + rot[:, :64] * 0), 1)
    want_k, want_v = U.quantise(rot)[2], U.quantise(x[:, 128:])[2]
    for want, got in ((want_k, kv.k_view(0, 0)), (want_v, kv.v_view(0, 0))):
        got = got[0, :rows].double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
        # and the format's own promise: off by at most half of its largest step, that is one scale, of which 3.5 are below the largest magnitude (where no clamp applies)
        src = (rot if want is want_k else x[:, 128:].double()).unflatten(-1, (4, 32))
        err, top = (want.unflatten(-1, (4, 32)) - src).abs(), src.abs().amax(-1, keepdim=True)
        sane = (torch.isfinite(top) & (top > 2.0 ** -120) & (top < 2.0 ** 127)).expand_as(err)
        assert bool((err <= top / 3.5)[sane].all())


@pytest.mark.parametrize("kv_heads,lmax", [(1, 32), (4, 96)])
def test_read_back(dev, kv_heads, lmax):
    from livecc_amd import ops
    k, v = rand((3, kv_heads, lmax, 128), dev, 1), rand((3, kv_heads, lmax, 128), dev, 2)
    v[1, 0, 3, 70] = math.nan
    kv = filled(dev, k, v, layers=2, layer=1)
    stream = [0, 2, 1, -1, 3, 1, 1, 0, 2]
    pos = [0, lmax - 1, 3, 3, 3, -1, lmax, 17, 31]
    gk, gv = ops.kv4_read(kv, 1, i32(stream, dev), i32(pos, dev))
    for i, (s, p) in enumerate(zip(stream, pos)):
        if 0 <= s < 3 and 0 <= p < lmax:
            assert torch.equal(gk[i], kv.k_view(s, 1)[:, p])
            assert torch.equal(gv[i].nan_to_num(9.0), kv.v_view(s, 1)[:, p].nan_to_num(9.0))
        else:
            assert not gk[i].any() and not gv[i].any()


# ---- attention of single tokens
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (7, 1), (28, 4), (3, 3), (32, 2)])
@pytest.mark.parametrize("nsplit", [1, 2, 5])
def test_decode(dev, heads, kv_heads, nsplit):
    from livecc_amd import ops
    L, n = 224, 4
    k, v = rand((n, kv_heads, L, 128), dev, 1), rand((n, kv_heads, L, 128), dev, 2)
    kv = filled(dev, k, v)
    lens = [0, 31, 32, 223]
    slots = [3, 0, 2, 1, 2]
    q = rand((len(slots), heads * 128), dev, 3)
    got = ops.attn_decode4(q, kv, 0, i32(slots, dev), i32(lens, dev), heads, nsplit)
    for i, s in enumerate(slots):
        kk, vv = values(kv, s)
        want, tol = U.attention(q[i:i + 1].cpu().view(1, heads, 128), kk, vv, [lens[s]])
        U.assert_within(got[i], want[0].flatten(), tol[0].flatten(), f"row {i}, length {lens[s]}")


@pytest.mark.parametrize("keys", [1, 2, 33, 129, 517, 1000])
def test_decode_default_splits_and_large_scores(dev, keys):
    """queries and keys of several times the usual size: one key takes most of the weight"""
    from livecc_amd import ops
    heads, kv_heads = 14, 2
    kv = filled(dev, rand((1, kv_heads, keys, 128), dev, 1, 3.0), rand((1, kv_heads, keys, 128), dev, 2))
    q = rand((1, heads * 128), dev, 3, 3.0)
    kk, vv = values(kv, 0)
    want, tol = U.attention(q.cpu().view(1, heads, 128), kk, vv, [keys - 1])
    lens = i32([keys - 1], dev)
    for nsplit in (0, ops.kv4_decode_splits([keys], kv_heads), 64):
        got = ops.attn_decode4(q, kv, 0, i32([0], dev), lens, heads, nsplit)
        U.assert_within(got, want.flatten(1), tol.flatten(1), f"nsplit {nsplit}")


def test_decode_rows_without_keys_and_garbage_behind_the_length(dev):
    """A length of -1 and slots out of range: zeros.  Bytes behind a stream's last key -- any codes, any scales, NaN's and those that overflow -- do not reach its result; a
    length behind the arena counts as the arena's."""
    from livecc_amd import ops
    heads, kv_heads, L = 14, 2, 96
    kv = filled(dev, rand((5, kv_heads, L, 128), dev, 1), rand((5, kv_heads, L, 128), dev, 2))
    lens = [-1, 40, 95, 4000, -7]
    clean = [values(kv, s) for s in range(5)]
    kc, vc, ks, vs = kv._layer(1, 0)
    ks.view(kv_heads, L, 4)[:, 41:] = 255
    kc.view(kv_heads, L, 64)[:, 41:] = 0x77
    scales = vs.view(kv_heads, L // 32, 4, 4, 8)
    scales[:, 2] = 254
    scales[:, 1, 2:] = 255                        # positions 48 ..
    scales[:, 1, 1, :, 1:] = 253                  # positions 41 .. 47
    q = rand((7, heads * 128), dev, 3)
    slots = [0, 1, 2, 3, 4, -1, 5]
    for nsplit in (1, 3):
        got = ops.attn_decode4(q, kv, 0, i32(slots, dev), i32(lens, dev), heads, nsplit)
        for i, s in enumerate(slots):
            if s in (1, 2, 3):
                want, tol = U.attention(q[i:i + 1].cpu().view(1, heads, 128), *clean[s], [min(lens[s], L - 1)])
                U.assert_within(got[i], want[0].flatten(), tol[0].flatten(), f"row {i}")
            else:
                assert not got[i].any(), i


def test_decode_nan_reaches_the_channels_and_heads_that_read_it(dev):
    from livecc_amd import ops
    heads, kv_heads, L = 4, 2, 64
    k, v = rand((1, kv_heads, L, 128), dev, 1), rand((1, kv_heads, L, 128), dev, 2)
    v[0, 1, 5, 40] = math.nan                     # group 1 of KV head 1
    kv = filled(dev, k, v)
    got = ops.attn_decode4(rand((1, heads * 128), dev, 3), kv, 0, i32([0], dev), i32([L - 1], dev), heads, 1).view(heads, 128)
    nan = torch.isnan(got).cpu()
    assert not nan[:2].any() and bool(nan[2:, 32:64].all()) and not nan[2:, :32].any() and not nan[2:, 64:].any()


# ---- attention of chunks
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (7, 1), (28, 4), (3, 3), (32, 2), (64, 8)])
@pytest.mark.parametrize("segments", [[(0, 1, 0)], [(1, 5, 59)], [(0, 37, 0), (1, 3, 61), (2, 0, 5), (0, 2, 37)], [(2, 33, 30), (1, 64, 32)]])
@pytest.mark.parametrize("nsplit", [1, 3])
@pytest.mark.parametrize("columns", [16, 128, 256])
def test_chunk(dev, heads, kv_heads, segments, nsplit, columns):
    """the three kernels: tiles of up to 16, 128 and 256 (row, head) columns"""
    from livecc_amd import ops
    L = 96
    kv = filled(dev, rand((3, kv_heads, L, 128), dev, 1), rand((3, kv_heads, L, 128), dev, 2))
    S = sum(n for _, n, _ in segments)
    q = rand((S, heads * 128), dev, 3)
    plan = ops.kv4_prefill_plan(segments, heads, kv_heads, dev, nsplit, columns * kv_heads // heads)
    got = ops.attn_prefill4(q, kv, 0, plan, heads)
    row = 0
    for slot, n, past in segments:
        if n == 0:
            continue
        kk, vv = values(kv, slot)
        want, tol = U.attention(q[row:row + n].cpu().view(n, heads, 128), kk, vv, [past + r for r in range(n)])
        U.assert_within(got[row:row + n], want.flatten(1), tol.flatten(1), f"{slot} {n} {past}")
        row += n
    if nsplit == 1:                               # the segments themselves are a plan; the default split count
        U.assert_within(ops.attn_prefill4(q, kv, 0, segments, heads)[row - n:row], want.flatten(1), tol.flatten(1))


@pytest.mark.parametrize("rows,past,heads,kv_heads", [(150, 1000, 7, 1), (2, 700, 28, 4), (300, 0, 12, 2), (20, 5000, 28, 4)])
@pytest.mark.parametrize("columns", [0, 16, 128, 256])
def test_chunk_longer(dev, rows, past, heads, kv_heads, columns):
    from livecc_amd import ops
    L = rows + past
    kv = filled(dev, rand((1, kv_heads, L, 128), dev, 1, 2.0), rand((1, kv_heads, L, 128), dev, 2))
    q = rand((rows, heads * 128), dev, 3, 1.5)
    kk, vv = values(kv, 0)
    got = ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(0, rows, past)], heads, kv_heads, dev, 0, columns * kv_heads // heads), heads)
    at = sorted({0, 1, rows // 2, rows - 2, rows - 1} & set(range(rows)))
    want, tol = U.attention(q[at].cpu().view(len(at), heads, 128), kk, vv, [past + r for r in at])
    U.assert_within(got[at], want.flatten(1), tol.flatten(1))
    # every row against another order of the same sums
    one = torch.cat([ops.attn_decode4(q[r:r + 1], kv, 0, i32([0], dev), i32([past + r], dev), heads, 1) for r in range(0, rows, 7)])
    wide = (one.float() - got[::7].float()).abs()
    top = kv.v_view(0, 0).float().abs().max()
    assert bool((wide <= 2.0 ** -7 * top + 2.0 ** -7 * one.float().abs()).all())


@pytest.mark.parametrize("columns", [16, 128, 256])
def test_chunk_rows_do_not_see_later_keys(dev, columns):
    """NaN keys and values of later rows of the same chunk, and garbage behind the stream's last key, reach no earlier row; the rows that see them are NaN where they are."""
    from livecc_amd import ops
    heads, kv_heads, L, past, n = 14, 2, 128, 50, 40
    k, v = rand((1, kv_heads, L, 128), dev, 1), rand((1, kv_heads, L, 128), dev, 2)
    ck, cv = k.clone(), v.clone()
    v[0, 0, 70, 3] = math.nan                     # group 0 of KV head 0, seen from row 20 on
    v[0, 1, 66, 127] = math.inf                   # group 3 of KV head 1, from row 16
    k[0, 1, 80, 9] = math.nan                     # all of KV head 1, from row 30
    clean, kv = filled(dev, ck, cv), filled(dev, k, v)
    kc, vc, ks, vs = kv._layer(0, 0)
    ks.view(kv_heads, L, 4)[:, 90:] = 255
    vs.view(kv_heads, L // 32, 4, 4, 8)[:, 3] = 253
    vs.view(kv_heads, L // 32, 4, 4, 8)[:, 2, 3, :, 2:] = 255     # positions 90 ..
    q = rand((n, heads * 128), dev, 3)
    kk, vv = values(clean, 0)
    want, tol = U.attention(q.cpu().view(n, heads, 128), kk, vv, [past + r for r in range(n)])
    want[20:, :7, :32] = math.nan
    want[16:, 7:, 96:] = math.nan
    want[30:, 7:] = math.nan
    for nsplit in (1, 2):
        got = ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(0, n, past)], heads, kv_heads, dev, nsplit, columns * kv_heads // heads), heads)
        U.assert_within(got, want.flatten(1), tol.flatten(1), f"nsplit {nsplit}")


@pytest.mark.parametrize("columns", [16, 128, 256])
def test_chunk_of_a_slot_that_does_not_exist(dev, columns):
    from livecc_amd import ops
    kv = filled(dev, rand((2, 1, 64, 128), dev, 1), rand((2, 1, 64, 128), dev, 2))
    q = rand((9, 7 * 128), dev, 3)
    for nsplit in (1, 2):
        got = ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(-1, 3, 0), (1, 3, 20), (2, 3, 4)], 7, 1, dev, nsplit, columns // 7), 7)
        assert not got[:3].any() and not got[6:].any() and bool(got[3:6].any())


# ---- the set together
@pytest.mark.parametrize("heads,kv_heads", [(7, 1), (12, 2)])
def test_a_stream_is_prefilled_and_decoded(dev, heads, kv_heads):
    """Two streams: first turn, a second chunk, then single tokens, each appended and attended to as a layer does it; the reference works on the 64-bit definition from
    the projections on."""
    from livecc_amd import ops
    lmax, layers, layer = 160, 2, 1
    kv = ops.Kv4Arena(3, layers, kv_heads, lmax, dev)
    qn, kn = rand((128,), dev, 11), rand((128,), dev, 12)
    slots = (2, 0)
    have = {s: (torch.zeros(kv_heads, lmax, 128, dtype=torch.float64), torch.zeros(kv_heads, lmax, 128, dtype=torch.float64), 0) for s in slots}
    for turn, new in enumerate([(37, 50), (40, 3), (1, 1), (1, 1)]):
        stream = [s for s, n in zip(slots, new) for _ in range(n)]
        pos = [have[s][2] + r for s, n in zip(slots, new) for r in range(n)]
        qkv = rand((len(stream), (heads + 2 * kv_heads) * 128), dev, 20 + turn)
        cos, sin = tables(pos, dev)
        decode = max(new) == 1
        lens = i32([have.get(s, (0, 0, 0))[2] for s in range(3)], dev)
        q = ops.qk_norm_rope_kv_append(qkv, cos, sin, i32(stream, dev), None if decode else i32(pos, dev), kv, layer, heads, q_norm=qn, k_norm=kn, kv_len=lens if decode else None)
        if decode:
            got = ops.attn_decode4(q, kv, layer, i32(stream, dev), lens, heads, 2)
        else:
            got = ops.attn_prefill4(q, kv, layer, [(s, n, have[s][2]) for s, n in zip(slots, new)], heads)
        x = qkv.cpu().view(len(stream), heads + 2 * kv_heads, 128)
        wq = U.norm_rope(x[:, :heads], qn.cpu(), cos.cpu(), sin.cpu())
        wk = U.quantise(U.norm_rope(x[:, heads:heads + kv_heads], kn.cpu(), cos.cpu(), sin.cpu()))[2]
        wv = U.quantise(x[:, heads + kv_heads:])[2]
        row = 0
        for s, n in zip(slots, new):
            k, v, p = have[s]
            k[:, p:p + n], v[:, p:p + n] = wk[row:row + n].transpose(0, 1), wv[row:row + n].transpose(0, 1)
            want, tol = U.attention(wq[row:row + n], k, v, [p + r for r in range(n)])
            U.assert_within(got[row:row + n], want.flatten(1), tol.flatten(1), f"turn {turn} slot {s}")
            have[s] = (k, v, p + n)
            row += n


def test_a_captured_step_is_replayed(dev):
    """append + decode attention + chunk attention in one graph: replays follow what the buffers then hold, with eager work in between"""
    from livecc_amd import ops
    heads, kv_heads, lmax = 12, 2, 640
    kv, kv2 = ops.Kv4Arena(2, 1, kv_heads, lmax, dev), ops.Kv4Arena(2, 1, kv_heads, lmax, dev)
    qn, kn = rand((128,), dev, 11), rand((128,), dev, 12)
    qkv, st, lens = rand((2, 16 * 128), dev, 1), i32([0, 1], dev), i32([500, 77], dev)
    cos, sin = tables([500, 77], dev)
    qc = rand((60, heads * 128), dev, 2)
    plan = ops.kv4_prefill_plan([(0, 40, 440), (1, 20, 50)], heads, kv_heads, dev, 2)

    def step(c):
        q = ops.qk_norm_rope_kv_append(qkv, cos, sin, st, None, c, 0, heads, q_norm=qn, k_norm=kn, kv_len=lens)
        return q, ops.attn_decode4(q, c, 0, st, lens, heads, 3), ops.attn_prefill4(qc, c, 0, plan, heads)
    for c in (kv, kv2):
        hist = rand((2 * lmax, 4 * 128), dev, 3)
        one = torch.ones(2 * lmax, 64, dtype=torch.bfloat16, device=dev)
        ops.qk_norm_rope_kv_append(hist, one, one * 0, torch.arange(2, dtype=torch.int32, device=dev).repeat_interleave(lmax),
                                   torch.arange(lmax, dtype=torch.int32, device=dev).repeat(2), c, 0, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kv2)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(kv)
    for i in range(4):
        qkv.copy_(rand((2, 16 * 128), dev, 30 + i))
        lens.copy_(i32([500 + i, 77 - i], dev))
        g.replay()
        want = step(kv2)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        assert torch.equal(kv.buf, kv2.buf)


def test_on_a_stream_of_its_own_and_two_at_once(dev):
    from livecc_amd import ops
    heads, kv_heads, L = 28, 4, 700
    kv = filled(dev, rand((2, kv_heads, L, 128), dev, 1), rand((2, kv_heads, L, 128), dev, 2))
    q = [rand((2, heads * 128), dev, 3 + i) for i in range(2)]
    slots, lens = i32([0, 1], dev), i32([L - 1, 333], dev)
    want = [ops.attn_decode4(x, kv, 0, slots, lens, heads, 4) for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attn_decode4(q[i], kv, 0, slots, lens, heads, 4))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


def test_offsets_beyond_32_bits(dev):
    """the last layer of a slot of more than 4 GiB"""
    from livecc_amd import ops
    heads, kv_heads, lmax, layers = 16, 8, 32768, 124
    kv = ops.Kv4Arena(1, layers, kv_heads, lmax, dev)
    assert kv.per_slot > 1 << 32
    last, n = layers - 1, 70
    pos = list(range(lmax - n, lmax))
    qkv = rand((n, 32 * 128), dev, 1)
    cos, sin = tables(pos, dev)
    st = i32([0] * n, dev)
    q = ops.qk_norm_rope_kv_append(qkv, cos, sin, st, i32(pos, dev), kv, last, heads)
    k, v = ops.kv4_read(kv, last, st, i32(pos, dev))
    x = qkv.cpu().view(n, 32, 128)
    assert torch.equal(v.double().cpu(), U.quantise(x[:, 24:])[2])
    assert torch.equal(k.double().cpu(), U.quantise(U.norm_rope(x[:, 16:24], None, cos.cpu(), sin.cpu()))[2])
    kk, vv = values(kv, 0, last)
    assert torch.equal(kk[:, -n:].transpose(0, 1), k.double().cpu())
    want, tol = U.attention(q[-1:].cpu().view(1, heads, 128), kk, vv, [lmax - 1])
    U.assert_within(ops.attn_decode4(q[-1:].contiguous(), kv, last, i32([0], dev), i32([lmax - 1], dev), heads), want.flatten(1), tol.flatten(1))
    U.assert_within(ops.attn_prefill4(q[-1:].contiguous(), kv, last, [(0, 1, lmax - 1)], heads), want.flatten(1), tol.flatten(1))


@pytest.mark.parametrize("through", ["torch", "ctypes"])
def test_refusals(dev, through, monkeypatch):
    from livecc_amd import _lib, ops, torch_ops
    if through == "ctypes":
        monkeypatch.setattr(torch_ops, "op", lambda name: None)
    heads, kv_heads, S = 4, 2, 3
    kv, kv16 = ops.Kv4Arena(2, 1, kv_heads, 64, dev), ops.KvArena(2, 1, kv_heads, 64, dev)
    qkv, st, pos = rand((S, 8 * 128), dev, 1), i32([0, 1, 1], dev), i32([0, 0, 1], dev)
    cos, sin = tables([0, 0, 1], dev)
    w = rand((128,), dev, 2)
    err = (_lib.LccError, ValueError, TypeError)
    for bad in (lambda: ops.qk_norm_rope_kv_append(None, cos, sin, st, pos, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv.float(), cos, sin, st, pos, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv[:, :-128].contiguous(), cos, sin, st, pos, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin[:2], st, pos, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st[:2], pos, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, None, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, None, kv, 0, heads, kv_len=st[:1]),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st.long(), pos, kv, 0, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, pos, kv, 1, heads),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, pos, kv, 0, heads, q_norm=w[:64]),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, pos, kv, 0, heads, q_norm=w, eps=0.0),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, pos, kv, 0, heads, q_norm=w, eps=float("nan")),
                lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, st, pos, kv, 0, heads, bias=rand((8 * 128,), dev, 1)),
                lambda: ops.qk_norm_rope_kv_append(None, cos, sin, st, pos, kv, 0, heads, partial=torch.zeros(9, S, 8 * 128, device=dev)),
                lambda: ops.kv4_read(kv, 0, st, pos[:2]), lambda: ops.kv4_read(kv16, 0, st, pos), lambda: ops.kv4_read(kv, -1, st, pos),
                lambda: ops.attn_decode4(qkv[:, :512].contiguous(), kv16, 0, st, pos, heads),
                lambda: ops.attn_decode4(qkv[:, :512], kv, 0, st, pos, heads),
                lambda: ops.attn_decode4(qkv[:, :512].contiguous(), kv, 0, st[:2], pos, heads),
                lambda: ops.attn_decode4(qkv[:, :512].contiguous(), kv, 0, st, pos[:1], heads),
                lambda: ops.attn_decode4(qkv[:, :512].contiguous(), kv, 0, st, pos, heads, 65),
                lambda: ops.attn_decode4(qkv[:, :384].contiguous(), kv, 0, st, pos, 3),
                lambda: ops.attn_decode4(rand((S, 34 * 128), dev, 1), kv, 0, st, pos, 34),
                lambda: ops.attn_prefill4(qkv[:, :512].contiguous(), kv, 0, [(0, 2, 0)], heads),
                lambda: ops.attn_prefill4(qkv[:, :512].contiguous(), kv, 0, [(0, 3, 62)], heads),
                lambda: ops.attn_prefill4(qkv[:, :512].contiguous(), kv, 0, ops.kv4_prefill_plan([(0, 3, 0)], heads, kv_heads, dev, 65), heads),
                lambda: ops.attn_prefill4(qkv[:, :512].contiguous(), kv, 0, ops.kv4_prefill_plan([(0, 3, 0)], 8, kv_heads, dev), heads),
                lambda: ops.attn_prefill4(qkv[:, :512].contiguous(), kv, 0, ops.kv4_prefill_plan([(0, 3, 0)], heads, kv_heads, dev, 0, 129), heads)):
        with pytest.raises(err):
            bad()
    assert not kv.buf.any()
    # and calls of nothing
    z = qkv[:0]
    assert ops.qk_norm_rope_kv_append(z, cos[:0], sin[:0], st[:0], pos[:0], kv, 0, heads).shape == (0, 512)
    assert ops.attn_decode4(z[:, :512].contiguous(), kv, 0, st[:0], pos, heads).shape == (0, 512)
    assert ops.attn_prefill4(z[:, :512].contiguous(), kv, 0, [], heads).shape == (0, 512)
    assert ops.kv4_read(kv, 0, st[:0], pos[:0])[0].shape == (0, kv_heads, 128)


@pytest.mark.parametrize("bits", [16, 4])
def test_through_the_c_abi_as_through_torch(dev, bits, monkeypatch):
    from livecc_amd import ops, torch_ops
    heads, kv_heads, S = 7, 1, 40
    qkv, cs = rand((S, 9 * 128), dev, 1), tables(range(S), dev)
    st, pos, w = i32([0] * S, dev), i32(list(range(S)), dev), rand((128,), dev, 2)

    def go():
        kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(1, 1, kv_heads, 64, dev)
        q = ops.qk_norm_rope_kv_append(qkv, *cs, st, pos, kv, 0, heads, q_norm=w, k_norm=w)
        if bits == 16:
            return q, kv.buf
        return (q, kv.buf, *ops.kv4_read(kv, 0, st, pos), ops.attn_decode4(q[:2].contiguous(), kv, 0, st[:2], i32([S - 1], dev), heads, 2),
                ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(0, S, 0)], heads, kv_heads, dev, 2), heads))
    n = sum(torch_ops.CALLS[k] for k in ("qk_norm_rope_kv_append", "attn_decode4", "attn_prefill4", "kv4_read"))
    a = go()
    assert sum(torch_ops.CALLS[k] for k in ("qk_norm_rope_kv_append", "attn_decode4", "attn_prefill4", "kv4_read")) == n + (4 if bits == 4 else 1)
    monkeypatch.setattr(torch_ops, "op", lambda name: None)
    for x, y in zip(a, go()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("columns", [16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 3, 12])
def test_chunk_rows_of_no_tile_stay_as_they_were(dev, columns, nsplit):
    """Rows between and behind the tiles, whatever the workspace holds for them; a tile that says more rows than q has."""
    import ctypes
    from livecc_amd import _lib, ops
    heads, kv_heads, L = 14, 2, 96
    kv = filled(dev, rand((2, kv_heads, L, 128), dev, 1), rand((2, kv_heads, L, 128), dev, 2))
    S, height = 40, columns * kv_heads // heads
    tiles = [(0, 2, min(2, height), 50), (1, 10, min(9, height), 80), (0, 38, height, 0)]
    q, out = rand((S, heads * 128), dev, 3), rand((S, heads * 128), dev, 4)
    before, t = out.clone(), i32([list(c) for c in zip(*tiles)], dev)
    ws = torch.full((S * heads * nsplit * 130,), math.nan, device=dev)
    at, st = t.data_ptr(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.load().lcc_attn_prefill_kv4(q.data_ptr(), out.data_ptr(), at, at + 12, at + 24, at + 36, kv.ptrs.data_ptr(), 2, kv.lay, 0, 3, heads, height, nsplit, S,
                                                ws.data_ptr(), ws.data_ptr() + S * heads * nsplit * 512, st), "lcc_attn_prefill_kv4")
    left = set(range(S))
    for slot, q0, nq, pos in tiles:
        nq = min(nq, S - q0)
        want, tol = U.attention(q[q0:q0 + nq].cpu().view(nq, heads, 128), *values(kv, slot), [pos + r for r in range(nq)])
        U.assert_within(out[q0:q0 + nq], want.flatten(1), tol.flatten(1), f"rows {q0}..")
        left -= set(range(q0, q0 + nq))
    left = sorted(left)
    assert torch.equal(out[left], before[left])


@pytest.mark.parametrize("columns", [0, 16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 2])
def test_keys_whose_scores_are_minus_infinity(dev, columns, nsplit):
    """The first 64 keys' scores leave the type's range downwards, the others' are zero: the mean of the others' values.  Tolerance: half a step of bf16 for the
    result, none for the probabilities (all one), 2^-16 for the sums.  columns 0: single tokens."""
    from livecc_amd import ops
    heads, kv_heads, L = 14, 2, 320
    k, v = torch.zeros(1, kv_heads, L, 128, dtype=torch.bfloat16, device=dev), rand((1, kv_heads, L, 128), dev, 2)
    k[:, :, :64, 7] = -3e38
    kv = filled(dev, k, v)
    q = torch.zeros(1, heads, 128, dtype=torch.bfloat16, device=dev)
    q[..., 7] = 3e38
    q = q.flatten(1)
    if columns == 0:
        got = ops.attn_decode4(q, kv, 0, i32([0], dev), i32([L - 1], dev), heads, nsplit)
    else:
        got = ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(0, 1, L - 1)], heads, kv_heads, dev, nsplit, columns * kv_heads // heads), heads)
    vv = values(kv, 0)[1][:, 64:].repeat_interleave(heads // kv_heads, 0)
    want, tol = vv.mean(1), 2.0 ** -8 * vv.mean(1).abs() + 2.0 ** -16 * vv.abs().mean(1)
    U.assert_within(got, want.flatten()[None], tol.flatten()[None])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads,kv_heads", [(28, 4), (64, 8), (30, 2), (31, 1), (0, 3), (5, 5)])
@pytest.mark.parametrize("rows,slabs", [(513, 0), (700, 2)])
def test_append_in_one_call_as_in_many(dev, bits, heads, kv_heads, rows, slabs):
    """rows enough for V to go by windows, against the same rows a hundred at a time: the same queries and the same cache, bit for bit"""
    from livecc_amd import ops
    lmax, width = 416, (heads + 2 * kv_heads) * 128
    src = rand((slabs, rows, width), dev, 1).float() if slabs else rand((rows, width), dev, 1, 2.0)
    cos, sin = tables(range(rows), dev)
    qn, kn = rand((128,), dev, 2), rand((128,), dev, 3)
    half = rows // 2 + 9
    st = i32([1] * half + [0] * (rows - half), dev)
    pos = i32([3 + r for r in range(half)] + list(range(rows - half)), dev)
    out = []
    for step in (rows, 100):
        kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(2, 1, kv_heads, lmax, dev)
        q = [ops.qk_norm_rope_kv_append(None if slabs else src[i:i + step], cos[i:i + step], sin[i:i + step], st[i:i + step], pos[i:i + step], kv, 0, heads, q_norm=qn, k_norm=kn,
                                        partial=src[:, i:i + step].contiguous() if slabs else None) for i in range(0, rows, step)]
        out.append((torch.cat(q), kv.buf))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_decode_of_many_rows_of_few_slots(dev):
    """600 rows, most of them of the same slots: each as alone"""
    from livecc_amd import ops
    heads, kv_heads, L = 6, 2, 160
    kv = filled(dev, rand((3, kv_heads, L, 128), dev, 1), rand((3, kv_heads, L, 128), dev, 2))
    slots = i32([(7 * r) % 3 if r % 11 else -1 for r in range(600)], dev)
    lens, q = i32([159, 64, 7], dev), rand((600, heads * 128), dev, 3)
    for nsplit in (1, 2):
        got = ops.attn_decode4(q, kv, 0, slots, lens, heads, nsplit)
        for i in (0, 1, 2, 22, 301, 599):
            assert torch.equal(got[i:i + 1], ops.attn_decode4(q[i:i + 1].contiguous(), kv, 0, slots[i:i + 1].contiguous(), lens, heads, nsplit)), i


def test_inputs_that_would_record_a_gradient_are_refused(dev):
    from livecc_amd import ops
    heads, kv_heads = 4, 2
    kv = ops.Kv4Arena(1, 1, kv_heads, 64, dev)
    qkv, at = rand((1, 8 * 128), dev, 1).requires_grad_(), i32([0], dev)
    cos, sin = tables([0], dev)
    q = rand((1, heads * 128), dev, 2).requires_grad_()
    for call in (lambda: ops.qk_norm_rope_kv_append(qkv, cos, sin, at, at, kv, 0, heads), lambda: ops.attn_decode4(q, kv, 0, at, at, heads),
                 lambda: ops.attn_prefill4(q, kv, 0, [(0, 1, 0)], heads)):
        with pytest.raises(RuntimeError):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("seed", range(6))
def test_append_of_runs_of_all_lengths(dev, bits, seed):
    """Runs of 1 to 40 consecutive positions of shuffled slots, rows of no stream between them: octets begin, end and break anywhere in a window and across two.  In one call as
    in calls of few rows."""
    import random
    from livecc_amd import ops
    heads, kv_heads, n, lmax = 3, 1, 5, 224
    rng = random.Random(seed)
    runs, left = [], []
    for slot in range(n):
        p = rng.choice((0, 1, 7, 8))
        while p < lmax:
            k = min(rng.choice((1, 2, 7, 8, 9, 16, 23, 40)), lmax - p)
            runs.append([(slot, p + r) for r in range(k)])
            p += k + rng.choice((0, 0, 1, 8))
    rng.shuffle(runs)
    for run in runs:
        left += run + [(-1, 3)] * rng.choice((0, 0, 0, 1, 5))
    if seed == 0:
        left = [x for slot in range(n) for x in sorted(y for y in left if y[0] == slot)]      # whole streams, one behind the other
    if seed == 1:
        left = left[::-1]                                                                     # positions fall
    rows = len(left)
    assert rows > 300
    qkv, (cos, sin) = rand((rows, 5 * 128), dev, seed), tables(range(rows), dev)
    st, pos = i32([s for s, _ in left], dev), i32([p for _, p in left], dev)
    out = []
    for step in (rows, 37):
        kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(n, 1, kv_heads, lmax, dev)
        for i in range(0, rows, step):
            ops.qk_norm_rope_kv_append(qkv[i:i + step], cos[i:i + step], sin[i:i + step], st[i:i + step], pos[i:i + step], kv, 0, heads)
        out.append(kv.buf)
    assert torch.equal(*out)


def by_tiles(through, q, kv, tiles, heads, height, nsplit):
    """Attention of chunks by tiles (slot, first row, rows, first position) below the Python wrapper, which refuses positions behind the arena."""
    import ctypes
    from livecc_amd import _lib, torch_ops
    S, t = q.shape[0], i32([list(c) for c in zip(*tiles)], q.device)
    if through == "torch":
        return torch_ops.load().attn_prefill4(q, kv.ptrs, kv.buf, kv.n_layers, kv.n_kv_heads, kv.lmax, 0, t, heads, height, nsplit)
    out, ws = torch.empty_like(q), torch.empty(S * heads * nsplit * 130, device=q.device)
    at, n, st = t.data_ptr(), 4 * len(tiles), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.load().lcc_attn_prefill_kv4(q.data_ptr(), out.data_ptr(), at, at + n, at + 2 * n, at + 3 * n, kv.ptrs.data_ptr(), kv.buf.shape[0], kv.lay, 0, len(tiles), heads,
                                                height, nsplit, S, ws.data_ptr(), ws.data_ptr() + S * heads * nsplit * 512, st), "lcc_attn_prefill_kv4")
    return out


@pytest.mark.parametrize("through", ["torch", "ctypes"])
@pytest.mark.parametrize("columns", [16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 2])
@pytest.mark.parametrize("lmax", [32, 96, 128, 160])
def test_chunk_rows_behind_the_arena_see_all_of_it(dev, through, columns, nsplit, lmax):
    """A row at a position of lmax or more sees keys 0 .. lmax - 1, whatever the tile's height, and whether the arena ends inside a stage of 64 keys or with one."""
    heads, kv_heads, height = 14, 2, columns * 2 // 14
    kv = filled(dev, rand((2, kv_heads, lmax, 128), dev, 1), rand((2, kv_heads, lmax, 128), dev, 2))
    runs = [(0, 10, lmax - 6), (1, 3, lmax), (1, 2, lmax + 31), (0, 2, 2 ** 31 - 2)]
    tiles, at, S = [], [], sum(n for _, n, _ in runs)
    for slot, n, pos in runs:
        tiles += [(slot, len(at) + o, min(height, n - o), pos + o) for o in range(0, n, height)]
        at += [(slot, pos + r) for r in range(n)]
    q = rand((S, heads * 128), dev, 3)
    got = by_tiles(through, q, kv, tiles, heads, height, nsplit)
    for i, (slot, p) in enumerate(at):
        want, tol = U.attention(q[i:i + 1].cpu().view(1, heads, 128), *values(kv, slot), [min(p, lmax - 1)])
        U.assert_within(got[i], want[0].flatten(), tol[0].flatten(), f"row {i}, position {p} of {lmax}")


def attend(q, kv, heads, nsplit, columns):
    """one row at the arena's last position: a decode step (columns 0), or a chunk by tiles of so many columns"""
    from livecc_amd import ops
    if columns == 0:
        return ops.attn_decode4(q, kv, 0, i32([0], q.device), i32([kv.lmax - 1], q.device), heads, nsplit)
    return ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(0, 1, kv.lmax - 1)], heads, kv.n_kv_heads, q.device, nsplit, columns * kv.n_kv_heads // heads), heads)


@pytest.mark.parametrize("columns", [0, 16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 2])
@pytest.mark.parametrize("size", [120, -120])
def test_large_and_small_values_under_a_rising_maximum(dev, columns, nsplit, size):
    """Values of 6 * 2^size and keys whose weight is 2^6.1 times that of the keys of the blocks before: every weighted mean is the value itself.  A weight above one would take the large values'
    products out of fp32's range, weights of 2^-14 take the small ones' below its normal range.  Tolerance: half a step of bf16 for the probabilities, as many for the result, 2^-16 for the
    sums (a product of 2^-131 is held to 2^-149)."""
    heads, kv_heads, L = 14, 2, 320
    k, v = torch.zeros(1, kv_heads, L, 128, dtype=torch.bfloat16, device=dev), torch.full((1, kv_heads, L, 128), 6 * 2.0 ** size, dtype=torch.bfloat16, device=dev)
    v[..., 1::2] *= -1
    k[:, :, (130, 258, 290), 7] = 48.0
    kv = filled(dev, k, v)
    q = torch.zeros(1, heads, 128, dtype=torch.bfloat16, device=dev)
    q[..., 7] = 1.0
    want = v[0, :, 0].double().cpu().repeat_interleave(heads // kv_heads, 0).flatten()[None] * 2.0 ** -size
    got = attend(q.flatten(1), kv, heads, nsplit, columns).double() * 2.0 ** -size
    U.assert_within(got, want, want.abs() * (2.0 ** -7 + 2.0 ** -16))


@pytest.mark.parametrize("columns", [0, 16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 2, 5])
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_scores_of_any_size(dev, columns, nsplit, order):
    """Scores of 2^30 to 2^113, of more bits than fp32 holds once they are scaled, whose neighbours lie so far apart that the keys of the highest share all of the weight: their mean.
    Tolerance: half a step of bf16 for the result, none for the weights (all one), 2^-16 for the sums."""
    heads, kv_heads, L = 14, 2, 320
    k, v = torch.zeros(1, kv_heads, L, 128, dtype=torch.bfloat16, device=dev), rand((1, kv_heads, L, 128), dev, 2)
    steps = torch.tensor([1.0, 1.5, 2.0, 3.0, 4.0], device=dev).repeat_interleave(64)
    k[..., 7] = steps if order == "rising" else steps.flip(0)
    k[..., 45, 7] = 4.0
    kv = filled(dev, k, v)
    size = [30, 31, 32, 33, 34, 35, 36, 37, 38, 40, 47, 60, 77, 110]
    for sign in (1, -1):
        top = (k[0, 0, :, 7] == (4.0 if sign > 0 else 1.0)).cpu()
        vv = values(kv, 0)[1][:, top].repeat_interleave(heads // kv_heads, 0)
        want, tol = vv.mean(1), 2.0 ** -8 * vv.mean(1).abs() + 2.0 ** -16 * vv.abs().mean(1)
        q = torch.zeros(1, heads, 128, dtype=torch.bfloat16, device=dev)
        q[0, :, 7] = sign * torch.pow(2.0, torch.tensor(size, device=dev)) * (1 + (2 * torch.arange(heads, device=dev) * 9 % 64 + 1) / 128)
        U.assert_within(attend(q.flatten(1), kv, heads, nsplit, columns), want.flatten()[None], tol.flatten()[None], f"sign {sign}")


@pytest.mark.parametrize("columns", [0, 16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_heads_of_very_different_scores(dev, columns, nsplit):
    """queries of 1 to 4,096 times the usual size in one call: scores of a few units beside ones of several thousand, in the same wave"""
    heads, kv_heads, L = 14, 2, 288
    kv = filled(dev, rand((1, kv_heads, L, 128), dev, 1), rand((1, kv_heads, L, 128), dev, 2))
    size = torch.pow(2.0, (torch.arange(heads) * 5 % 13).double())
    q = (rand((1, heads, 128), "cpu", 3) * size[None, :, None].to(torch.bfloat16)).to(dev)
    want, tol = U.attention(q.cpu(), *values(kv, 0), [L - 1])
    U.assert_within(attend(q.flatten(1), kv, heads, nsplit, columns), want.flatten(1), tol.flatten(1))


@pytest.mark.parametrize("through", ["torch", "ctypes"])
def test_no_route_loses_a_gradient(dev, through, monkeypatch):
    """Whichever input would record a gradient is refused, through the registered ops and through the C-ABI binding; under no_grad all of them may be parameters."""
    from livecc_amd import ops, torch_ops
    if through == "ctypes":
        monkeypatch.setattr(torch_ops, "op", lambda name: None)
    heads, kv_heads, at = 4, 2, i32([0], dev)
    kv = ops.Kv4Arena(1, 1, kv_heads, 64, dev)
    cos, sin = tables([0], dev)
    rows = dict(qkv=rand((1, 8 * 128), dev, 1), q_norm=rand((128,), dev, 2), k_norm=rand((128,), dev, 3), cos=cos, sin=sin)
    slabs = dict(qkv=None, partial=rand((2, 1, 8 * 128), dev, 4).float(), bias=rand((8 * 128,), dev, 5), cos=cos, sin=sin)

    def append(qkv, cos, sin, **kw):
        return ops.qk_norm_rope_kv_append(qkv, cos, sin, at, at, kv, 0, heads, **kw)
    calls = [(append, a, name) for a in (rows, slabs) for name, t in a.items() if t is not None]
    calls += [(lambda q: ops.attn_decode4(q, kv, 0, at, at, heads), dict(q=rand((1, heads * 128), dev, 6)), "q"),
              (lambda q: ops.attn_prefill4(q, kv, 0, [(0, 1, 0)], heads), dict(q=rand((1, heads * 128), dev, 6)), "q")]
    for call, args, name in calls:
        args = dict(args, **{name: args[name].clone().requires_grad_()})
        before = kv.buf.clone()
        with pytest.raises(RuntimeError, match="no_grad"):
            call(**args)
        assert torch.equal(kv.buf, before), name
        with torch.no_grad():
            assert not call(**args).requires_grad


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("kv_heads", [1, 4])
@pytest.mark.parametrize("rows", [1, 9, 61, 150, 333])
def test_append_writes_its_own_bytes_and_no_others(dev, bits, kv_heads, rows):
    """Every byte of every slot and layer against the layout: the bytes of the (slot, head, position) written, put back, leave the whole cache as it was; and each of them was written (two
    fills).  Rows alone, and rows enough for V to go by windows; runs that begin and end within octets, rows of no stream and of positions outside between them."""
    from livecc_amd import ops
    n, lmax, layers, layer, heads = 4, 192, 3, 1, 3
    at, S = [], rows
    for i in range(rows):                                        # slots 2 and 0, slot 1 stays; 13 .. upwards and 190 .. downwards
        at.append((2, 13 + i // 2) if i % 2 == 0 and rows < 100 else (0, 190 - i) if rows < 100 else (2, 5 + i) if i < 180 else (0, i - 177))
        if i % 23 == 11:
            at[-1] = ((-1, 3), (2, lmax), (n, 7), (0, -1))[i // 23 % 4]
    stream, pos = (i32([a[z] for a in at], dev) for z in range(2))
    live = [(s, p) for s, p in at if 0 <= s < n and 0 <= p < lmax]
    assert len(set(live)) == len(live)
    s, p = (torch.tensor([a[z] for a in live]) for z in range(2))
    h = torch.arange(kv_heads)[None, :, None]
    if bits == 16:                                               # [layer][K [head][position][128] | V [head][position / 32][128][position % 32]], bf16
        c, kv_layer = torch.arange(128), 2 * kv_heads * lmax * 128
        k = (h * lmax + p[:, None, None]) * 128 + c
        v = ((kv_heads + h) * lmax + p[:, None, None] // 32 * 32) * 128 + c * 32 + p[:, None, None] % 32
        own = [(layer * kv_layer + torch.cat((k, v), -1))[..., None] * 2 + torch.arange(2)]
    else:                                                        # [layer][K codes | V codes | K scales | V scales], bytes
        q, g, e = p[:, None, None], p[:, None, None] % 32 // 8, p[:, None, None] % 8
        it, t, base = torch.arange(64), torch.arange(4), layer * kv_heads * lmax * 136
        own = [base + (h * lmax + q) * 64 + it, base + (kv_heads + h) * lmax * 64 + q // 32 * 2048 + g * 512 + it * 8 + e,
               base + kv_heads * lmax * 128 + (h * lmax + q) * 4 + t, base + kv_heads * lmax * 132 + h * lmax * 4 + q // 32 * 128 + g * 32 + t * 8 + e]
    own = torch.cat([x.reshape(len(live), -1) for x in own], 1)
    assert own.shape[1] == kv_heads * (512 if bits == 16 else 136)
    qkv, (cos, sin) = rand((S, (heads + 2 * kv_heads) * 128), dev, rows), tables([a[1] for a in at], dev)
    w, written = rand((128,), dev, 2), []
    for fill in (0x3B, 0xC4):
        kv = (ops.Kv4Arena if bits == 4 else ops.KvArena)(n, layers, kv_heads, lmax, dev)
        kv.buf.view(torch.uint8).fill_(fill)
        ops.qk_norm_rope_kv_append(qkv, cos, sin, stream, pos, kv, layer, heads, q_norm=w, k_norm=w)
        held = kv.buf.view(torch.uint8).cpu()
        assert held.shape[1] > int(own.max())
        written.append(held[s[:, None], own].clone())
        held[s[:, None], own] = fill
        assert bool((held == fill).all()), f"{int((held != fill).sum())} bytes of others"
    assert torch.equal(*written)


@pytest.mark.parametrize("through", ["torch", "ctypes"])
@pytest.mark.parametrize("columns", [16, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 2])
def test_chunk_rows_below_position_zero_see_nothing(dev, through, columns, nsplit):
    """A tile that begins below zero: its rows there are zeros, whatever the first keys hold (NaN among them), the others see keys 0 .. p."""
    heads, kv_heads, lmax, height = 14, 2, 96, columns * 2 // 14
    k, v = rand((2, kv_heads, lmax, 128), dev, 1), rand((2, kv_heads, lmax, 128), dev, 2)
    k[1, :, 0, 5] = v[1, :, 0, :] = math.nan
    kv = filled(dev, k, v)
    runs = [(0, 12, -5), (1, 12, -5), (0, 3, -3), (1, 2, -2 ** 31), (0, 2, -1)]
    tiles, at = [], []
    for slot, n, pos in runs:
        tiles += [(slot, len(at) + o, min(height, n - o), pos + o) for o in range(0, n, height)]
        at += [(slot, pos + r) for r in range(n)]
    q = rand((len(at), heads * 128), dev, 3)
    got = by_tiles(through, q, kv, tiles, heads, height, nsplit)
    for i, (slot, p) in enumerate(at):
        if p < 0:
            assert not got[i].any(), (i, p)
        elif slot == 1:
            assert bool(torch.isnan(got[i]).all()), (i, p)
        else:
            want, tol = U.attention(q[i:i + 1].cpu().view(1, heads, 128), *values(kv, slot), [p])
            U.assert_within(got[i], want[0].flatten(), tol[0].flatten(), f"row {i}, position {p}")


@pytest.mark.parametrize("nsplit", [1, 2])
def test_as_many_rows_and_tiles_as_a_launch_takes(dev, nsplit):
    """65,535 rows of a decode step and 65,535 tiles of a chunk, each as alone; one more is refused"""
    from livecc_amd import ops
    heads, kv_heads, L, most = 2, 1, 64, 65535
    kv = filled(dev, rand((3, kv_heads, L, 128), dev, 1), rand((3, kv_heads, L, 128), dev, 2))
    q = rand((most + 1, heads * 128), dev, 3)
    slots, lens = torch.arange(most + 1, dtype=torch.int32, device=dev) % 4 - 1, i32([63, 40, 0], dev)
    got = ops.attn_decode4(q[:most], kv, 0, slots[:most], lens, heads, nsplit)
    for i in (0, 1, 2, 3, 32768, 65533, 65534):
        assert torch.equal(got[i:i + 1], ops.attn_decode4(q[i:i + 1], kv, 0, slots[i:i + 1], lens, heads, nsplit)), i
    assert not got[slots[:most] < 0].any()
    plan = ops.kv4_prefill_plan([(r % 3, 1, r % 61) for r in range(most)], heads, kv_heads, dev, nsplit, 4)
    got = ops.attn_prefill4(q[:most], kv, 0, plan, heads)
    for i in (0, 1, 60, 32768, 65534):
        one = ops.kv4_prefill_plan([(i % 3, 1, i % 61)], heads, kv_heads, dev, nsplit, 4)
        assert torch.equal(got[i:i + 1], ops.attn_prefill4(q[i:i + 1], kv, 0, one, heads)), i
    with pytest.raises(RuntimeError):
        ops.attn_decode4(q, kv, 0, slots, lens, heads, nsplit)
    with pytest.raises(RuntimeError):
        ops.attn_prefill4(q, kv, 0, ops.kv4_prefill_plan([(0, 1, 0)] * (most + 1), heads, kv_heads, dev, nsplit, 4), heads)
