"""CPU tier of the 4-bit KV cache: layout and values of the arena, launch plans, refusals of the C entries and of the wrappers (no GPU, nothing is launched)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from livecc_amd import _lib
from tests import kv4_util as U


def put(arena, slot, layer, k, v):
    """keys and values [Hkv, L, 128] into a CPU arena, byte by byte from the layout in include/livecc_amd.h"""
    hkv, lmax, L = arena.n_kv_heads, arena.lmax, k.shape[1]
    buf = arena.buf[slot].numpy()
    at = layer * hkv * lmax * 136
    (ck, ek, _), (cv, ev, _) = U.quantise(k), U.quantise(v)
    for h in range(hkv):
        for p in range(L):
            for b in range(64):
                buf[at + (h * lmax + p) * 64 + b] = int(ck[h, p, 2 * b]) | int(ck[h, p, 2 * b + 1]) << 4
            blk, g, e = p // 32, p % 32 // 8, p % 8
            for t in range(4):
                for i in range(16):
                    buf[at + (hkv + h) * lmax * 64 + blk * 2048 + ((g * 16 + i) * 4 + t) * 8 + e] = int(cv[h, p, 32 * t + i]) | int(cv[h, p, 32 * t + 16 + i]) << 4
                buf[at + hkv * lmax * 128 + (h * lmax + p) * 4 + t] = int(ek[h, p, t])
                buf[at + hkv * lmax * 132 + h * lmax * 4 + blk * 128 + (g * 4 + t) * 8 + e] = int(ev[h, p, t])


def test_views_of_an_arena(built_lib):
    from livecc_amd import ops
    kv = ops.Kv4Arena(2, 2, 2, 64, "cpu")
    assert kv.per_slot == 2 * 2 * 64 * 136 == built_lib.lcc_kv4_slot_bytes(kv.lay) and kv.ptrs.tolist() == [kv.buf[i].data_ptr() for i in range(2)]
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 50, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    k[1, 7, 33] = math.nan
    put(kv, 1, 1, k, v)
    for view, x in ((kv.k_view(1, 1), k), (kv.v_view(1, 1), v)):
        want = U.quantise(x)[2]
        assert view.dtype == torch.bfloat16 and view.shape == (2, 64, 128)
        assert torch.equal(torch.isnan(view[:, :50]), torch.isnan(want)) and torch.equal(view[:, :50].double().nan_to_num(0), want.nan_to_num(0))
        assert not view[:, 50:].any()
    assert not kv.k_view(1, 0).any() and not kv.v_view(0, 1).any()


def test_the_format_is_off_by_at_most_its_scale():
    """half of the step between 4 and 6 under a scale of which seven reach the largest magnitude and three and a half do not"""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(200, 128, generator=g) * torch.exp(3 * torch.randn(200, 1, generator=g))).to(torch.bfloat16).double()
    codes, e, val = U.quantise(x)
    top = x.unflatten(-1, (4, 32)).abs().amax(-1, keepdim=True)
    scale = torch.pow(2.0, e - 127).unsqueeze(-1)
    assert bool((top <= 7 * scale).all()) and bool((top > 3.5 * scale).all())
    err = (val - x).unflatten(-1, (4, 32)).abs()
    assert bool((err <= top / 3.5).all()) and bool((err <= scale).all())
    assert bool((codes >= 0).all()) and bool((codes <= 15).all())


def test_arenas_that_cannot_be(built_lib):
    from livecc_amd import ops
    for args in ((1, 1, 1, 40), (1, 1, 1, 0), (1, 0, 1, 64), (1, 1, 0, 64)):
        with pytest.raises(ValueError):
            ops.Kv4Arena(*args, "cpu")
    assert built_lib.lcc_kv4_slot_bytes(_lib.KvLayout(1, 1, 64, 64)) == 0


def test_slot_bytes_and_offsets_beyond_32_bits(built_lib):
    assert built_lib.lcc_kv4_slot_bytes(_lib.KvLayout(80, 8, 32768, 128)) == 80 * 8 * 32768 * 136


def test_decode_splits(built_lib):
    from livecc_amd import ops
    assert ops.kv4_decode_splits([1], 1) == 1
    for n in (1, 31, 33, 517, 6500, 32768, 1 << 20):
        for streams in (1, 3, 64):
            for heads in (1, 4, 8):
                k = ops.kv4_decode_splits([n] * streams, heads)
                assert 1 <= k <= 64 and k <= max(1, math.ceil(n / 32))
    assert ops.kv4_decode_splits([-3], 4) == 1
    with pytest.raises(_lib.LccError):
        ops.kv4_decode_splits([], 4)
    with pytest.raises(_lib.LccError):
        ops.kv4_decode_splits([5], 0)


@pytest.mark.parametrize("heads,kv_heads", [(28, 4), (64, 8), (7, 1), (3, 3), (32, 2)])
def test_prefill_plans(built_lib, heads, kv_heads):
    from livecc_amd import ops
    seg = [(2, 386, 6120), (0, 0, 5), (1, 1, 0), (4, 37, 12)]
    plan = ops.kv4_prefill_plan(seg, heads, kv_heads, "cpu")
    assert plan.rows == 424 and plan.max_keys == 6506 and 1 <= plan.nsplit <= 64 and 1 <= plan.tile_rows <= 256 // (heads // kv_heads)
    rows = [None] * plan.rows
    for slot, q0, nq, pos0 in plan.tiles.T.tolist():
        assert 1 <= nq <= plan.tile_rows
        for r in range(nq):
            assert rows[q0 + r] is None
            rows[q0 + r] = (slot, pos0 + r)
    assert rows == [(s, p + r) for s, n, p in seg for r in range(n)]
    none = ops.kv4_prefill_plan([], heads, kv_heads, "cpu")
    assert none.rows == 0 and none.tiles.shape == (4, 0) and none.max_keys == 0
    assert ops.kv4_prefill_plan(seg, heads, kv_heads, "cpu", 5).nsplit == 5
    for bad in ([(0, -1, 4)], [(0, 3, -2)]):
        with pytest.raises(_lib.LccError):
            ops.kv4_prefill_plan(bad, heads, kv_heads, "cpu")
    for h, k in ((5, 2), (34, 2), (0, 1), (4, 0)):
        with pytest.raises(_lib.LccError):
            ops.kv4_prefill_plan(seg, h, k, "cpu")


def test_c_entries_refuse_before_any_launch(built_lib):
    lib = built_lib
    mem = np.zeros(4096, dtype=np.uint8)
    p = (mem.ctypes.data + 255) // 256 * 256
    lay, odd = _lib.KvLayout(1, 2, 64, 128), p + 8
    ERR_ARG, ERR_SHAPE, ERR_ALIGN = -1, -2, -3

    def append(fn, **kw):
        a = dict(qkv=p, part=None, nsplit=0, bias=None, qn=p, kn=p, eps=1e-6, cos=p, sin=p, st=p, pos=p, length=None, base=p, slots=1, lay=lay, layer=0, q=p, S=1, H=4)
        a.update(kw)
        return fn(a["qkv"], a["part"], a["nsplit"], a["bias"], a["qn"], a["kn"], a["eps"], a["cos"], a["sin"], a["st"], a["pos"], a["length"], a["base"], a["slots"], a["lay"],
                  a["layer"], a["q"], a["S"], a["H"], None)
    for fn in (lib.lcc_qk_norm_rope_kv_append_bf16, lib.lcc_qk_norm_rope_kv4_append):
        for kw in (dict(qkv=None), dict(part=p), dict(cos=None), dict(sin=None), dict(st=None), dict(pos=None), dict(base=None), dict(q=None), dict(bias=p), dict(eps=0.0),
                   dict(eps=math.nan)):
            assert append(fn, **kw) == ERR_ARG, kw
        for kw in (dict(qkv=odd), dict(qn=odd), dict(kn=odd), dict(cos=odd), dict(sin=odd), dict(q=odd)):
            assert append(fn, **kw) == ERR_ALIGN, kw
        for kw in (dict(lay=_lib.KvLayout(1, 2, 64, 64)), dict(lay=_lib.KvLayout(1, 2, 48, 128)), dict(lay=_lib.KvLayout(1, 0, 64, 128)), dict(layer=1), dict(layer=-1), dict(S=-1),
                   dict(H=-1), dict(H=65536), dict(slots=-1), dict(lay=_lib.KvLayout(1, 2, (1 << 30) + 32, 128)), dict(S=0x7fffffff), dict(qkv=None, part=p, nsplit=0), dict(qkv=None, part=p, nsplit=9)):
            assert append(fn, **kw) == ERR_SHAPE, kw

    def read(**kw):
        a = dict(base=p, slots=1, lay=lay, layer=0, st=p, pos=p, k=p, v=p, S=1)
        a.update(kw)
        return lib.lcc_kv4_read(*a.values(), None)
    assert [read(**{n: None}) for n in ("base", "st", "pos", "k", "v")] == [ERR_ARG] * 5
    assert read(k=odd) == read(v=odd) == ERR_ALIGN and read(S=-1) == read(layer=3) == read(slots=-1) == ERR_SHAPE

    def decode(**kw):
        a = dict(q=p, out=p, slots=p, length=p, base=p, n=1, lay=lay, layer=0, B=1, H=4, nsplit=1, o=None, ml=None)
        a.update(kw)
        return lib.lcc_attn_decode_kv4(*a.values(), None)
    assert [decode(**{n: None}) for n in ("q", "out", "slots", "length", "base")] == [ERR_ARG] * 5
    assert decode(nsplit=2) == decode(nsplit=2, o=p) == ERR_ARG
    for kw in (dict(H=3), dict(H=34), dict(H=0), dict(nsplit=0), dict(nsplit=65, o=p, ml=p), dict(B=-1), dict(B=65536), dict(B=65535, H=65536, lay=_lib.KvLayout(1, 8192, 32, 128)), dict(layer=1), dict(lay=_lib.KvLayout(1, 2, 33, 128))):
        assert decode(**kw) == ERR_SHAPE, kw
    assert decode(q=odd) == decode(out=odd) == decode(o=odd, ml=p, nsplit=2) == ERR_ALIGN

    def chunk(**kw):
        a = dict(q=p, out=p, t0=p, t1=p, t2=p, t3=p, base=p, n=1, lay=lay, layer=0, tiles=1, H=4, rows=8, nsplit=1, S=1, o=None, ml=None)
        a.update(kw)
        return lib.lcc_attn_prefill_kv4(*a.values(), None)
    assert [chunk(**{n: None}) for n in ("q", "out", "t0", "t1", "t2", "t3", "base")] == [ERR_ARG] * 7
    assert chunk(nsplit=2) == ERR_ARG
    for kw in (dict(H=3), dict(H=34), dict(nsplit=0), dict(nsplit=65, o=p, ml=p), dict(tiles=-1), dict(tiles=65536), dict(rows=0), dict(rows=129), dict(S=-1), dict(S=1 << 30), dict(layer=1)):
        assert chunk(**kw) == ERR_SHAPE, kw
    assert chunk(q=odd) == chunk(out=odd) == ERR_ALIGN


def test_cpu_tensors_are_refused(built_lib):
    from livecc_amd import ops
    kv = ops.Kv4Arena(1, 1, 1, 32, "cpu")
    x, i = torch.zeros(1, 3 * 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    cos = torch.zeros(1, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.qk_norm_rope_kv_append(x, cos, cos, i, i, kv, 0, 1), lambda: ops.kv4_read(kv, 0, i, i),
                 lambda: ops.attn_decode4(x[:, :128].contiguous(), kv, 0, i, i, 1, 1), lambda: ops.attn_prefill4(x[:, :128].contiguous(), kv, 0, [(0, 1, 0)], 1)):
        with pytest.raises(_lib.LccError):
            call()
    with pytest.raises(TypeError):
        ops.kv4_read(object(), 0, i, i)


def test_sizes_beyond_a_launch_or_63_bits_are_refused(built_lib):
    """more than 2^32 threads; heads * layers whose offsets would wrap"""
    lib, mem = built_lib, np.zeros(512, dtype=np.uint8)
    p = (mem.ctypes.data + 255) // 256 * 256
    lay = _lib.KvLayout(1, 8, 64, 128)
    for S in (1 << 26, 0x7fffffff):
        assert lib.lcc_kv4_read(p, 1, lay, 0, p, p, p, p, S, None) == -2
        for fn in (lib.lcc_qk_norm_rope_kv_append_bf16, lib.lcc_qk_norm_rope_kv4_append):
            assert fn(p, None, 0, None, None, None, 1e-6, p, p, p, p, None, p, 1, lay, 0, p, S, 64, None) == -2
    for layers, heads in ((65535, 65535), (1 << 24, 2), (0x7fffffff, 1)):
        assert lib.lcc_kv4_slot_bytes(_lib.KvLayout(layers, heads, 64, 128)) == 0
        assert lib.lcc_kv4_read(p, 1, _lib.KvLayout(layers, heads, 64, 128), 0, p, p, p, p, 1, None) == -2
    assert lib.lcc_kv4_slot_bytes(_lib.KvLayout(1 << 14, 1 << 10, 1 << 30, 128)) == 136 << 54
