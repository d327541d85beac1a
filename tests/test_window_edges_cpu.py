"""What the window attention, rotary and cache entry points refuse or decide on the host beyond the shapes: operands that share memory, bounds past 32
bits, grids past the hardware's, plans, launch forms.  No GPU: every refused call ends before a launch."""
import ctypes as C

import pytest
import torch

from star_amd import _lib as L
from star_amd import ops

A = 1 << 20          # operands A apart, none of them longer


def _refused(rc, *words):
    said = L.lib().star_last_error().decode()
    assert rc != 0 and all(w in said for w in words), (rc, said)


def _attn(**kw):
    a = dict(qkv=A, out=2 * A, lse=3 * A, dout=4 * A, dqkv=5 * A, ws=6 * A, ld=8 * 64, R=40, NB=2, L=20, H=4, KV=2, hd=64, left=5, right=0, sinks=1,
             scale=0.125, dt=L.BF16)
    a.update(kw)
    return L.StarAttnWindow(**a)


# rows of qkv: 40 of 1024 bytes; of out and dout: 40 of 512; lse: 4 x 40 floats
@pytest.mark.parametrize("change,words", [
    (dict(out=A), "out overlaps qkv"), (dict(out=A + 1024 * 40 - 16), "out overlaps qkv"), (dict(out=A - 512 * 40 + 16), "out overlaps qkv"),
    (dict(out=A, ld=2048), "out overlaps qkv"), (dict(out=A + 1024, ld=2048), "out overlaps qkv"), (dict(lse=A + 1024), "lse overlaps"),
    (dict(lse=2 * A + 512 * 40 - 4), "lse overlaps")])
def test_window_forward_refuses_shared_memory(change, words):
    _refused(L.lib().star_attn_window_fwd(C.byref(_attn(**change)), None), "star_attn_window_fwd", words)


@pytest.mark.parametrize("change,words", [
    (dict(dqkv=A), "dqkv overlaps"), (dict(dqkv=A + 1024 * 40 - 16), "dqkv overlaps"), (dict(dqkv=A - 1024 * 40 + 16), "dqkv overlaps"),
    (dict(dqkv=2 * A), "dqkv overlaps"), (dict(dqkv=4 * A + 512 * 39), "dqkv overlaps"), (dict(dqkv=3 * A + 4 * 40 * 4 - 16), "dqkv overlaps"),
    (dict(ws=A), "ws overlaps"), (dict(ws=2 * A), "ws overlaps"), (dict(ws=3 * A), "ws overlaps"), (dict(ws=4 * A), "ws overlaps"), (dict(ws=5 * A), "ws overlaps")])
def test_window_backward_refuses_shared_memory(change, words):
    _refused(L.lib().star_attn_window_bwd(C.byref(_attn(**change)), None), "star_attn_window_bwd", words)


# rows of qkv: 2 of 1024 bytes; cache: 2 x 2 x 2 x 64 rows of 128 bytes
@pytest.mark.parametrize("change,words", [
    (dict(out=A), "out overlaps qkv"), (dict(out=A + 512), "out overlaps qkv"), (dict(NB=1, out=A + 16), "out overlaps qkv"), (dict(cache=A + 2032), "cache overlaps"),
    (dict(out=2 * A + 64), "cache overlaps"), (dict(NB=1, cap=1 << 16, left=1 << 15, cache=1 << 34, ws=A), "ws overlaps"),
    (dict(NB=1, cap=1 << 16, left=1 << 15, cache=1 << 34, ws=4 * A), "ws overlaps"), (dict(NB=1, cap=1 << 16, left=1 << 15, cache=1 << 34, ws=1 << 34), "ws overlaps")])
def test_step_refuses_shared_memory(change, words):
    a = dict(qkv=A, cache=2 * A, lengths=3 * A, out=4 * A, ws=5 * A, ld=8 * 64, NB=2, H=4, KV=2, hd=64, cap=64, left=31, sinks=4, scale=0.125, dt=L.BF16)
    a.update(change)
    _refused(L.lib().star_attn_window_step(C.byref(L.StarAttnStep(**a)), None), "star_attn_window_step", words)


@pytest.mark.parametrize("cache", [A, A + 40 * 1024 - 16, A - 2 * 2 * 2 * 64 * 64 * 2 + 16])
def test_append_refuses_shared_memory(cache):
    _refused(L.lib().star_kv_append(A, 8 * 64, None, cache, 8 * A, 40, 2, 20, 4, 2, 64, 64, 4, L.BF16, None), "star_kv_append", "cache overlaps")


# ---- bounds past 32 bits: ctypes alone would keep their low half ----------------------------------------------------------------
@pytest.mark.parametrize("over", [(1 << 31), (1 << 32), (1 << 32) + 5, (1 << 63) + 1])
def test_bounds_past_32_bits_stay_bounds(over):
    x = torch.zeros(20, 8 * 16)
    g = ops._window(x, 1, 20, 4, 16, 2, over, over, over, None, None)
    assert (g.left, g.right, g.sinks, g.L, g.NB) == (2147483647, 2147483647, 2147483647, 20, 1)
    g = ops._window(x, 1, 20, 4, 16, 2, -over, -over, -over, None, None)
    assert (g.left, g.right, g.sinks) == (-1, -1, -1)
    g = ops._window(x, 1, over, 4, 16, 2, None, 0, 0, torch.zeros(2, dtype=torch.int64), None)
    assert (g.L, g.left) == (2147483647, 2147483647)
    assert list(ops._ints(5, over, 0, -over)) == [5, 2147483647, 0, -1] and list(ops._ints(0, 7, 2147483647)) == [0, 7, 2147483647]


def test_a_plan_is_the_callers_own():
    first = ops.rope_plan((8, 8), base=500.0)
    kept = list(first.rev)
    first.rev[3] = 0.25
    first.axis[3] = 7
    again = ops.rope_plan((8, 8), base=500.0)
    assert list(again.rev) == kept and again.axis[3] == 0
    held, axes = ops._rope_ref((8, 8), 500.0, False, False)          # what the single-token step hands over
    assert list(held.contents.rev) == kept and axes == 2
    assert list(ops._rope_plan((8, 8), 500.0, False, False).rev) == kept


def test_the_stride_of_a_single_row_does_not_matter():
    for ld in (65, 1 << 20):
        wide = torch.zeros(2, ld)
        assert ops._rows2d(wide[:1, :64], (1, 64), "x") == 64 and ops._rows2d(wide[:, :64], (2, 64), "x") == ld


# ---- launch forms ---------------------------------------------------------------------------------------------------------------
def _far_floats(rows, nb, l, h, kv, hd, left, sinks, dt=L.BF16):
    """what the far queries of the sinks take of the backward pass' workspace, behind the row dots; 0: they are left to the sinks' own blocks"""
    return L.lib().star_attn_window_bwd_ws(rows, nb, l, h, kv, hd, left, sinks, dt) - (h * rows + 63) // 64 * 64


def test_far_queries_of_many_sinks():
    """one sink more or less does not decide it: few blocks with a long sweep among many with short ones are shared out whatever their sinks' number"""
    for hd, dt in ((64, L.BF16), (128, L.BF16), (16, L.BF16), (128, L.F32)):
        for sinks in (1, 256, 257, 512, 2000):
            lists, per = (sinks + 31) // 32, 2 * 32 * max(32, hd)
            assert _far_floats(8192, 1, 8192, 4, 1, hd, 512, sinks, dt) in [lists * parts * per for parts in range(2, 17)], sinks
        assert _far_floats(8192, 1, 8192, 4, 1, hd, 512, 3000, dt) == 0                  # over a third of the keys
        assert _far_floats(16 * 8192, 16, 8192, 16, 16, hd, 512, 600, dt) == 0           # 4864 blocks of sinks
        assert _far_floats(8192, 1, 8192, 4, 1, hd, 8191, 300, dt) == 0                  # no query beyond the window


# ---- grids: the hardware counts a launch's threads in 32 bits -------------------------------------------------------------------
def test_grids_past_the_hardwares_are_refused():
    far = [(i + 1) << 44 for i in range(6)]
    for nb, l, offsets in ((1 << 20, 1, None), (1 << 14, 128 * 64, None), (1 << 20, 100, 1 << 20)):          # 2^24 blocks of 256 threads
        a = _attn(qkv=far[0], out=far[1], lse=far[2], dout=far[3], dqkv=far[4], ws=far[5], ld=48 * 16, NB=nb, L=l, R=nb * l, H=16, KV=16, hd=16, offsets=offsets)
        for name in ("star_attn_window_fwd", "star_attn_window_bwd"):
            _refused(getattr(L.lib(), name)(C.byref(a), None), name, "grid")
    a = L.StarAttnStep(qkv=far[0], cache=far[1], lengths=far[2], out=far[3], ws=far[4], ld=48, NB=1 << 22, H=1, KV=1, hd=16, cap=64, left=31, sinks=4, scale=0.25, dt=L.F32)
    _refused(L.lib().star_attn_window_step(C.byref(a), None), "star_attn_window_step", "grid")
