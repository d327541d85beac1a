"""Refusals of the window attention, rotary and cache entry points (no GPU: every bad call ends before a launch), the rotation plans, and
the ctypes structs against the header."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from star_amd import _lib as L
from star_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _refused(rc, *words):
    said = L.lib().star_last_error().decode()
    assert rc != 0 and all(w in said for w in words), (rc, said)


def _attn(**kw):
    a = dict(qkv=1 << 20, out=1 << 20, lse=1 << 20, dout=1 << 20, dqkv=1 << 20, ws=1 << 20, ld=8 * 64, R=40, NB=2, L=20, H=4, KV=2, hd=64,
             left=5, right=0, sinks=1, scale=0.125, dt=L.BF16)
    a.update(kw)
    return L.StarAttnWindow(**a)


@pytest.mark.parametrize("change,words", [
    (dict(qkv=None), "null"), (dict(out=None), "null"), (dict(dt=2), "dtype"), (dict(hd=48), "head dim"), (dict(hd=256), "head dim"),
    (dict(H=3), "bad shape"), (dict(KV=0), "bad shape"), (dict(NB=0), "bad shape"), (dict(L=0), "bad shape"), (dict(NB=-2), "bad shape"),
    (dict(R=41), "rows"), (dict(R=-1), "rows"), (dict(left=-1), "negative"), (dict(right=-1), "negative"), (dict(sinks=-1), "negative"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
    (dict(ld=8 * 64 - 8), "qkv rows"), (dict(ld=8 * 64 + 4), "qkv rows"), (dict(qkv=(1 << 20) + 8), "qkv rows"), (dict(out=(1 << 20) + 2), "aligned"),
    (dict(NB=1 << 23, L=1 << 14, R=1 << 37), "grid"), (dict(L=1 << 29, R=1 << 30), "sequences"), (dict(H=4096, KV=2, ld=1 << 20), "columns")])
def test_window_attention_refuses(change, words):
    for name in ("star_attn_window_fwd", "star_attn_window_bwd"):
        _refused(getattr(L.lib(), name)(C.byref(_attn(**change)), None), name, words)
    _refused(L.lib().star_attn_window_fwd(None, None), "null")


@pytest.mark.parametrize("field", ["lse", "dout", "dqkv", "ws"])
def test_window_backward_refuses_missing_operands(field):
    _refused(L.lib().star_attn_window_bwd(C.byref(_attn(**{field: None})), None), "star_attn_window_bwd", "null")


def _step(**kw):
    a = dict(qkv=1 << 20, cache=1 << 20, lengths=1 << 20, out=1 << 20, ws=1 << 20, ld=8 * 64, NB=2, H=4, KV=2, hd=64, cap=64, left=31, sinks=4, scale=0.125, dt=L.F32)
    a.update(kw)
    return L.StarAttnStep(**a)


@pytest.mark.parametrize("change,words", [
    (dict(qkv=None), "null"), (dict(cache=None), "null"), (dict(lengths=None), "null"), (dict(out=None), "null"), (dict(dt=2), "dtype"), (dict(hd=40), "head dim"),
    (dict(KV=3), "bad shape"), (dict(NB=0), "bad shape"), (dict(left=60), "does not hold"), (dict(sinks=-1), "does not hold"), (dict(left=-1), "does not hold"),
    (dict(cap=0), "does not hold"), (dict(left=2147483647), "does not hold"), (dict(cap=2147483647), "slots"), (dict(scale=0.0), "scale"), (dict(ld=100), "rows"), (dict(ld=8 * 64 + 2), "rows"),
    (dict(cache=(1 << 20) + 8), "aligned"), (dict(cap=1 << 20, left=1 << 19, NB=1, ws=None), "workspace")])
def test_step_refuses(change, words):
    _refused(L.lib().star_attn_window_step(C.byref(_step(**change)), None), "star_attn_window_step", words)


def test_step_refuses_bad_rotations():
    for plan, pos, words in ((ops.rope_plan((8, 8)), None, "positions"), (ops.rope_plan((64,)), 1 << 20, "pairs"), (L.StarRope(pairs=0, axes=1), 1 << 20, "pairs"),
                             (L.StarRope(pairs=8, axes=0), 1 << 20, "pairs")):
        _refused(L.lib().star_attn_window_step(C.byref(_step(h_rope=C.pointer(plan), pos=pos, pos_ld=2)), None), words)
    plan = L.StarRope(pairs=8, axes=1)
    plan.axis[3] = 1
    _refused(L.lib().star_attn_window_step(C.byref(_step(h_rope=C.pointer(plan), pos=1 << 20, pos_ld=2)), None), "axis")


@pytest.mark.parametrize("change,words", [
    (dict(qkv=None), "null"), (dict(cache=None), "null"), (dict(lengths=None), "null"), (dict(dt=5), "dtype"), (dict(hd=12), "bad shape"), (dict(ld=64), "bad shape"),
    (dict(NB=0), "bad shape"), (dict(NB=70000, R=1400000), "bad shape"), (dict(L=-1), "bad shape"), (dict(sinks=64), "does not hold"), (dict(sinks=-1), "does not hold"),
    (dict(R=39), "rows"), (dict(ld=8 * 64 + 4), "aligned"), (dict(cap=2147483647), "slots")])
def test_append_refuses(change, words):
    a = dict(qkv=1 << 20, ld=8 * 64, offsets=None, cache=1 << 20, lengths=1 << 20, R=40, NB=2, L=20, H=4, KV=2, hd=64, cap=64, sinks=4, dt=L.BF16)
    a.update(change)
    _refused(L.lib().star_kv_append(*[a[k] for k in ("qkv", "ld", "offsets", "cache", "lengths", "R", "NB", "L", "H", "KV", "hd", "cap", "sinks", "dt")], None),
             "star_kv_append", words)


@pytest.mark.parametrize("change,words", [
    (dict(x=None), "null"), (dict(pos=None), "null"), (dict(dt=2), "dtype"), (dict(hd=24), "bad shape"), (dict(W=300), "bad shape"), (dict(rot=0), "bad shape"),
    (dict(rot=9), "bad shape"), (dict(R=-1), "bad shape"), (dict(hd=16), "pairs"), (dict(x_ld=8 * 64 - 8), "rows"), (dict(y_ld=8 * 64 + 2), "rows"),
    (dict(y=(1 << 20) + 8), "aligned"), (dict(pos_ld=3), "position"), (dict(y=1 << 20, y_ld=8 * 64 + 8), "strides"),
    (dict(y=(1 << 20) + 1024), "overlap"), (dict(y=(1 << 20) - 1024 * 9), "overlap"), (dict(x_ld=1200, y_ld=1200, y=(1 << 20) + 1008), "overlap"),
    (dict(x_ld=1200, y_ld=1200, y=(1 << 20) + 2 * 704), "overlap"), (dict(x_ld=1200, y_ld=1208, y=(1 << 20) + 2 * 600), "overlap")])
def test_rope_refuses(change, words):
    plan = ops.rope_plan((8, 12, 12))
    a = dict(x=1 << 20, x_ld=8 * 64, y=1 << 22, y_ld=8 * 64, pos=1 << 20, pos_ld=10, R=10, W=8 * 64, rot=6, hd=64, dt=L.BF16)
    a.update(change)
    _refused(L.lib().star_rope(a["x"], a["x_ld"], a["y"], a["y_ld"], a["pos"], a["pos_ld"], C.byref(plan), a["R"], a["W"], a["rot"], a["hd"], 0, a["dt"], None),
             "star_rope", words)


def test_rope_plan():
    plan = ops.rope_plan((2, 3, 3), base=100.0)
    assert (plan.pairs, plan.axes) == (8, 3) and list(plan.axis)[:8] == [0, 0, 1, 1, 1, 2, 2, 2]
    assert all(abs(plan.rev[i] * 2 * math.pi - 100.0 ** (-i / 8)) < 1e-15 for i in range(8))
    plan = ops.rope_plan((2, 6), base=100.0, per_axis=True, interleaved=True)
    assert plan.interleaved == 1
    assert all(abs(plan.rev[2 + i] * 2 * math.pi - 100.0 ** (-i / 6)) < 1e-15 for i in range(6))
    for bad in ((), (4,), (3, 4), (72,), (-8, 16), (8,) + (0,) * 8):
        with pytest.raises(ValueError):
            ops.rope_plan(bad)
    for base in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            ops.rope_plan((8,), base=base)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(4, 192)
    n = torch.zeros(4, dtype=torch.int32)
    cache = torch.zeros(2, 4, 4, 8, 16)
    for call in (lambda: ops.attn_window_fwd(x, 1, 4, 4, 16), lambda: ops.attn_window_bwd(x, x, x, x, 1, 4, 4, 16), lambda: ops.kv_append(x, cache, n, 1, 4),
                 lambda: ops.attn_window_step(x, cache, n, 4), lambda: ops.rope_fwd(x, n, 8, 16, (8,)), lambda: ops.rope_bwd(x, n, 8, 16, (8,))):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()


def test_step_takes_positions_and_sections_together():
    x, cache, n = torch.zeros(4, 192, device="meta"), torch.zeros(2, 4, 4, 8, 16, device="meta"), torch.zeros(4, dtype=torch.int32, device="meta")
    fn = ops._window_step.__wrapped__
    for pos, sections in ((None, (8,)), (torch.zeros(1, 4, dtype=torch.int32, device="meta"), None)):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(ops, "_home", lambda *t: 0)
            with pytest.raises(AssertionError, match="pos and sections"):
                fn(0, x, cache, n, 4, None, 0, pos, sections, 10000.0, False, False, None, None)


def test_structs_match_the_header(tmp_path):
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "star_hip.h"\nint main(void) { printf("%zu %zu %zu", sizeof(StarRope), sizeof(StarAttnWindow), sizeof(StarAttnStep)); return 0; }\n')
    subprocess.run(["cc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    sizes = [int(v) for v in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [C.sizeof(L.StarRope), C.sizeof(L.StarAttnWindow), C.sizeof(L.StarAttnStep)]
