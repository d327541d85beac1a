"""Sliding-window attention with sinks, rotary positions and the rolling key/value cache against float64, at the sizes, windows and layouts
where they can go wrong.  Bounds are derived in window_util."""
import pytest
import torch

from window_util import assert_within, half, heads, reference, rotate, seen, slot_of, unpack

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from star_amd import ops

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float32]


def _rand(g, *shape, dtype=torch.float32, mul=1.0):
    return (torch.randn(*shape, generator=g) * mul).to(DEV).to(dtype)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _check(qkv, dout, lens, h, kv, hd, left, right, sinks, offsets=None, l=None, scale=None, backward=True):
    """forward and backward of a batch against float64, sequence by sequence; -> (out, lse, dqkv)"""
    nb, l = len(lens), max(lens) if l is None else l
    kw = dict(kv_heads=kv, left=left, right=right, sinks=sinks, offsets=offsets, scale=scale)
    out, lse = ops.attn_window_fwd(qkv, nb, l, h, hd, **kw)
    dqkv = ops.attn_window_bwd(qkv, out, dout, lse, nb, l, h, hd, **kw) if backward else None
    at = 0 if offsets is None else int(offsets[0])
    for n in lens:
        if n:
            q, k, v = unpack(qkv[at:at + n].contiguous(), h, kv, hd)
            want = reference(q, k, v, left, right, sinks, scale, heads(dout[at:at + n], hd) if backward else None, qkv.dtype)
            assert_within(heads(out[at:at + n], hd), want["out"], want["tol_out"], "out of %d" % n)
            assert_within(lse[:, at:at + n].cpu().double(), want["lse"], want["tol_lse"], "lse of %d" % n)
            if backward:
                assert_within(heads(dqkv[at:at + n], hd), want["dqkv"], want["tol_dqkv"], "dqkv of %d" % n)
        at += n
    return out, lse, dqkv


WINDOWS = [(None, 0, 0), (None, None, 0), (0, 0, 0), (5, 0, 1), (63, 0, 4), (64, 7, 0), (65, 0, 70), (20, None, 2), (128, 128, 1), (40, 3, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("window", WINDOWS)
def test_window_attention_against_float64(dtype, hd, window):
    left, right, sinks = window
    g = _gen(hd + sinks)
    for n, h, kv in ((1, 2, 1), (33, 3, 3), (129, 4, 2), (321, 2, 1)):
        qkv = _rand(g, 2 * n, (h + 2 * kv) * hd, dtype=dtype, mul=1.3)
        _check(qkv, _rand(g, 2 * n, h * hd, dtype=dtype), [n, n], h, kv, hd, left, right, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("window", WINDOWS)
def test_many_sequences(dtype, hd, window):
    """enough heads and sequences that four waves share a block's tiles (fewer: each wave sweeps its own part): three of them against float64"""
    left, right, sinks = window
    g = _gen(hd + sinks + 1)
    n, h, nb = 161, 12, 40
    qkv, dout = _rand(g, nb * n, 3 * h * hd, dtype=dtype, mul=1.3), _rand(g, nb * n, h * hd, dtype=dtype)
    kw = dict(left=left, right=right, sinks=sinks)
    out, lse = ops.attn_window_fwd(qkv, nb, n, h, hd, **kw)
    dqkv = ops.attn_window_bwd(qkv, out, dout, lse, nb, n, h, hd, **kw)
    for b in (0, 17, nb - 1):
        rows = slice(b * n, (b + 1) * n)
        q, k, v = unpack(qkv[rows], h, h, hd)
        want = reference(q, k, v, left, right, sinks, None, heads(dout[rows], hd), dtype)
        assert_within(heads(out[rows], hd), want["out"], want["tol_out"], "out %d" % b)
        assert_within(lse[:, rows].cpu().double(), want["lse"], want["tol_lse"], "lse %d" % b)
        assert_within(heads(dqkv[rows], hd), want["dqkv"], want["tol_dqkv"], "dqkv %d" % b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,rep", [(32, 2), (64, 4), (128, 3)])
def test_many_ragged_sequences_with_shared_heads(dtype, hd, rep):
    g = _gen(hd * rep)
    lens = [0, 300, 1, 64, 129, 31, 257, 500, 128, 2] * 6
    kv = 8
    h = kv * rep
    qkv, dout = _rand(g, sum(lens) + 3, (h + 2 * kv) * hd, dtype=dtype), _rand(g, sum(lens) + 3, h * hd, dtype=dtype)
    offsets = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], device=DEV)
    kw = dict(kv_heads=kv, left=70, right=9, sinks=5, offsets=offsets)
    out, lse = ops.attn_window_fwd(qkv, len(lens), 500, h, hd, **kw)
    dqkv = ops.attn_window_bwd(qkv, out, dout, lse, len(lens), 500, h, hd, **kw)
    for b in (1, 3, 6, 57, 58, 59):
        rows = slice(sum(lens[:b]), sum(lens[:b + 1]))
        q, k, v = unpack(qkv[rows], h, kv, hd)
        want = reference(q, k, v, 70, 9, 5, None, heads(dout[rows], hd), dtype)
        assert_within(heads(out[rows], hd), want["out"], want["tol_out"], "out %d" % b)
        assert_within(heads(dqkv[rows], hd), want["dqkv"], want["tol_dqkv"], "dqkv %d" % b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 31, 32, 63, 64, 65, 127, 128, 257, 512])
def test_every_tile_border(dtype, n):
    g = _gen(n)
    h, kv, hd = 2, 2, 64
    qkv = _rand(g, n, (h + 2 * kv) * hd, dtype=dtype)
    for left, right, sinks in ((31, 0, 1), (n, n, 0), (64, 1, 33), (1, 0, 65)):
        _check(qkv, _rand(g, n, h * hd, dtype=dtype), [n], h, kv, hd, left, right, sinks)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 32), (torch.bfloat16, 128)])
@pytest.mark.parametrize("window", [(None, 0, 0), (0, None, 0), (300, 0, 70)])
def test_long_sweeps(dtype, hd, window):
    """over 2048 rows: unequal sweeps of a window open to one side; sinks with a thousand queries beyond their window"""
    g = _gen(hd)
    n, h, kv = 2110, 2, 1
    left, right, sinks = window
    _check(_rand(g, n, (h + 2 * kv) * hd, dtype=dtype, mul=1.2), _rand(g, n, h * hd, dtype=dtype), [n], h, kv, hd, left, right, sinks)


@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_batch_leaves_rows_outside_every_sequence(dtype):
    g = _gen(5)
    h, kv, hd, lens = 6, 2, 32, [0, 1, 200, 0, 65, 31]
    first, rows = 3, 3 + sum(lens) + 9
    qkv = _rand(g, rows, (h + 2 * kv) * hd, dtype=dtype)
    dout = _rand(g, rows, h * hd, dtype=dtype)
    for t in (qkv, dout):                  # what no sequence holds is not read, whatever it is
        t[:first] = float("nan")
        t[first + sum(lens):] = float("inf")
    offsets = torch.tensor([first] + [first + sum(lens[:i + 1]) for i in range(len(lens))], device=DEV)
    out, lse, dqkv = _check(qkv, dout, lens, h, kv, hd, 40, 2, 3, offsets=offsets, l=256)
    for t in (out, dqkv):
        assert not t[:first].any() and not t[first + sum(lens):].any()
    kw = dict(kv_heads=kv, left=40, right=2, sinks=3, offsets=offsets)
    kept, grad = torch.full_like(out, 7.0), torch.full_like(dqkv, 7.0)
    ops.attn_window_fwd(qkv, len(lens), 256, h, hd, out=kept, **kw)
    ops.attn_window_bwd(qkv, out, dout, lse, len(lens), 256, h, hd, dqkv=grad, **kw)
    body = slice(first, first + sum(lens))
    assert torch.equal(kept[body], out[body]) and torch.equal(grad[body], dqkv[body])
    for t in (kept, grad):
        assert (t[:first] == 7).all() and (t[body.stop:] == 7).all()
    # a sequence over l rows takes part with its first l; offsets that lie outside the rows stay harmless
    short, _ = ops.attn_window_fwd(qkv[first:], 1, 64, h, hd, kv_heads=kv, offsets=torch.tensor([1, 201], device=DEV))
    want, _ = ops.attn_window_fwd(qkv[first + 1:first + 65].contiguous(), 1, 64, h, hd, kv_heads=kv)
    assert torch.equal(short[1:65], want) and not short[65:].any()
    wild, _ = ops.attn_window_fwd(qkv, 3, 64, h, hd, kv_heads=kv, offsets=torch.tensor([-5, -1, rows + 4, rows + 900], device=DEV))
    assert wild.shape == (rows, h * hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,l,front,back", [([5, 0, 90], 90, 700, 0), ([40, 7, 33], 20, 0, 1500), ([3, 70, 1, 0, 64, 65] * 120, 33, 5, 9), ([0, 0], 4, 0, 0), ([10], 10, 0, 0)])
def test_rows_of_no_sequence_become_zeros(dtype, lens, l, front, back):
    """in matrices that the calls make, whose memory held something else before: rows in front, behind, and of sequences over l rows"""
    g = _gen(len(lens) + l)
    h, kv, hd, rows = 4, 2, 32, front + sum(lens) + back
    if rows == 0:
        front, rows = 3, 3
    w = (h + 2 * kv) * hd
    qkv, dout = _rand(g, rows, w, dtype=dtype), _rand(g, rows, h * hd, dtype=dtype)
    at = [front]
    inside = torch.zeros(rows, dtype=torch.bool, device=DEV)
    for n in lens:
        inside[at[-1]:at[-1] + min(n, l)] = True
        at.append(at[-1] + n)
    offsets = torch.tensor(at, device=DEV)
    kw = dict(kv_heads=kv, left=20, sinks=2, offsets=offsets)
    kept, grad = torch.zeros(rows, h * hd, dtype=dtype, device=DEV), torch.zeros(rows, w, dtype=dtype, device=DEV)
    _, lse = ops.attn_window_fwd(qkv, len(lens), l, h, hd, out=kept, **kw)
    ops.attn_window_bwd(qkv, kept, dout, lse, len(lens), l, h, hd, dqkv=grad, **kw)
    for _ in range(3):
        poison = [torch.full((rows, c), float("nan"), dtype=dtype, device=DEV) for c in (h * hd, w) for _ in range(2)]
        del poison
        out, lse = ops.attn_window_fwd(qkv, len(lens), l, h, hd, **kw)
        dqkv = ops.attn_window_bwd(qkv, out, dout, lse, len(lens), l, h, hd, **kw)
        assert not out[~inside].any() and not dqkv[~inside].any()
        assert torch.equal(out, kept) and torch.equal(dqkv, grad)


def test_an_upper_bound_far_over_the_lengths():
    """l only bounds the sequences: a bound of millions costs and changes nothing"""
    g = _gen(71)
    h, kv, hd, lens = 4, 2, 64, [90, 0, 41]
    rows = sum(lens)
    qkv, dout = _rand(g, rows, (h + 2 * kv) * hd), _rand(g, rows, h * hd)
    offsets = torch.tensor([0, 90, 90, rows], device=DEV)
    got = []
    for l in (90, 1 << 28):
        kw = dict(kv_heads=kv, left=30, sinks=2, offsets=offsets)
        out, lse = ops.attn_window_fwd(qkv, 3, l, h, hd, **kw)
        cache = torch.zeros(2, 3, kv, 100, hd, device=DEV)
        ops.kv_append(qkv, cache, torch.tensor(lens, dtype=torch.int32, device=DEV), l, h, sinks=2, offsets=offsets)
        got.append((out, lse, ops.attn_window_bwd(qkv, out, dout, lse, 3, l, h, hd, **kw), cache))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("nb", [1, 40])
@pytest.mark.parametrize("window", [(None, 0, 0), (20, 0, 0), (33, 7, 0), (40, 0, 3)])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, hd, nb, window):
    """rows that hold infinities and NaN, in few and in many sequences: every row that sees none of them keeps its result and its gradient"""
    left, right, sinks = window
    g = _gen(hd + nb)
    n, h, kv = 150, 12, 6
    see = seen(n, left, right, sinks)
    clean, dout = _rand(g, nb * n, (h + 2 * kv) * hd, dtype=dtype), _rand(g, nb * n, h * hd, dtype=dtype)
    wild = torch.zeros(n, dtype=torch.bool)
    wild[[70, 71, 140] + list(range(147, 150))] = True
    for value, cols in ((float("nan"), slice(None)), (float("inf"), slice((h + kv) * hd, None))):
        qkv, grad = clean.clone().view(nb, n, -1), dout.clone().view(nb, n, -1)
        qkv[:, wild.to(DEV), cols] = value
        if cols == slice(None):
            grad[:, wild.to(DEV)] = value
        qkv, grad = qkv.view(nb * n, -1), grad.view(nb * n, -1)
        kw = dict(kv_heads=kv, left=left, right=right, sinks=sinks)
        out, lse = ops.attn_window_fwd(qkv, nb, n, h, hd, **kw)
        dqkv = ops.attn_window_bwd(qkv, out, grad, lse, nb, n, h, hd, **kw)
        hit = (see & wild).any(1) | (wild if cols == slice(None) else False)       # queries that see such a row
        hit_key = (see & hit[:, None]).any(0) | wild                              # keys that such a query sees
        for b in {0, nb // 2, nb - 1}:
            rows = slice(b * n, (b + 1) * n)
            q, k, v = unpack(clean[rows], h, kv, hd)
            want = reference(q, k, v, left, right, sinks, None, heads(dout[rows], hd), dtype)
            o, d = heads(out[rows], hd), heads(dqkv[rows], hd)
            assert not torch.isfinite(o[:, hit]).all(-1).any()
            assert cols != slice(None) or lse[:, rows].cpu()[:, hit].isnan().all()
            assert_within(o[:, ~hit], want["out"][:, ~hit], want["tol_out"][:, ~hit], "out")
            assert_within(d[:h, ~hit], want["dqkv"][:h, ~hit], want["tol_dqkv"][:h, ~hit], "dq")
            assert_within(d[h:, ~hit_key], want["dqkv"][h:, ~hit_key], want["tol_dqkv"][h:, ~hit_key], "dk, dv")


@pytest.mark.parametrize("n,hd", [(3, 64), (7, 128), (40, 32), (130, 16)])
@pytest.mark.parametrize("nb", [9, 300])
def test_gradients_of_few_visible_keys_carry_two_roundings(n, hd, nb):
    """dP - delta cancels where a key dominates, so a delta from rounded rows would be felt.  Left are the rounding of P or dS and that of the
    result, each off by at most half a step and evenly spread, so 1/sqrt(3) of that in the mean square: half(bf16) sqrt(2 / 3) together"""
    g = _gen(n)
    h = 6
    qkv, dout = _rand(g, nb * n, 3 * h * hd, dtype=torch.bfloat16, mul=1.2), _rand(g, nb * n, h * hd, dtype=torch.bfloat16)
    out, lse = ops.attn_window_fwd(qkv, nb, n, h, hd)
    dqkv = ops.attn_window_bwd(qkv, out, dout, lse, nb, n, h, hd)
    want = []
    for b in range(nb):
        rows = slice(b * n, (b + 1) * n)
        want.append(reference(*unpack(qkv[rows], h, h, hd), None, 0, 0, dout=heads(dout[rows], hd), dtype=torch.bfloat16)["dqkv"].transpose(0, 1).reshape(n, -1))
    want, got = torch.cat(want), dqkv.cpu().double()
    for i in range(3):
        cols = slice(i * h * hd, (i + 1) * h * hd)
        assert (got[:, cols] - want[:, cols]).norm() <= half(torch.bfloat16) * (2 / 3) ** 0.5 * want[:, cols].norm(), "dqdkdv"[2 * i:2 * i + 2]


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_scale(dtype):
    g = _gen(9)
    n, h, kv, hd = 150, 4, 1, 64
    w = (h + 2 * kv) * hd
    wide = _rand(g, 2 * n, w + 64, dtype=dtype)
    _check(wide[:, 32:32 + w], _rand(g, 2 * n, h * hd, dtype=dtype), [n, n], h, kv, hd, 70, 0, 2, scale=0.31)


def test_sharp_and_growing_scores():
    """scores that grow along the keys raise the running maximum in every tile; scores of hundreds leave one weight"""
    h, hd, n = 2, 64, 320
    for dtype in TYPES:
        g = _gen(3)
        qkv = _rand(g, n, 3 * h * hd, dtype=dtype)
        ramp = torch.linspace(0, 6, n, device=DEV)[:, None].to(dtype)
        qkv[:, h * hd:2 * h * hd] = ramp
        qkv[:, :h * hd] = qkv[:, :h * hd].abs()
        _check(qkv, _rand(g, n, h * hd, dtype=dtype), [n], h, h, hd, None, 0, 0)
        _check(qkv.flip(0).contiguous(), _rand(g, n, h * hd, dtype=dtype), [n], h, h, hd, 100, None, 5)
    sharp = _rand(_gen(4), n, 3 * h * hd, mul=12.0)
    _check(sharp, _rand(_gen(4), n, h * hd), [n], h, h, hd, 90, 0, 2)


def test_unbounded_window_is_the_dense_attention():
    nb, l, h, hd = 2, 200, 4, 32
    qkv = _rand(_gen(1), nb * l, 3 * h * hd)
    dout = _rand(_gen(2), nb * l, h * hd)
    out, lse = ops.attn_window_fwd(qkv, nb, l, h, hd, left=None, right=None)
    ref, rlse = ops.attn_fwd(qkv, nb, l, h, hd)
    torch.testing.assert_close(out, ref, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(lse.view(h, nb, l).transpose(0, 1), rlse, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(ops.attn_window_bwd(qkv, out, dout, lse, nb, l, h, hd, left=None, right=None),
                               ops.attn_bwd(qkv, ref, dout, rlse, nb, l, h, hd), rtol=1e-4, atol=1e-5)


def test_gradient_against_differences():
    """float32: (f(x + e d) - f(x - e d)) / 2e against <gradient, d>.  f = sum w out; out is off by some 1e-6 of its size, so the quotient by
    2^-24 * 16 * sqrt(elements) / e, and the third-order term by e^2: both under 2e-3 of the value's scale sqrt(elements)."""
    g = _gen(11)
    n, h, kv, hd, e = 90, 4, 2, 32, 2e-2
    args = (1, n, h, hd)
    kw = dict(kv_heads=kv, left=17, right=1, sinks=2)
    x, w, d = (_rand(g, n, c) for c in ((h + 2 * kv) * hd, h * hd, (h + 2 * kv) * hd))
    out, lse = ops.attn_window_fwd(x, *args, **kw)
    grad = ops.attn_window_bwd(x, out, w, lse, *args, **kw)
    up, down = (ops.attn_window_fwd(x + s * e * d, *args, **kw)[0].double() for s in (1, -1))
    slope, want = float(((up - down) * w.double()).sum() / (2 * e)), float((grad.double() * d.double()).sum())
    assert abs(slope - want) < 2e-3 * (n * h * hd) ** 0.5, (slope, want)


def test_same_bits_every_time_and_on_another_stream():
    g = _gen(8)
    nb, l, h, kv, hd = 3, 500, 8, 2, 64
    qkv, dout = _rand(g, nb * l, (h + 2 * kv) * hd, dtype=torch.bfloat16), _rand(g, nb * l, h * hd, dtype=torch.bfloat16)
    kw = dict(kv_heads=kv, left=100, sinks=4)

    def both():
        out, lse = ops.attn_window_fwd(qkv, nb, l, h, hd, **kw)
        return out, lse, ops.attn_window_bwd(qkv, out, dout, lse, nb, l, h, hd, **kw)

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    again = both()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


# ---- rotary positions ---------------------------------------------------------------------------------------------------------
def _rope_tol(x, dtype):
    """two products and a sum in float32, cosine and sine within 2^-22, then the rounding to the row type"""
    big = x.detach().cpu().double().abs().amax() * 1.5
    return big * (6 * 2.0 ** -24 + 2 * 2.0 ** -22 + half(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,sections", [(16, (2, 3, 3)), (32, (4, 6, 6)), (32, (0, 8)), (64, (8, 8, 8)), (128, (16, 24, 24)), (128, (64,)), (144, (8, 8))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_against_float64(dtype, hd, sections, interleaved):
    g = _gen(hd)
    for r, rot, more in ((1, 1, 0), (77, 5, 24), (1500, 3, 2 * hd)):
        w = rot * hd + more
        x = _rand(g, r, w, dtype=dtype)
        pos = torch.randint(-50, 3000000, (len(sections), r), generator=g).to(torch.int32).to(DEV)
        kw = dict(per_axis=r == 77, interleaved=interleaved, base=500.0 if r == 1 else 10000.0)
        y = ops.rope_fwd(x, pos, rot, hd, sections, **kw)
        want = rotate(x, pos, hd, rot, sections, **kw)
        assert_within(y.cpu().double(), want, _rope_tol(x, dtype), "rope")
        assert torch.equal(y[:, rot * hd:], x[:, rot * hd:])
        back = ops.rope_bwd(x, pos, rot, hd, sections, **kw)
        assert_within(back.cpu().double(), rotate(x, pos, hd, rot, sections, sign=-1.0, **kw), _rope_tol(x, dtype), "rope gradient")
        # in place, in rows of a wider matrix
        wide = torch.full((r, w + 40), 3.0, dtype=dtype, device=DEV)
        view = wide[:, 16:16 + w]
        view.copy_(x)
        assert ops.rope_fwd(view, pos, rot, hd, sections, out=view, **kw) is view
        assert torch.equal(view, y) and (wide[:, :16] == 3).all() and (wide[:, 16 + w:] == 3).all()
        assert torch.equal(ops.rope_fwd(view.copy_(x), pos, rot, hd, sections, **kw), y)
        both = torch.zeros(r, 2 * w, dtype=dtype, device=DEV)      # from one half of a matrix into the other
        both[:, :w] = x
        assert torch.equal(ops.rope_fwd(both[:, :w], pos, rot, hd, sections, out=both[:, w:], **kw), y) and torch.equal(both[:, :w], x)


def test_rope_gradient_is_the_adjoint_and_matches_differences():
    """a linear map: <rope(x), w> = <x, rope_bwd(w)>, and its difference quotient along d is <d, rope_bwd(w)> exactly but for rounding:
    sums of n products, each within 2^-21 of 2, in float64 -> n^0.5 * 2^-20 * 8"""
    g = _gen(2)
    r, rot, hd, sections = 200, 6, 64, (8, 12, 12)
    x, w, d = (_rand(g, r, (rot + 2) * hd) for _ in range(3))
    pos = torch.randint(0, 100000, (3, r), generator=g).to(torch.int32).to(DEV)
    f = lambda v: ops.rope_fwd(v, pos, rot, hd, sections).double()      # noqa: E731
    grad = ops.rope_bwd(w, pos, rot, hd, sections).double()
    tol = x.numel() ** 0.5 * 2.0 ** -17
    assert abs(float((f(x) * w.double()).sum() - (x.double() * grad).sum())) < tol
    slope = float(((f(x + d) - f(x - d)) * w.double()).sum() / 2)
    assert abs(slope - float((d.double() * grad).sum())) < 4 * tol


# ---- the rolling cache ----------------------------------------------------------------------------------------------------------
def _append_reference(cache, qkv, spans, lengths, h, sinks):
    kv, cap, hd = cache.shape[2:]
    ring = cap - sinks
    want = cache.clone()
    x = qkv.reshape(qkv.shape[0], h + 2 * kv, hd)
    for b, (lo, hi) in enumerate(spans):
        for t in range(lo, hi):
            p = lengths[b] - (hi - t)
            if p >= 0 and (p < sinks or p >= lengths[b] - ring):
                want[0, b, :, slot_of(p, sinks, cap)] = x[t, h:h + kv]
                want[1, b, :, slot_of(p, sinks, cap)] = x[t, h + kv:]
    return want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,h,cap,sinks", [(16, 3, 3, 40, 4), (64, 2, 8, 33, 0), (128, 1, 2, 300, 70), (32, 4, 4, 5, 4)])
def test_kv_append(dtype, hd, kv, h, cap, sinks):
    g = _gen(cap)
    for lens, before in (([3, 3], 0), ([1, 1], 500), ([0, 90, 7, 400], 11), ([64], 2)):
        ragged = len(set(lens)) > 1
        nb, rows = len(lens), sum(lens) + (5 if ragged else 0)
        wide = _rand(g, rows, (h + 2 * kv) * hd + 32, dtype=dtype)
        qkv = wide[:, :(h + 2 * kv) * hd]
        starts = [sum(lens[:b]) for b in range(nb)]
        lengths = [before + n for n in lens]
        cache = _rand(g, 2, nb, kv, cap, hd, dtype=dtype)
        want = _append_reference(cache, qkv, [(s, s + n) for s, n in zip(starts, lens)], lengths, h, sinks)
        offsets = torch.tensor(starts + [sum(lens)], device=DEV) if ragged else None
        got = ops.kv_append(qkv, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), max(lens), h, sinks=sinks, offsets=offsets)
        assert got is cache and torch.equal(cache, want), (lens, before)


def _step_reference(qkv, cache, lengths, h, left, sinks, pos, rope, scale):
    """float64 result, its bound and the cache afterwards (its type's values)"""
    nb = qkv.shape[0]
    kv, cap, hd = cache.shape[2:]
    rep = h // kv
    x = rotate(qkv, pos, hd, h + kv, **rope) if rope else qkv.detach().cpu().double()
    x = x.view(nb, h + 2 * kv, hd)
    want = cache.clone()
    out, tol = torch.zeros(nb, h, hd, dtype=torch.float64), torch.full((nb, h, hd), 1e-30, dtype=torch.float64)
    for b in range(nb):
        p = lengths[b] - 1
        if p < 0:
            continue
        new = slot_of(p, sinks, cap)
        want[0, b, :, new], want[1, b, :, new] = x[b, h:h + kv].to(cache.dtype).to(DEV), x[b, h + kv:].to(cache.dtype).to(DEV)
        at = sorted(set(range(min(sinks, p + 1))) | set(range(max(0, p - left), p + 1)))
        at = [slot_of(i, sinks, cap) for i in at]
        k, v = (t[b][:, at].cpu().double().repeat_interleave(rep, 0) for t in want)
        q = x[b, :h, None]
        s = (q @ k.transpose(1, 2)) * scale
        w = torch.softmax(s, 2)
        # float32 throughout: the turned query within 2^-20 of its size, sums of hd, the new key possibly one rounding step of its type off
        es = (scale * (q.abs() @ k.abs().transpose(1, 2))).amax(2, keepdim=True) * (2.0 ** -24 * (hd + 4) + 2.0 ** -20)
        rel = 2 * es + 2.0 ** -24 * (2 * len(at) + 16)
        out[b] = (w @ v)[:, 0]
        new_key = scale * (q.abs()[:, 0] * k.abs()[:, -1]).sum(1) * 2 * half(cache.dtype) if rope else torch.zeros(h)
        tol[b] = (rel * (w @ v.abs()))[:, 0] + half(cache.dtype) * out[b].abs() + new_key[:, None] * 2 * (w @ v.abs())[:, 0] * w[:, 0, -1:] + 1e-30
    return out.view(nb, -1), tol.view(nb, -1), want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,h", [(16, 2, 2), (32, 1, 3), (64, 2, 10), (64, 12, 12), (128, 2, 16), (128, 1, 12)])
def test_step(dtype, hd, kv, h):
    g = _gen(hd + h)
    rope = dict(sections=(hd // 8, hd // 8, hd // 4), interleaved=hd == 32)
    for cap, left, sinks, lengths in ((40, 35, 4, [1, 4, 5, 0, 39, 40, 41, 200]), (700, 600, 70, [700, 3000, 65, 71, 601]), (9, 0, 8, [3, 50]), (2000, None, 0, [1999, 2001])):
        for rp in (rope, None):
            nb = len(lengths)
            qkv = _rand(g, nb, (h + 2 * kv) * hd + 16, dtype=dtype)[:, :(h + 2 * kv) * hd]
            cache = _rand(g, 2, nb, kv, cap, hd, dtype=dtype)
            for b, n in enumerate(lengths):          # slots that hold no token yet are not read, whatever they are
                cache[:, b, :, min(cap, max(0, n - 1)):] = float("nan")
            if left is not None and left < cap - sinks - 1:
                for b, n in enumerate(lengths):      # nor are tokens that lie between the sinks and the window
                    for q in range(sinks, n - 1 - left):
                        if q >= n - (cap - sinks):
                            cache[:, b, :, slot_of(q, sinks, cap)] = float("inf")
            pos = torch.randint(0, 300000, (3, nb), generator=g).to(torch.int32).to(DEV) if rp else None
            bound = cap - sinks - 1 if left is None else left
            want, tol, after = _step_reference(qkv, cache, lengths, h, bound, sinks, pos, rp, hd ** -0.5)
            n32 = torch.tensor(lengths, dtype=torch.int32, device=DEV)
            out = ops.attn_window_step(qkv, cache, n32, h, left=left, sinks=sinks, pos=pos, **(rp or {}))
            assert_within(out.cpu().double(), want, tol, "step cap %d" % cap)
            assert not out[[i for i, n in enumerate(lengths) if n == 0]].any()
            same = (cache == after) | (cache.isnan() & after.isnan())
            if rp and not same.all():      # a turned key may round to the neighbouring value
                off = (cache.double() - after.double()).abs()[~same]
                assert (off <= 2 * 2 * half(dtype) * after.double().abs()[~same] + 2.0 ** -20).all()
            else:
                assert same.all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,rep,nb,cap,left", [(128, 8, 4, 36, 300, 290), (128, 8, 4, 36, 900, 880), (64, 8, 8, 34, 700, 600), (64, 8, 8, 34, 2500, 2400), (16, 16, 3, 20, 9000, 8990),
                                                   (32, 8, 5, 32, 3500, 3400), (32, 8, 8, 40, 100, 90)])
def test_step_with_key_heads_enough_to_fill_the_chip(dtype, hd, kv, rep, nb, cap, left):
    """four and eight query heads a block, whole sequences and splits"""
    g = _gen(hd + cap)
    h, sinks = kv * rep, 4
    lengths = [1 + (cap + 50) * b // (nb - 1) for b in range(nb)]
    lengths[nb // 2] = 0
    qkv = _rand(g, nb, (h + 2 * kv) * hd, dtype=dtype)
    cache = torch.randn(2, nb, kv, cap, hd, generator=torch.Generator(DEV).manual_seed(3), device=DEV).to(dtype)
    want, tol, after = _step_reference(qkv, cache, lengths, h, left, sinks, None, None, hd ** -0.5)
    out = ops.attn_window_step(qkv, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), h, left=left, sinks=sinks)
    assert_within(out.cpu().double(), want, tol, "step")
    assert torch.equal(cache, after)


@pytest.mark.parametrize("dtype", TYPES)
def test_prefill_then_steps_are_the_whole_sequence(dtype):
    """rotate + attend + fill the cache for a prompt, then single tokens: the rows of one forward pass over the whole sequence"""
    g = _gen(21)
    h, kv, hd, left, sinks, cap, prompt, total = 8, 2, 64, 50, 3, 60, 100, 131
    sections = (8, 12, 12)
    qkv = _rand(g, total, (h + 2 * kv) * hd, dtype=dtype)
    t = torch.arange(total, device=DEV)
    pos = torch.stack((4000 + t // 16, t // 4 % 4, t % 4)).to(torch.int32)
    turned = ops.rope_fwd(qkv, pos, h + kv, hd, sections)
    whole, _ = ops.attn_window_fwd(turned, 1, total, h, hd, kv_heads=kv, left=left, sinks=sinks, want_lse=False)
    cache = torch.full((2, 1, kv, cap, hd), float("nan"), dtype=dtype, device=DEV)
    n = torch.tensor([prompt], dtype=torch.int32, device=DEV)
    ops.kv_append(turned[:prompt], cache, n, prompt, h, sinks=sinks)
    q, k, v = unpack(turned, h, kv, hd)
    want = reference(q, k, v, left, 0, sinks, dtype=dtype)
    assert_within(heads(whole, hd), want["out"], want["tol_out"], "whole")
    for i in range(prompt, total):
        n += 1
        row = ops.attn_window_step(qkv[i:i + 1], cache, n, h, left=left, sinks=sinks, pos=pos[:, i:i + 1].contiguous(), sections=sections)
        # the step turns the query without rounding it to the row type: one rounding of q more in the whole pass' scores
        more = 4 * half(dtype) * (q[:, i].abs()[:, None] @ k.abs().repeat_interleave(h // kv, 0).transpose(1, 2)).amax() * hd ** -0.5 * v.abs().max()
        assert_within(heads(row, hd)[:, 0], want["out"][:, i], want["tol_out"][:, i] + more, "token %d" % i)


def test_training_chain_against_float64():
    """rotate, attend, backward through both: the gradient of the packed rows before the rotation"""
    g = _gen(31)
    n, h, kv, hd, sections = 140, 4, 2, 32, (4, 6, 6)
    x, w = _rand(g, n, (h + 2 * kv) * hd), _rand(g, n, h * hd)
    pos = torch.randint(0, 5000, (3, n), generator=g).to(torch.int32).to(DEV)
    turned = ops.rope_fwd(x, pos, h + kv, hd, sections)
    out, lse = ops.attn_window_fwd(turned, 1, n, h, hd, kv_heads=kv, left=30, sinks=2)
    grad = ops.attn_window_bwd(turned, out, w, lse, 1, n, h, hd, kv_heads=kv, left=30, sinks=2)
    grad = ops.rope_bwd(grad, pos, h + kv, hd, sections, out=grad)
    q, k, v = unpack(rotate(x, pos, hd, h + kv, sections), h, kv, hd)
    want = reference(q, k, v, 30, 0, 2, dout=heads(w, hd))
    rows = rotate(want["dqkv"].transpose(0, 1).reshape(n, -1), pos, hd, h + kv, sections, sign=-1.0)
    # float32 rotations of q, k (2^-20 of their size) move the scores by some 1e-5; everything is of size one
    torch.testing.assert_close(grad.cpu().double(), rows, rtol=1e-4, atol=2e-4)


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_replayed(dtype):
    """one graph of a training pass and one of a decoding step; replays interleaved with eager work give the eager results every time"""
    g = _gen(41)
    nb, l, h, kv, hd, cap, sinks = 2, 300, 4, 2, 64, 700, 5
    sections = (8, 12, 12)
    w = (h + 2 * kv) * hd
    x, dout = _rand(g, nb * l, w, dtype=dtype), _rand(g, nb * l, h * hd, dtype=dtype)
    pos = torch.randint(0, 5000, (3, nb * l), generator=g).to(torch.int32).to(DEV)
    row, rpos = _rand(g, nb, w, dtype=dtype), torch.randint(0, 5000, (3, nb), generator=g).to(torch.int32).to(DEV)
    lengths = torch.tensor([l, l], dtype=torch.int32, device=DEV)
    cache = torch.zeros(2, nb, kv, cap, hd, dtype=dtype, device=DEV)

    def train():
        t = ops.rope_fwd(x, pos, h + kv, hd, sections)
        out, lse = ops.attn_window_fwd(t, nb, l, h, hd, kv_heads=kv, left=80, sinks=sinks)
        return out, ops.rope_bwd(ops.attn_window_bwd(t, out, dout, lse, nb, l, h, hd, kv_heads=kv, left=80, sinks=sinks), pos, h + kv, hd, sections)

    def step():
        lengths.add_(1)
        return ops.attn_window_step(row, cache, lengths, h, sinks=sinks, pos=rpos, sections=sections)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), step()
    torch.cuda.current_stream().wait_stream(side)
    lengths.fill_(l)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        got_train = train()
    with torch.cuda.graph(graphs[1]):
        got_step = step()
    for i in range(4):
        x.copy_(_rand(g, nb * l, w, dtype=dtype))
        row.copy_(_rand(g, nb, w, dtype=dtype))
        lengths.fill_(l + 100 * i)
        before = cache.clone()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (*got_train, got_step, cache, lengths)]
        cache.copy_(before)
        lengths.fill_(l + 100 * i)
        eager = (*train(), step(), cache, lengths)
        for a, b in zip(kept, eager):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_lie_past_two_to_the_31_elements(dtype):
    """the last rows of a matrix of over 2^31 elements (and, float32, 2^33 bytes): rotation, both passes, append"""
    g = _gen(51)
    h, kv, hd, sections = 4, 2, 64, (8, 12, 12)
    w, ld = (h + 2 * kv) * hd, 1 << 16
    lens = [70, 0, 129]
    rows = (1 << 15) + 900
    first = rows - sum(lens)
    wide = torch.empty(rows, ld, dtype=dtype, device=DEV)
    qkv = wide[:, ld - w:]
    assert first * ld > 1 << 31
    qkv[first:] = _rand(g, sum(lens), w, dtype=dtype)
    pos = torch.randint(0, 5000, (3, rows), generator=g).to(torch.int32).to(DEV)
    want = ops.rope_fwd(qkv[first:].contiguous(), pos[:, first:].contiguous(), h + kv, hd, sections)
    assert torch.equal(ops.rope_fwd(qkv, pos, h + kv, hd, sections, out=qkv)[first:], want)
    offsets = torch.tensor([first, first + 70, first + 70, rows], device=DEV)
    dout = torch.zeros(rows, h * hd, dtype=dtype, device=DEV)
    dout[first:] = _rand(g, sum(lens), h * hd, dtype=dtype)
    at = first
    kw = dict(kv_heads=kv, left=40, sinks=2, offsets=offsets)
    out, lse = ops.attn_window_fwd(qkv, 3, 129, h, hd, **kw)
    dqkv = ops.attn_window_bwd(qkv, out, dout, lse, 3, 129, h, hd, **kw)
    for n in lens:
        if n:
            q, k, v = unpack(qkv[at:at + n].contiguous(), h, kv, hd)
            ref = reference(q, k, v, 40, 0, 2, dout=heads(dout[at:at + n], hd), dtype=dtype)
            assert_within(heads(out[at:at + n], hd), ref["out"], ref["tol_out"], "out of %d" % n)
            assert_within(heads(dqkv[at:at + n], hd), ref["dqkv"], ref["tol_dqkv"], "dqkv of %d" % n)
        at += n
    cache = torch.zeros(2, 3, kv, 140, hd, dtype=dtype, device=DEV)
    lengths = torch.tensor([70, 0, 129], dtype=torch.int32, device=DEV)
    ops.kv_append(qkv, cache, lengths, 129, h, sinks=2, offsets=offsets)
    x = qkv[first:].reshape(-1, h + 2 * kv, hd)
    assert torch.equal(cache[0, 2, :, :129], x[70:, h:h + kv].transpose(0, 1)) and torch.equal(cache[1, 0, :, :70], x[:70, h + kv:].transpose(0, 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_cache_past_two_to_the_31_elements(dtype):
    """two sequences of millions of slots: what the steps read and write lies behind 2^31 elements; the ring's end is passed on the way"""
    g = _gen(52)
    h, kv, hd, cap, sinks, left = 4, 1, 64, 1 << 24, 3, 500
    cache = torch.empty(2, 2, kv, cap, hd, dtype=dtype, device=DEV)
    lengths = [cap + 200, cap - 5]
    for b, n in enumerate(lengths):
        for p in list(range(sinks)) + list(range(n - 2 - left, n)):
            cache[:, b, :, slot_of(p, sinks, cap)] = _rand(g, 2, kv, hd, dtype=dtype)
    n32 = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    small = torch.zeros(2, 2, kv, 700, hd, dtype=dtype, device=DEV)      # the same tokens in a cache of the ordinary size, counted from there
    shift = [n - 650 for n in lengths]
    for b, n in enumerate(lengths):
        for p in list(range(sinks)) + list(range(n - 2 - left, n)):
            small[:, b, :, p if p < sinks else slot_of(p - shift[b], sinks, 700)] = cache[:, b, :, slot_of(p, sinks, cap)]
    s32 = torch.full((2,), 650, dtype=torch.int32, device=DEV)
    for _ in range(3):
        row = _rand(g, 2, (h + 2 * kv) * hd, dtype=dtype)
        out = ops.attn_window_step(row, cache, n32, h, left=left, sinks=sinks)
        assert torch.equal(out, ops.attn_window_step(row, small, s32, h, left=left, sinks=sinks))
        for b in range(2):
            slot = slot_of(int(n32[b]) - 1, sinks, cap)
            assert torch.equal(cache[0, b, 0, slot], row[b, h * hd:(h + 1) * hd]) and torch.equal(cache[1, b, 0, slot], row[b, (h + 1) * hd:])
        n32 += 1
        s32 += 1


def test_many_short_sequences():
    """more sequences than a grid has rows in its second dimension, one and two tokens each"""
    g = _gen(53)
    nb, h, kv, hd = 70000, 2, 1, 16
    qkv = _rand(g, nb, (h + 2 * kv) * hd, dtype=torch.bfloat16)
    dout = _rand(g, nb, h * hd, dtype=torch.bfloat16)
    out, lse = ops.attn_window_fwd(qkv, nb, 1, h, hd, kv_heads=kv)
    dqkv = ops.attn_window_bwd(qkv, out, dout, lse, nb, 1, h, hd, kv_heads=kv)
    v = qkv[:, 3 * hd:]
    assert torch.equal(out, v.repeat(1, 2))              # one visible key: its value, and a softmax without a gradient
    got = dqkv[:, 3 * hd:].double()
    want = dout.double().view(nb, 2, hd).sum(1)
    assert ((got - want).abs() <= half(torch.bfloat16) * want.abs() + 2.0 ** -20).all()
    # P dP - P delta: both are the same float32 sum but for its order and out's rounding (none here) -> a few 2^-24 of sums of 16 products
    assert (dqkv[:, :3 * hd].double().abs() < 2.0 ** -14).all()
    cache = torch.zeros(2, nb, kv, 4, hd, dtype=torch.bfloat16, device=DEV)
    n = torch.ones(nb, dtype=torch.int32, device=DEV)
    assert torch.equal(ops.attn_window_step(qkv, cache, n, h), out)
    assert torch.equal(cache[1, :, 0, 0], v) and not cache[:, :, :, 1:].any()


def test_calls_are_timed_by_the_profiler():
    g = _gen(61)
    h, kv, hd, nb, l = 4, 2, 32, 2, 40
    qkv, dout = _rand(g, nb * l, (h + 2 * kv) * hd), _rand(g, nb * l, h * hd)
    pos = torch.zeros(1, nb * l, dtype=torch.int32, device=DEV)
    cache, n = torch.zeros(2, nb, kv, 64, hd, device=DEV), torch.full((nb,), l, dtype=torch.int32, device=DEV)

    def run():
        x = ops.rope_fwd(qkv, pos, h + kv, hd, (8,))
        out, lse = ops.attn_window_fwd(x, nb, l, h, hd, kv_heads=kv)
        grad = ops.attn_window_bwd(x, out, dout, lse, nb, l, h, hd, kv_heads=kv)
        ops.kv_append(x, cache, n, l, h)
        return out, grad, ops.attn_window_step(qkv[:nb], cache, n, h)

    want = run()
    ops.PROFILER = ops.Profiler()
    try:
        got = run()
        torch.cuda.synchronize()
        tags = [r[0] for r in ops.PROFILER.records]
    finally:
        ops.PROFILER = None
    assert tags == ["rope", "attn_window_fwd", "attn_window_bwd", "kv_append", "attn_window_step"]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_batches():
    none = torch.zeros(0, 192, device=DEV)
    out, lse = ops.attn_window_fwd(none, 2, 0, 4, 16, offsets=torch.zeros(3, dtype=torch.int64, device=DEV))
    assert out.shape == (0, 64) and lse.shape == (4, 0)
    assert ops.attn_window_bwd(none, out, out, lse, 2, 0, 4, 16, offsets=torch.zeros(3, dtype=torch.int64, device=DEV)).shape == (0, 192)
    assert ops.rope_fwd(none, torch.zeros(1, 0, dtype=torch.int32, device=DEV), 8, 16, (8,)).shape == (0, 192)
    cache = torch.ones(2, 2, 4, 8, 16, device=DEV)
    ops.kv_append(none, cache, torch.zeros(2, dtype=torch.int32, device=DEV), 0, 4)
    out = ops.attn_window_step(torch.ones(2, 192, device=DEV), cache, torch.zeros(2, dtype=torch.int32, device=DEV), 4)
    assert not out.any() and (cache == 1).all()
    idle, _ = ops.attn_window_fwd(torch.ones(5, 192, device=DEV), 2, 4, 4, 16, offsets=torch.zeros(3, dtype=torch.int64, device=DEV))
    assert not idle.any()
