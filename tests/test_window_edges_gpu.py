"""Calls of the window attention, rotary and cache operators at the edges of what they take: results on operands, bounds past 32 bits, rows
without a finite score, data that has gone NaN, the far queries of many sinks, very many rows."""
import pytest
import torch

from window_util import assert_within, heads, reference, seen, unpack

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from star_amd import ops

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float32]


def _rand(g, *shape, dtype=torch.float32, mul=1.0):
    return (torch.randn(*shape, generator=g) * mul).to(DEV).to(dtype)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- results that would lie on operands ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_results_on_operands_are_refused(dtype):
    g = _gen(1)
    n, h, kv, hd = 70, 4, 2, 32
    w = (h + 2 * kv) * hd
    qkv, dout = _rand(g, n, w, dtype=dtype), _rand(g, n, h * hd, dtype=dtype)
    out, lse = ops.attn_window_fwd(qkv, 1, n, h, hd, kv_heads=kv)
    want = ops.attn_window_bwd(qkv, out, dout, lse, 1, n, h, hd, kv_heads=kv)
    kept = qkv.clone()
    with pytest.raises(RuntimeError, match="dqkv overlaps"):
        ops.attn_window_bwd(qkv, out, dout, lse, 1, n, h, hd, kv_heads=kv, dqkv=qkv)
    with pytest.raises(RuntimeError, match="out overlaps"):
        ops.attn_window_fwd(qkv, 1, n, h, hd, kv_heads=kv, out=qkv.view(-1)[:n * h * hd].view(n, h * hd))
    cache, lengths = torch.zeros(2, 2, kv, 8, hd, dtype=dtype, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="out overlaps"):
        ops.attn_window_step(qkv[:2], cache, lengths, h, out=qkv.view(-1)[:2 * h * hd].view(2, h * hd))
    assert torch.equal(qkv, kept) and not cache.any()
    # between the rows of a wider matrix there is room for results
    wide = torch.zeros(3, w + 4 * h * hd, dtype=dtype, device=DEV)
    wide[:2, :w] = qkv[:2]
    gap = wide.view(-1)[w:w + 2 * h * hd].view(2, h * hd)
    assert torch.equal(ops.attn_window_fwd(wide[:2, :w], 1, 2, h, hd, kv_heads=kv, out=gap)[0], ops.attn_window_fwd(qkv[:2], 1, 2, h, hd, kv_heads=kv)[0])
    # and a single row may be computed in place
    row = qkv[3:4].clone()
    alone, _ = ops.attn_window_fwd(row, 1, 1, h, hd, kv_heads=kv)
    one = torch.zeros(2, 1, kv, 8, hd, dtype=dtype, device=DEV)
    step = ops.attn_window_step(row, one, lengths[:1], h)
    for call, result in ((lambda r: ops.attn_window_fwd(r, 1, 1, h, hd, kv_heads=kv, out=r[:, :h * hd]), alone),
                         (lambda r: ops.attn_window_step(r, one, lengths[:1], h, out=r[:, :h * hd]), step)):
        r = row.clone()
        call(r)
        assert torch.equal(r[:, :h * hd], result) and torch.equal(r[:, h * hd:], row[:, h * hd:])
    assert torch.equal(ops.attn_window_bwd(qkv, out, dout, lse, 1, n, h, hd, kv_heads=kv), want)


def test_bounds_past_32_bits():
    """a bound of any size over the sequence is no bound; lengths, heads and sizes past 32 bits are refused, not cut to their low half"""
    g = _gen(2)
    n, h, kv, hd = 90, 4, 2, 32
    qkv, dout = _rand(g, n, (h + 2 * kv) * hd), _rand(g, n, h * hd)
    for over in (1 << 31, 1 << 32, (1 << 32) + 5, 1 << 63):
        got = []
        for big in (None, over):
            kw = dict(kv_heads=kv, left=big, right=big)
            out, lse = ops.attn_window_fwd(qkv, 1, n, h, hd, **kw)
            got += [(out, lse, ops.attn_window_bwd(qkv, out, dout, lse, 1, n, h, hd, **kw))]
        out, lse = ops.attn_window_fwd(qkv, 1, n, h, hd, kv_heads=kv, left=3, right=0, sinks=over)
        ref, _ = ops.attn_window_fwd(qkv, 1, n, h, hd, kv_heads=kv, left=None, right=0)
        assert all(torch.equal(a, b) for a, b in zip(*got)) and torch.equal(out, ref)
        offsets = torch.tensor([0, n], device=DEV)
        cache, n32 = torch.zeros(2, 1, kv, 100, hd, device=DEV), torch.full((1,), n, dtype=torch.int32, device=DEV)
        pos = torch.zeros(1, n, dtype=torch.int32, device=DEV)
        for call in (lambda: ops.attn_window_fwd(qkv, 1, over, h, hd, kv_heads=kv, offsets=offsets), lambda: ops.attn_window_fwd(qkv, 1, n, h, hd, kv_heads=kv, left=-over),
                     lambda: ops.kv_append(qkv, cache, n32, over, h, offsets=offsets), lambda: ops.kv_append(qkv, cache, n32, n, h, sinks=over),
                     lambda: ops.attn_window_step(qkv[:1], cache, n32, h, left=over), lambda: ops.attn_window_step(qkv[:1], cache, n32, h, left=3, sinks=over),
                     lambda: ops.rope_fwd(qkv, pos, over + 2, hd, (8,)), lambda: ops.rope_fwd(qkv, pos, 2, over + 32, (8,))):
            with pytest.raises(RuntimeError, match="libstar_hip"):
                call()
        assert not cache.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_single_row_of_any_stride(dtype):
    """one token out of a matrix whose rows are no multiple of 16 bytes apart, or over 2^24 bytes: the stride of a single row does not matter"""
    g = _gen(3)
    h, kv, hd, sections = 4, 2, 32, (4, 6, 6)
    w = (h + 2 * kv) * hd
    lone = _rand(g, 1, w, dtype=dtype)
    pos = torch.full((3, 1), 77, dtype=torch.int32, device=DEV)
    n32 = torch.ones(1, dtype=torch.int32, device=DEV)

    def run(x):
        out, lse = ops.attn_window_fwd(x, 1, 1, h, hd, kv_heads=kv)
        cache = torch.zeros(2, 1, kv, 8, hd, dtype=dtype, device=DEV)
        ops.kv_append(x, cache, n32, 1, h)
        step = ops.attn_window_step(x, cache, n32, h, pos=pos, sections=sections)
        return out, lse, ops.attn_window_bwd(x, out, out, lse, 1, 1, h, hd, kv_heads=kv), cache, step, ops.rope_fwd(x, pos, h + kv, hd, sections)

    want = run(lone)
    for ld in (w + 1, (1 << 24) + 8):
        wide = torch.zeros(2, ld, dtype=dtype, device=DEV)
        wide[0, :w] = lone[0]
        for a, b in zip(run(wide[:1, :w]), want):
            assert torch.equal(a, b)
        view = wide[:1, :w]
        assert ops.rope_fwd(view, pos, h + kv, hd, sections, out=view) is view and torch.equal(view, want[-1])


# ---- rows without a finite score ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("nb", [1, 200])
def test_a_row_whose_scores_are_all_minus_infinity_is_nan(dtype, hd, nb):
    """the softmax of such a row is 0 / 0, in few sequences as in many; its neighbours keep their results"""
    g = _gen(hd)
    n, h, left = 70, 4, 3
    qkv = _rand(g, nb * n, 3 * h * hd, dtype=dtype)
    qkv[:, :h * hd] = qkv[:, :h * hd].abs() + 0.1
    clean = qkv.clone()
    x = qkv.view(nb, n, -1)
    x[:, [0, 40, 41, 42, 43], h * hd:2 * h * hd] = -float("inf")          # query 0 sees key 0 alone, query 43 keys 40 .. 43
    hit = torch.zeros(n, dtype=torch.bool)
    hit[[0, 43]] = True
    out, lse = ops.attn_window_fwd(qkv, nb, n, h, hd, left=left)
    out, lse = out.view(nb, n, -1).cpu(), lse.view(h, nb, n).cpu()
    assert out[:, hit].isnan().all() and (lse[:, :, hit] == -float("inf")).all()
    assert out[:, ~hit].isfinite().all() and lse[:, :, ~hit].isfinite().all()
    assert torch.equal(out[:, 50:], ops.attn_window_fwd(clean, nb, n, h, hd, left=left)[0].view(nb, n, -1)[:, 50:].cpu())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("nb,cap", [(3, 6000), (3, 40), (300, 40)])
def test_a_step_whose_scores_are_all_minus_infinity_is_nan(dtype, hd, nb, cap):
    """over split sequences as over whole ones; idle entries stay zeros"""
    g = _gen(hd + cap)
    h = kv = 4
    qkv = _rand(g, nb, 3 * h * hd, dtype=dtype)
    qkv[:, :h * hd] = qkv[:, :h * hd].abs() + 0.1
    cache = torch.randn(2, nb, kv, cap, hd, generator=torch.Generator(DEV).manual_seed(3), device=DEV).to(dtype)
    lengths = torch.full((nb,), cap, dtype=torch.int32, device=DEV)
    cache[0, 0] = -float("inf")
    qkv[0, h * hd:2 * h * hd] = -float("inf")
    lengths[1] = 0
    out = ops.attn_window_step(qkv, cache, lengths, h)
    assert out[0].isnan().all() and not out[1].any() and out[2:].isfinite().all()


# ---- data that has gone NaN -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,hd,left", [(torch.bfloat16, 64, None), (torch.bfloat16, 128, 600), (torch.float32, 32, None)])
def test_gradients_that_are_all_nan_take_no_sweep_of_their_own(dtype, hd, left):
    """a gradient of the result that is NaN everywhere: so is every gradient, in about the time of an ordinary pass.  (Rows formed again one
    visible row at a time would take 80 times as long.)"""
    g = _gen(hd)
    nb, n, h, kv = 2, 2048, 8, 2
    qkv, dout = _rand(g, nb * n, (h + 2 * kv) * hd, dtype=dtype), _rand(g, nb * n, h * hd, dtype=dtype)
    kw = dict(kv_heads=kv, left=left)
    out, lse = ops.attn_window_fwd(qkv, nb, n, h, hd, **kw)
    took = []
    for grad in (dout, torch.full_like(dout, float("nan"))):
        times = []
        for _ in range(6):
            marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            marks[0].record()
            dqkv = ops.attn_window_bwd(qkv, out, grad, lse, nb, n, h, hd, **kw)
            marks[1].record()
            torch.cuda.synchronize()
            times.append(marks[0].elapsed_time(marks[1]))
        took.append(min(times))
        assert (dqkv.isnan().all() if grad is not dout else dqkv.isfinite().all())
    assert took[1] < 10 * took[0], took


# ---- the far queries of the sinks -----------------------------------------------------------------------------------------------
def _passes(qkv, dout, nb, n, h, hd, **kw):
    out, lse = ops.attn_window_fwd(qkv, nb, n, h, hd, **kw)
    return out, lse, ops.attn_window_bwd(qkv, out, dout, lse, nb, n, h, hd, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("nb,sinks", [(1, 2), (48, 33), (1, 280), (1, 256), (1, 320), (40, 280)])
def test_far_queries(dtype, hd, nb, sinks):
    """sinks whose sweeps run far beyond the window, in few and in many sequences: shared out over blocks of their own, or (320 of 900 keys; 40 sequences
    of 280) left to the sinks' blocks"""
    g = _gen(hd + sinks)
    n, h, kv, left, right = 900, 4, 2, 20, 3
    qkv, dout = _rand(g, nb * n, (h + 2 * kv) * hd, dtype=dtype, mul=1.2), _rand(g, nb * n, h * hd, dtype=dtype)
    out, lse, dqkv = _passes(qkv, dout, nb, n, h, hd, kv_heads=kv, left=left, right=right, sinks=sinks)
    for b in sorted({0, nb - 1}):
        rows = slice(b * n, (b + 1) * n)
        want = reference(*unpack(qkv[rows], h, kv, hd), left, right, sinks, None, heads(dout[rows], hd), dtype)
        assert_within(heads(out[rows], hd), want["out"], want["tol_out"], "out")
        assert_within(heads(dqkv[rows], hd), want["dqkv"], want["tol_dqkv"], "dqkv")
    again = _passes(qkv, dout, nb, n, h, hd, kv_heads=kv, left=left, right=right, sinks=sinks)
    assert torch.equal(out, again[0]) and torch.equal(dqkv, again[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("nb", [1, 48])
def test_far_queries_that_are_not_finite_reach_their_sinks_alone(dtype, hd, nb):
    """infinities and NaN in rows far behind the sinks: the sinks and whoever else sees them take them, the keys beside the sinks do not"""
    g = _gen(hd + nb)
    n, h, kv, left, sinks = 1000, 4, 2, 24, 5
    see = seen(n, left, 0, sinks)
    clean, dout = _rand(g, nb * n, (h + 2 * kv) * hd, dtype=dtype), _rand(g, nb * n, h * hd, dtype=dtype)
    wild = torch.zeros(n, dtype=torch.bool)
    wild[[300, 301, 650] + list(range(960, 964))] = True
    at = wild.to(DEV)
    # every column of the rows and of the gradient NaN; values alone infinite; the gradient of the result alone
    for what, value in (("rows", float("nan")), ("values", float("inf")), ("gradient", float("nan")), ("gradient", float("inf"))):
        qkv, grad = clean.clone().view(nb, n, -1), dout.clone().view(nb, n, -1)
        if what != "gradient":
            qkv[:, at, 0 if what == "rows" else (h + kv) * hd:] = value
        if what != "values":
            grad[:, at] = value
        out, lse, dqkv = _passes(qkv.view(nb * n, -1), grad.view(nb * n, -1), nb, n, h, hd, kv_heads=kv, left=left, sinks=sinks)
        hit = (see & wild).any(1) if what != "gradient" else torch.zeros(n, dtype=torch.bool)          # queries whose result is not finite
        hit_q = hit | wild if what != "values" else hit
        hit_key = (see & hit_q[:, None]).any(0) | (wild if what != "gradient" else False)
        assert hit_key[:sinks].all() and not hit_key[sinks:250].any()
        for b in sorted({0, nb - 1}):
            rows = slice(b * n, (b + 1) * n)
            want = reference(*unpack(clean[rows], h, kv, hd), left, 0, sinks, None, heads(dout[rows], hd), dtype)
            o, d = heads(out[rows], hd), heads(dqkv[rows], hd)
            assert_within(o[:, ~hit], want["out"][:, ~hit], want["tol_out"][:, ~hit], "out")
            assert_within(d[:h, ~hit_q], want["dqkv"][:h, ~hit_q], want["tol_dqkv"][:h, ~hit_q], "dq")
            assert_within(d[h:, ~hit_key], want["dqkv"][h:, ~hit_key], want["tol_dqkv"][h:, ~hit_key], "dk, dv")
            if what == "rows" or what == "gradient":
                assert not torch.isfinite(d[h:, :sinks]).any()


# ---- very many rows -------------------------------------------------------------------------------------------------------------
def test_rope_of_more_rows_than_one_grid_holds():
    """2^27 rows and some, of one head: blocks of 256 threads for eight rows each are over 2^32 threads"""
    rows, hd, sections, part = (1 << 27) + 1003, 16, (4, 4), 1 << 25
    g = torch.Generator(DEV).manual_seed(7)
    x = torch.empty(rows, hd, dtype=torch.bfloat16, device=DEV)
    for at in range(0, rows, part):
        x[at:at + part] = torch.randn(min(part, rows - at), hd, generator=g, device=DEV)
    pos = torch.randint(0, 100000, (2, rows), generator=g, device=DEV, dtype=torch.int32)
    y = ops.rope_fwd(x, pos, 1, hd, sections)
    for at in range(0, rows, part):
        assert torch.equal(y[at:at + part], ops.rope_fwd(x[at:at + part], pos[:, at:at + part].contiguous(), 1, hd, sections)), at
    ops.rope_fwd(x, pos, 1, hd, sections, out=x)
    assert torch.equal(x, y)


# ---- prompts among idle entries -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nb", [40, 3000])
def test_append_of_unequal_prompts_among_many(dtype, nb):
    """more rows than a sequence's blocks take in one go, the sinks among them, beside empty and short sequences"""
    g = _gen(nb)
    h, kv, hd, cap, sinks = 2, 2, 64, 300, 5
    lens = [0] * nb
    lens[3], lens[nb // 2], lens[nb - 1], lens[7] = 20000, 1, 400, 290
    before = [(17 * b) % 700 for b in range(nb)]
    rows = sum(lens)
    qkv = torch.randn(rows, (h + 2 * kv) * hd, generator=torch.Generator(DEV).manual_seed(nb), device=DEV).to(dtype)
    cache = torch.randn(2, nb, kv, cap, hd, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(dtype)
    want = cache.clone()
    ends = torch.tensor(lens).cumsum(0)
    lengths = [n + c for n, c in zip(lens, before)]
    x = qkv.view(rows, h + 2 * kv, hd)
    for b, n in enumerate(lens):
        p = torch.arange(lengths[b] - n, lengths[b])
        keep = (p < sinks) | (p >= lengths[b] - (cap - sinks))
        slot = torch.where(p < sinks, p, sinks + (p - sinks) % (cap - sinks))[keep].to(DEV)
        src = x[int(ends[b]) - n:int(ends[b])][keep.to(DEV)]
        want[0, b][:, slot], want[1, b][:, slot] = src[:, h:h + kv].transpose(0, 1), src[:, h + kv:].transpose(0, 1)
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), ends)).to(DEV)
    ops.kv_append(qkv, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), max(lens), h, sinks=sinks, offsets=offsets)
    assert torch.equal(cache, want)


def test_append_takes_no_time_for_idle_entries():
    """one prompt among thousands of idle entries, against a call for the prompt alone.  (Entries that walk the longest one's rows take 2000 times
    its time.)"""
    rows, kv, hd, cap = 200000, 2, 64, 64
    qkv = torch.randn(rows, 3 * kv * hd, device=DEV)
    took = []
    for nb in (1, 4096):
        cache = torch.zeros(2, nb, kv, cap, hd, device=DEV)
        offsets = torch.full((nb + 1,), rows, dtype=torch.int64, device=DEV)
        offsets[0] = 0
        lengths = torch.zeros(nb, dtype=torch.int32, device=DEV)
        lengths[0] = rows
        times = []
        for _ in range(6):
            marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            marks[0].record()
            ops.kv_append(qkv, cache, lengths, rows, kv, offsets=offsets)
            marks[1].record()
            torch.cuda.synchronize()
            times.append(marks[0].elapsed_time(marks[1]))
        took.append(min(times))
    assert took[1] < 100 * took[0] and took[1] < 3.0, took


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("nb", [1, 48])
def test_one_element_that_is_not_finite_stays_in_its_column(dtype, hd, nb):
    """one NaN in one head's gradient of one result row, far behind the sinks: a column of dV, and dK, of the keys that the row sees, sinks included;
    the row's dQ; nothing else"""
    g = _gen(hd + nb)
    n, h, kv, left, sinks, row, col = 1300, 4, 2, 40, 5, 700, 11
    qkv, dout = _rand(g, nb * n, (h + 2 * kv) * hd, dtype=dtype), _rand(g, nb * n, h * hd, dtype=dtype)
    wild = dout.clone()
    wild.view(nb, n, h, hd)[:, row, 1, col] = float("nan")
    out, lse, dqkv = _passes(qkv, wild, nb, n, h, hd, kv_heads=kv, left=left, sinks=sinks)
    seen_keys = seen(n, left, 0, sinks)[row]
    for b in sorted({0, nb - 1}):
        rows = slice(b * n, (b + 1) * n)
        want = reference(*unpack(qkv[rows], h, kv, hd), left, 0, sinks, None, heads(dout[rows], hd), dtype)
        hit = torch.zeros(h + 2 * kv, n, hd, dtype=torch.bool)
        hit[1, row] = True                         # dQ of query head 1
        hit[h, seen_keys] = True                   # dK of its key head, 0
        hit[h + kv, seen_keys, col] = True         # and dV
        d = heads(dqkv[rows], hd)
        assert d[hit].isnan().all()
        assert_within(d[~hit], want["dqkv"][~hit], want["tol_dqkv"][~hit], "dqkv")


def test_a_far_element_that_is_not_finite_costs_no_sweep_of_the_sequence():
    """the sinks see every row: formed again one row at a time, their sums would take a second here.  The same element without sinks has the window's
    keys alone to form again."""
    g = _gen(9)
    n, h, hd, left = 32768, 8, 64, 100
    qkv, dout = _rand(g, n, (h + 2) * hd, dtype=torch.bfloat16), _rand(g, n, h * hd, dtype=torch.bfloat16)
    dout[20000, 5] = float("nan")
    took = []
    for sinks in (0, 4):
        kw = dict(kv_heads=1, left=left, sinks=sinks)
        out, lse = ops.attn_window_fwd(qkv, 1, n, h, hd, **kw)
        times = []
        for _ in range(3):
            marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            marks[0].record()
            ops.attn_window_bwd(qkv, out, dout, lse, 1, n, h, hd, **kw)
            marks[1].record()
            torch.cuda.synchronize()
            times.append(marks[0].elapsed_time(marks[1]))
        took.append(min(times))
    assert took[1] < 5 * took[0], took
