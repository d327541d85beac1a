"""What is measured of the rotary positions, the sliding-window attention and its rolling key/value cache: the cases, the operators in
plain torch (`own` false) and through star_amd.ops (`own` true), and their definition in 64 bits (`exact`).

Rows are packed as the qkv Linear lays them out: [query heads | key heads | value heads] x hd.  A query at position i sees a key at
position j when j <= i + right and (j >= i - left or j < sinks); a bound of -1 in a case means no bound."""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # 40 frames of 32 x 32 patches at two time stamps' worth of tokens, the light encoder's heads: q and k rotated in (t, y, x)
        dict(name="rope_frames", op="rope", way="fwd", type="bf16", rows=40960, heads=12, kv=12, hd=32, sections="4,6,6", interleaved=False),
        # gradient of the rotation in float32 for an odd number of tokens, far time stamps, adjacent pairs, part of every head rotated
        dict(name="rope_grad_f32", op="rope", way="bwd", type="f32", rows=997, heads=12, kv=4, hd=64, sections="8,8,8", interleaved=True),
        # a single odd sequence in float32: the smallest forward call
        dict(name="window_small_f32", op="attn", way="fwd", type="f32", nb=1, shortest=197, longest=197, ragged=False, heads=4, kv=4, hd=32,
             left=64, right=0, sinks=4),
        # a stream of four 1024-token frames per agent: every token sees the last frame's worth of tokens and the first 16
        dict(name="window_stream", op="attn", way="fwd", type="bf16", nb=5, shortest=4096, longest=4096, ragged=False, heads=12, kv=12, hd=64,
             left=1023, right=0, sinks=16),
        # long prefill with grouped heads: the largest forward
        dict(name="window_prefill", op="attn", way="fwd", type="bf16", nb=1, shortest=8192, longest=8192, ragged=False, heads=32, kv=8, hd=128,
             left=4095, right=0, sinks=4),
        # training on agents with different numbers of tokens (one of them absent), a window to both sides, grouped heads
        dict(name="train_ragged", op="attn", way="train", type="bf16", nb=7, shortest=0, longest=2043, ragged=True, heads=16, kv=4, hd=64,
             left=128, right=128, sinks=1),
        # training on long sequences with wide heads: the largest training step
        dict(name="train_long", op="attn", way="train", type="bf16", nb=2, shortest=8192, longest=8192, ragged=False, heads=16, kv=16, hd=128,
             left=2047, right=0, sinks=64),
        # float32 training at the light encoder's head size
        dict(name="train_f32", op="attn", way="train", type="f32", nb=2, shortest=1000, longest=1000, ragged=False, heads=12, kv=12, hd=32,
             left=255, right=0, sinks=8),
        # one frame's tokens of every agent put into the rolling caches behind what they hold
        dict(name="append_frame", op="append", type="bf16", nb=5, shortest=1024, longest=1024, ragged=False, before=1500, heads=12, kv=12, hd=64,
             cap=2064, sinks=16),
        # the caches of 16 requests filled from prompts of unequal lengths, the long ones longer than the ring
        dict(name="append_prompts", op="append", type="bf16", nb=16, shortest=301, longest=6000, ragged=True, before=0, heads=16, kv=8, hd=128,
             cap=4100, sinks=4),
        # one new token for each of five agents: the smallest call of serving
        dict(name="step_agents", op="step", type="bf16", nb=5, shortest=100, longest=2500, heads=12, kv=12, hd=64, cap=1040, left=1023, sinks=16,
             sections="8,12,12", interleaved=False),
        # one new token for each of 64 requests, long windows, grouped heads: the largest call of serving
        dict(name="step_requests", op="step", type="bf16", nb=64, shortest=3000, longest=20000, heads=32, kv=8, hd=128, cap=8196, left=8191,
             sinks=4, sections="16,24,24", interleaved=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rope", "fwd", "fwd", "train", "train", "append", "step", "step"])
    typ = rng.choice(["bf16", "bf16", "bf16", "f32"])
    hd = rng.choice([16, 32, 64, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 1, 2, 3, 4])
    n = hd // 2
    part = max(8, 3 * n // 32 * 8)            # three quarters of the head, where that is a multiple of eight pairs
    sections = rng.choice([(n // 4, n // 4 + n // 8, n - n // 2 - n // 8), (n // 2, n // 4, n // 4), (part // 4, part // 4, part // 2)])
    text = ",".join(str(s) for s in sections)
    if kind == "rope":
        return dict(op="rope", way=rng.choice(["fwd", "bwd"]), type=typ, rows=log(3, 30000), heads=heads, kv=kv, hd=hd, sections=text,
                    interleaved=rng.choice([False, True]))
    if kind in ("fwd", "train"):
        longest = log(1, 8000 if typ == "bf16" else 1500)
        nb = min(log(1, 16), max(1, int(1.5e9 / (heads * longest * longest))))      # what the largest listed case costs at most
        ragged = rng.choice([False, True])
        right = rng.choice([0, 0, 0, log(1, 600), -1])
        left = rng.choice([log(1, 4096), log(1, 600), -1])
        return dict(op="attn", way=kind, type=typ, nb=nb, shortest=rng.randint(0, longest) if ragged else longest, longest=longest, ragged=ragged,
                    heads=heads, kv=kv, hd=hd, left=left, right=right, sinks=rng.choice([0, 1, 4, 64, 100]))
    sinks = rng.choice([0, 1, 4, 16, 70])
    if kind == "append":
        longest = log(1, 5000)
        ragged = rng.choice([False, True])
        return dict(op="append", type=typ, nb=log(1, 16), shortest=rng.randint(0, longest) if ragged else longest, longest=longest, ragged=ragged,
                    before=rng.choice([0, log(1, 5000)]), heads=heads, kv=kv, hd=hd, cap=sinks + log(16, 4000), sinks=sinks)
    left = log(15, 8000)
    longest = log(1, 20000)
    most = int((2 if typ == "bf16" else 1) * 2.5e8 / ((left + 71) * kv * hd))           # what the largest listed case reads
    return dict(op="step", type=typ, nb=min(log(1, 64), max(1, most)), shortest=rng.randint(0, longest), longest=longest, heads=heads, kv=kv,
                hd=hd, cap=left + 1 + sinks + rng.choice([0, 0, 37]), left=left, sinks=sinks, sections=text, interleaved=rng.choice([False, True]))


def _spread(case):
    """the nb lengths of a case, evenly from the shortest to the longest"""
    nb, lo, hi = case["nb"], case["shortest"], case["longest"]
    return [hi if nb == 1 else lo + (hi - lo) * b // (nb - 1) for b in range(nb)]


def _visible_pairs(case, n):
    i = np.arange(n, dtype=np.int64)
    last = np.minimum(n - 1, i + case["right"]) if case["right"] >= 0 else np.full(n, n - 1)
    first = np.maximum(0, i - case["left"]) if case["left"] >= 0 else np.zeros(n, dtype=np.int64)
    return int((last - first + 1 + np.minimum(case["sinks"], first)).sum())


def work(case):
    es = 2 if case["type"] == "bf16" else 4
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    width = (h + 2 * kv) * hd
    if case["op"] == "rope":
        pairs = sum(int(s) for s in case["sections"].split(","))
        return {"bytes": 2 * case["rows"] * width * es + 12 * case["rows"], "flops": 6 * case["rows"] * (h + kv) * pairs}
    lens = _spread(case)
    if case["op"] == "attn":
        pairs = h * sum(_visible_pairs(case, n) for n in lens)
        rows = sum(lens)
        if case["way"] == "fwd":
            return {"bytes": rows * (width + h * hd) * es, "flops": 4 * hd * pairs}
        return {"bytes": rows * 2 * (width + h * hd) * es, "flops": 14 * hd * pairs}
    if case["op"] == "append":
        before, sinks = case["before"], case["sinks"]
        ring = case["cap"] - sinks
        kept = sum(max(0, min(sinks, before + n) - before) + max(0, before + n - max(sinks, before, before + n - ring)) for n in lens)
        return {"bytes": 2 * kept * 2 * kv * hd * es, "flops": 0}
    seen = sum(min(n, case["left"] + 1 + max(0, min(case["sinks"], n - 1 - case["left"]))) for n in lens)
    return {"bytes": seen * 2 * kv * hd * es + case["nb"] * (width + h * hd + 2 * kv * hd) * es, "flops": 4 * hd * h * seen}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _positions(g, rows):
    """(time, row, column) of the tokens of successive frames of 32 x 32 patches, the first frame somewhere in a long recording"""
    start = int(torch.randint(0, 200000, (1,), generator=g, device=DEV))
    t = torch.arange(rows, device=DEV)
    return torch.stack((start + t // 1024, (t // 32) % 32, t % 32)).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    typ = TYPES[case["type"]]
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    width = (h + 2 * kv) * hd

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(typ)

    st = {"case": case}
    if case["op"] == "rope":
        st["x"] = rand(case["rows"], width)
        st["pos"] = _positions(g, case["rows"])
        return st
    lens = _spread(case)
    ragged = case.get("ragged", False)
    if case["op"] in ("attn", "append"):
        rows = sum(lens) + (13 if ragged else 0)         # a ragged batch keeps a few rows behind its last sequence
        st["qkv"] = rand(rows, width)
        st["qkv"][:, :h * hd] *= 1.5                     # trained attention is sharper than that of unit normal rows
        if ragged:
            st["offsets"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int64, device=DEV)
        if case["op"] == "attn":
            if case["way"] == "train":
                st["dout"] = rand(rows, h * hd)
            return st
    st["cache"] = torch.empty(2, case["nb"], kv, case["cap"], hd, dtype=typ, device=DEV)
    if case["op"] == "append":
        st["cache"].zero_()
        st["lengths"] = torch.tensor([case["before"] + n for n in lens], dtype=torch.int32, device=DEV)
        return st
    for half in st["cache"]:
        half.normal_(generator=g)
    st["qkv"] = rand(case["nb"], width)
    st["qkv"][:, :h * hd] *= 1.5
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    last = st["lengths"].clamp(min=1) - 1
    st["pos"] = torch.stack((200000 + last // 1024, (last // 32) % 32, last % 32)).to(torch.int32)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def _bound(v):
    return None if v < 0 else v


def run(st):
    case = st["case"]
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    if own:
        from star_amd import ops
        if case["op"] == "rope":
            call = ops.rope_fwd if case["way"] == "fwd" else ops.rope_bwd
            return call(st["x"], st["pos"], h + kv, hd, _sections(case), interleaved=case["interleaved"])
        if case["op"] == "attn":
            args = dict(kv_heads=kv, left=_bound(case["left"]), right=_bound(case["right"]), sinks=case["sinks"], offsets=st.get("offsets"))
            out, lse = ops.attn_window_fwd(st["qkv"], case["nb"], case["longest"], h, hd, want_lse=case["way"] == "train", **args)
            if case["way"] == "fwd":
                return out
            return out, ops.attn_window_bwd(st["qkv"], out, st["dout"], lse, case["nb"], case["longest"], h, hd, **args)
        if case["op"] == "append":
            return ops.kv_append(st["qkv"], st["cache"], st["lengths"], case["longest"], h, sinks=case["sinks"], offsets=st.get("offsets"))
        out = ops.attn_window_step(st["qkv"], st["cache"], st["lengths"], h, left=case["left"], sinks=case["sinks"], pos=st["pos"],
                                   sections=_sections(case), interleaved=case["interleaved"])
        return out, st["cache"]
    if case["op"] == "rope":
        return _plain_rope(st["x"], st["pos"], h + kv, hd, _sections(case), case["interleaved"], 1.0 if case["way"] == "fwd" else -1.0).to(st["x"].dtype)
    if case["op"] == "attn":
        return _plain_attention(st)
    if case["op"] == "append":
        return _plain_append(st)
    return _plain_step(st)


def _plain_rope(x, pos, rot, hd, sections, interleaved, sign, base=10000.0):
    """float32 [rows, width]: the first `rot` heads rotated by sign * angle; angles in 64 bits (positions reach far)"""
    n = sum(sections)
    freq = base ** (-torch.arange(n, device=x.device, dtype=torch.float64) / n)
    angle = torch.cat([p.double()[:, None].expand(-1, width) for p, width in zip(pos, sections)], 1) * freq
    c, s = torch.cos(angle).float()[:, None], (sign * torch.sin(angle)).float()[:, None]
    y = x.float().clone()
    heads = y[:, :rot * hd].view(-1, rot, hd)[..., :2 * n]
    a, b = (heads[..., 0::2], heads[..., 1::2]) if interleaved else (heads[..., :n], heads[..., n:])
    ra, rb = a * c - b * s, b * c + a * s
    a.copy_(ra)
    b.copy_(rb)
    return y


def _index(st):
    """rows of the packed matrix as [nb, longest], and which of them are tokens"""
    case = st["case"]
    t = torch.arange(case["longest"], device=DEV)
    if "offsets" in st:
        start, end = st["offsets"][:-1, None], st["offsets"][1:, None]
    else:
        start = torch.arange(case["nb"], device=DEV)[:, None] * case["longest"]
        end = start + case["longest"]
    rows = start + t
    return rows.clamp(max=st["qkv"].shape[0] - 1), rows < end


def _plain_attention(st):
    case = st["case"]
    h, kv, hd, nb, l = case["heads"], case["kv"], case["hd"], case["nb"], case["longest"]
    rep, scale, typ = h // kv, hd ** -0.5, st["qkv"].dtype
    rows, real = _index(st)
    x = st["qkv"][rows].float().view(nb, l, h + 2 * kv, hd).transpose(1, 2)
    q, k, v = x[:, :h], x[:, h:h + kv].repeat_interleave(rep, 1), x[:, h + kv:].repeat_interleave(rep, 1)
    i, j = torch.arange(l, device=DEV)[:, None], torch.arange(l, device=DEV)[None]
    see = torch.ones(l, l, dtype=torch.bool, device=DEV)
    if case["right"] >= 0:
        see &= j <= i + case["right"]
    if case["left"] >= 0:
        see &= (j >= i - case["left"]) | (j < case["sinks"])
    hide = ~(see[None, None] & real[:, None, None, :])
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    p.masked_fill_(hide, -math.inf)
    p.sub_(p.amax(3, keepdim=True).nan_to_num(neginf=0.0)).exp_()
    p.div_(p.sum(3, keepdim=True).clamp(min=1e-30))
    o = torch.matmul(p, v)

    def packed(y):          # [nb, heads, l, hd] -> rows of the batch; rows of no sequence are zeros
        y = y.transpose(1, 2).reshape(nb * l, -1).to(typ)
        if not case["ragged"]:
            return y
        r = torch.zeros(st["qkv"].shape[0] + 1, y.shape[1], dtype=typ, device=DEV)       # the padding goes to a row behind the batch
        r[torch.where(real, rows, st["qkv"].shape[0]).view(-1)] = y
        return r[:-1]

    if case["way"] == "fwd":
        return packed(o)
    do = st["dout"][rows].float().view(nb, l, h, hd).transpose(1, 2) * real[:, None, :, None]
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    dp.sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq, dk = torch.matmul(dp, k), torch.matmul(dp.transpose(2, 3), q)
    dk, dv = dk.view(nb, kv, rep, l, hd).sum(2), dv.view(nb, kv, rep, l, hd).sum(2)
    return packed(o), packed(torch.cat((dq, dk, dv), 1))


def _held(case, last):
    """[nb, cap]: the position whose token a slot holds when `last` [nb, 1] is the newest one, or -1"""
    slot = torch.arange(case["cap"], device=DEV)
    sinks, ring = case["sinks"], case["cap"] - case["sinks"]
    p = torch.where(slot < sinks, slot, last - (last - slot) % ring)
    return torch.where((p <= last) & ((slot < sinks) | (p >= sinks)), p, -1)


def _plain_append(st):
    case = st["case"]
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    rows, real = _index(st)
    total = st["lengths"][:, None].long()
    held, first = _held(case, total - 1), total - real.sum(1, keepdim=True)
    t = (held - first).clamp(min=0)
    x = st["qkv"].view(-1, h + 2 * kv, hd)[rows.gather(1, t)].transpose(1, 2)           # [nb, heads, cap, hd]
    fresh = (held >= first)[:, None, :, None] & (held >= 0)[:, None, :, None]
    st["cache"].copy_(torch.where(fresh, torch.stack((x[:, h:h + kv], x[:, h + kv:])), st["cache"]))
    return st["cache"]


def _plain_step(st):
    case = st["case"]
    h, kv, hd, sinks, nb = case["heads"], case["kv"], case["hd"], case["sinks"], case["nb"]
    typ, cache = st["qkv"].dtype, st["cache"]
    x = _plain_rope(st["qkv"], st["pos"], h + kv, hd, _sections(case), case["interleaved"], 1.0).view(nb, h + 2 * kv, hd)
    last = st["lengths"][:, None].long() - 1
    held = _held(case, last)
    fresh = ((held == last) & (held >= 0))[:, None, :, None]
    cache[0].copy_(torch.where(fresh, x[:, h:h + kv, None].to(typ), cache[0]))
    cache[1].copy_(torch.where(fresh, x[:, h + kv:, None].to(typ), cache[1]))
    see = (held >= 0) & ((held >= last - case["left"]) | (held < sinks))
    q = x[:, :h].reshape(nb, kv, h // kv, hd)
    p = torch.matmul(q, cache[0].float().transpose(2, 3)) * hd ** -0.5
    p = p.masked_fill(~see[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(3, keepdim=True).nan_to_num(neginf=0.0))
    out = torch.matmul(p, cache[1].float()) / p.sum(3, keepdim=True).clamp(min=1e-30)
    return out.reshape(nb, h * hd).to(typ), cache


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def _exact_rotate(v, pos, sections, interleaved, sign):
    """v float64 [heads, rows, hd]"""
    n = sum(sections)
    out = v.clone()
    i = 0
    for axis, width in enumerate(sections):
        for _ in range(width):
            z = torch.polar(torch.ones_like(pos[axis], dtype=torch.float64), sign * pos[axis].double() * math.exp(-math.log(10000.0) * i / n))
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
            w = torch.complex(v[..., a], v[..., b]) * z
            out[..., a], out[..., b] = w.real, w.imag
            i += 1
    return out


def _exact_sequence(case, q, k, v, do):
    """one sequence in blocks of queries; q [h, n, hd], k and v [kv, n, hd] float64 -> out, dq, dk, dv"""
    h, n, hd = q.shape
    rep = h // k.shape[0]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for head in range(h):
        kk, vv = k[head // rep], v[head // rep]
        for lo in range(0, n, 2048):
            hi = min(n, lo + 2048)
            dist = torch.arange(n, device=DEV)[None] - torch.arange(lo, hi, device=DEV)[:, None]        # key minus query
            shut = torch.zeros_like(dist, dtype=torch.bool)
            if case["right"] >= 0:
                shut |= dist > case["right"]
            if case["left"] >= 0:
                shut |= (dist < -case["left"]) & (torch.arange(n, device=DEV)[None] >= case["sinks"])
            s = (q[head, lo:hi] @ kk.T) / math.sqrt(hd)
            s[shut] = -math.inf
            w = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
            out[head, lo:hi] = w @ vv
            if do is not None:
                g = do[head, lo:hi]
                dv[head // rep] += w.T @ g
                gw = g @ vv.T
                gs = w * (gw - (w * gw).sum(1, keepdim=True)) / math.sqrt(hd)
                dq[head, lo:hi] = gs @ kk
                dk[head // rep] += gs.T @ q[head, lo:hi]
    return out, dq, dk, dv


def exact(case, seed):
    st = prepare(case, seed)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "rope":
        x = st["x"].double()
        v = x[:, :(h + kv) * hd].reshape(-1, h + kv, hd).transpose(0, 1)
        v = _exact_rotate(v, st["pos"], _sections(case), case["interleaved"], 1.0 if case["way"] == "fwd" else -1.0)
        return torch.cat((v.transpose(0, 1).reshape(x.shape[0], -1), x[:, (h + kv) * hd:]), 1)
    lens = _spread(case)
    if case["op"] == "attn":
        train = case["way"] == "train"
        out = torch.zeros(st["qkv"].shape[0], h * hd, dtype=torch.float64, device=DEV)
        grad = torch.zeros(st["qkv"].shape, dtype=torch.float64, device=DEV)
        at = 0
        for n in lens:
            if n:
                x = st["qkv"][at:at + n].double().reshape(n, h + 2 * kv, hd).transpose(0, 1)
                do = st["dout"][at:at + n].double().reshape(n, h, hd).transpose(0, 1) if train else None
                o, dq, dk, dv = _exact_sequence(case, x[:h], x[h:h + kv], x[h + kv:], do)
                out[at:at + n] = o.transpose(0, 1).reshape(n, -1)
                grad[at:at + n] = torch.cat((dq, dk, dv)).transpose(0, 1).reshape(n, -1)
            at += n
        return (out, grad) if train else out
    cache = st["cache"].double() if case["op"] == "append" else st["cache"]
    sinks, ring = case["sinks"], case["cap"] - case["sinks"]
    if case["op"] == "append":
        at = 0
        for b, n in enumerate(lens):
            first = case["before"]
            pos = np.arange(first, first + n)
            x = st["qkv"][at:at + n].double().reshape(n, h + 2 * kv, hd)
            stay = np.flatnonzero((pos < sinks) | (pos >= first + n - ring))
            where = torch.from_numpy(np.where(pos < sinks, pos, sinks + (pos - sinks) % ring)[stay]).to(DEV)
            stay = torch.from_numpy(stay).to(DEV)
            cache[0, b][:, where] = x[stay, h:h + kv].transpose(0, 1)
            cache[1, b][:, where] = x[stay, h + kv:].transpose(0, 1)
            at += n
        return cache
    x = st["qkv"].double().reshape(-1, h + 2 * kv, hd).transpose(0, 1).contiguous()
    x[:h + kv] = _exact_rotate(x[:h + kv], st["pos"], _sections(case), case["interleaved"], 1.0)
    out = torch.zeros(case["nb"], h * hd, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        if not n:
            continue
        i = n - 1
        pos = np.concatenate((np.arange(0, min(sinks, i + 1)), np.arange(max(min(sinks, i + 1), i - case["left"]), i + 1)))
        where = torch.from_numpy(np.where(pos < sinks, pos, sinks + (pos - sinks) % ring)).to(DEV)
        mine = i if i < sinks else sinks + (i - sinks) % ring
        cache[0, b, :, mine], cache[1, b, :, mine] = x[h:h + kv, b].to(cache.dtype), x[h + kv:, b].to(cache.dtype)      # held in the cache's type
        k, v = cache[0, b][:, where].double(), cache[1, b][:, where].double()
        s = torch.matmul(k, x[:h, b].reshape(kv, h // kv, hd).transpose(1, 2).contiguous()) / math.sqrt(hd)
        w = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
        out[b] = torch.matmul(w.transpose(1, 2).contiguous(), v).reshape(-1)
    return out, cache.double()
