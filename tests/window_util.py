"""float64 reference of sliding-window attention with sinks, rotary positions and the rolling cache, and how far a kernel may be off it.

half(t) is half a rounding step of type t relative to the value.  Error bounds are elementwise and come from the kernels' roundings alone:
  scores   float32 sums of hd products and one scaling: ES = 2^-24 (hd + 4) scale sum|q k|; a weight p = exp(s - lse) is off by a relative
           W = 2 (max ES of its row) + 2^-24 (n + 16)  (its own score, the row's sum, exp2's few ulp)
  P        rounded to the row type before the product with V (bf16): + half(t)
  out      |out - O| <= (W + half) sum p|v| + half |O| + sums' 2^-24 n sum p|v|
  backward the same for dV; delta = rowsum(dO * out) carries out's rounding: D = sum |dO| tol(out) + 2^-24 hd sum|dO O|;
           dS = P (dP - delta) is off by P (D + 2^-24 (hd + 2) sum|dO v|) + (W + half + 2^-23) |dS|; dQ, dK sum it against |K|, |Q|."""
import torch


def half(dtype):
    return torch.finfo(dtype).eps / 2


def seen(n, left, right, sinks):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    see = torch.ones(n, n, dtype=torch.bool)
    if right is not None:
        see &= j <= i + right
    if left is not None:
        see &= (j >= i - left) | (j < sinks)
    return see


def reference(q, k, v, left, right, sinks, scale=None, dout=None, dtype=torch.float32):
    """one sequence: q [h, n, hd], k, v [kv, n, hd], dout [h, n, hd] -> dict of float64 results and their error bounds"""
    h, n, hd = q.shape
    rep = h // k.shape[0]
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double().repeat_interleave(rep, 0), v.double().repeat_interleave(rep, 0)
    see = seen(n, left, right, sinks)
    f32 = 2.0 ** -24
    low = half(dtype) if dtype == torch.bfloat16 else 0.0
    end = half(dtype)
    s = (q @ k.transpose(1, 2)) * scale
    es = (f32 * (hd + 4) * scale * (q.abs() @ k.abs().transpose(1, 2))).masked_fill(~see, 0).amax(2, keepdim=True)
    s = s.masked_fill(~see, float("-inf"))
    lse = torch.logsumexp(s, 2, keepdim=True)
    p = torch.exp(s - lse)
    w = 2 * es + f32 * (n + 16)
    o = p @ v
    pv = p @ v.abs()
    tol_o = (w + low + f32 * n) * pv * 1.01 + end * o.abs() + 1e-30
    out = dict(out=o, tol_out=tol_o, lse=lse[..., 0] / 0.6931471805599453, tol_lse=((w + f32 * 4 * lse.abs()) / 0.69)[..., 0])
    if dout is not None:
        g = dout.double()
        dp = g @ v.transpose(1, 2)
        adp = g.abs() @ v.abs().transpose(1, 2)
        delta = (g * o).sum(2, keepdim=True)
        d = (g.abs() * tol_o).sum(2, keepdim=True) + f32 * hd * (g * o).abs().sum(2, keepdim=True)
        ds = p * (dp - delta)
        eds = p * (d + f32 * (hd + 2) * adp) + (w + low + 2 * f32) * ds.abs()
        ads = ds.abs() + eds
        kv = k.shape[0] // rep

        def group(x):
            return x.view(kv, rep, n, hd).sum(1)

        dq, dk, dv = scale * (ds @ k), group(scale * (ds.transpose(1, 2) @ q)), group(p.transpose(1, 2) @ g)
        edq = scale * ((eds + f32 * n * ads) @ k.abs()) + end * dq.abs()
        edk = group(scale * ((eds + f32 * n * rep * ads).transpose(1, 2) @ q.abs())) + end * dk.abs()
        edv = group(((w + low + f32 * n * rep) * p).transpose(1, 2) @ g.abs()) + end * dv.abs()
        out.update(dqkv=torch.cat((dq, dk, dv)), tol_dqkv=torch.cat((edq, edk, edv)) * 1.01 + 1e-30)
    return out


def unpack(x, h, kv, hd):
    """packed rows [n, (h + 2 kv) hd] -> q, k, v [heads, n, hd] on the CPU in float64"""
    t = x.detach().cpu().double().view(x.shape[0], h + 2 * kv, hd).transpose(0, 1)
    return t[:h], t[h:h + kv], t[h + kv:]


def heads(x, hd):
    """[n, heads*hd] -> [heads, n, hd] on the CPU in float64"""
    return x.detach().cpu().double().view(x.shape[0], -1, hd).transpose(0, 1)


def assert_within(got, want, tol, what):
    off = (got - want).abs()
    assert torch.isfinite(got).all(), "%s: not finite" % what
    bad = off > tol
    assert not bad.any(), "%s: %d of %d off, worst %.3g times the bound" % (what, int(bad.sum()), bad.numel(), float((off / tol).max()))


def rotate(x, pos, hd, rot, sections, base=10000.0, per_axis=False, interleaved=False, sign=1.0):
    """float64 [R, W] with the first rot heads turned; pos [axes, R]"""
    x = x.detach().cpu().double().clone()
    pos = pos.cpu().double()
    n = sum(sections)
    v = x[:, :rot * hd].view(x.shape[0], rot, hd)
    i = 0
    for axis, m in enumerate(sections):
        for k in range(m):
            t = sign * pos[axis] * base ** (-(k / m if per_axis else i / n))
            c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
            x1, x2 = v[:, :, a].clone(), v[:, :, b].clone()
            v[:, :, a], v[:, :, b] = x1 * c - x2 * s, x2 * c + x1 * s
            i += 1
    return x


def slot_of(p, sinks, cap):
    return p if p < sinks else sinks + (p - sinks) % (cap - sinks)
