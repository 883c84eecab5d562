"""Plain 64-bit forms of the token operators and the error bounds their tolerances are derived from."""
import numpy as np
import torch

U32 = 2.0 ** -24            # half a step of fp32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def philox4x32(seed, counters):
    """Ten rounds of Philox4x32 on numpy uint64 counters (upper 64 counter bits zero) -> [n, 4] uint64 words."""
    return philox4x32_full([c for c in _words64(np.asarray(counters, dtype=np.uint64))] + [np.zeros(len(counters), np.uint64)] * 2,
                           [int(seed) & 0xFFFFFFFF, (int(seed) >> 32) & 0xFFFFFFFF])


def _words64(v):
    return v & np.uint64(0xFFFFFFFF), v >> np.uint64(32)


def philox4x32_full(c, key):
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(x, dtype=np.uint64) for x in c]
    k = list(key)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> sh) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def keep_mask(shape, p, seed, offset):
    """keep of every element of a 4-D map (NHWC order) or any other shape (row-major)."""
    n = int(np.prod(shape))
    ctr = (np.uint64(offset & 0xFFFFFFFFFFFFFFFF) + np.arange((n + 3) // 4, dtype=np.uint64))
    w = philox4x32(seed, ctr).reshape(-1)[:n]
    m = torch.from_numpy(w.astype(np.float64) >= round(p * 2 ** 32))
    if len(shape) == 4:
        b, c, h, ww = shape
        return m.reshape(b, h, ww, c).permute(0, 3, 1, 2)
    return m.reshape(shape)


def rotate(x, cos, sin):
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def norm_rotary(x, w, cos, sin, eps):
    return rotate(x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w, cos[..., None, :], sin[..., None, :])


def axis_bucket(d, num, far, both):
    """Bucket of one signed distance, straight from the definition in exact fractions."""
    half = num // 2 if both else num
    a = abs(d) if both else max(-d, 0)
    exact = half // 2
    if a < exact:
        b = a
    else:
        m = half - exact
        b = exact + max(t for t in range(m) if a ** m * exact ** t >= exact ** m * far ** t)
    return b + (half if both and d > 0 else 0)


def pair_buckets(shape, lq, lk, q_start, num, far, both=True):
    h, w = (1, shape) if isinstance(shape, int) else shape
    n = max(h, w)
    t = torch.tensor([axis_bucket(d, num, far, both) for d in range(-(n - 1), n)])
    q, k = q_start + torch.arange(lq), torch.arange(lk)
    bx = t[(k % w)[None] - (q % w)[:, None] + n - 1]
    return bx if h == 1 else t[(k // w)[None] - (q // w)[:, None] + n - 1] * num + bx


def attention(q, k, v, scale, mask=None, bias=None, dout=None, dtype=torch.float32, exact=False):
    """64-bit attention and, for every output, a bound on what the kernel's roundings can add up to.  q, k, v, dout: float64 holding the
    exact operand values; bias [H, Lq, Lk].  Returns {name: (value, bound)}."""
    b, lq, hq, d = q.shape
    g = hq // k.shape[2]
    kk, vv = (t.repeat_interleave(g, 2) for t in (k, v))
    if mask is not None:
        kk, vv = (torch.where(mask[:, :, None, None], t, 0.0) for t in (kk, vv))
    qh, kh, vh = (t.permute(0, 2, 1, 3) for t in (q, kk, vv))
    s = scale * (qh @ kh.transpose(-1, -2))
    sabs = scale * (qh.abs() @ kh.abs().transpose(-1, -2))
    if bias is not None:
        s = s + bias
        sabs = sabs + torch.where(bias.isfinite(), bias.abs(), 0.0)
    if mask is not None:
        s = s.masked_fill(~mask[:, None, None, :], -torch.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top.isfinite(), top, 0.0)
    e = (s - top).exp()
    z = e.sum(-1, keepdim=True)
    p = e / torch.where(z == 0, 1.0, z)
    o = p @ vh
    u = HALF_STEP[dtype]
    pu = 0.0 if dtype == torch.float32 else (0.0 if exact else u)       # rounding of the probabilities as product operands
    lk = s.shape[-1]
    # absolute error of a score (D products summed, the bias, the subtraction of the maximum), hence relative error of p and of its
    # row's sum; v_exp_f32 and the running rescale add a few steps more; Lk / 8 covers the sequential sums (fp32, worst case / 8)
    es = U32 * (d + 6) * sabs
    ep = 2 * es.amax(-1, keepdim=True) + U32 * (24 + lk / 8)
    ab = p @ vh.abs()
    eo = (pu + ep) * ab
    out = {"o": (o, eo + u * (o.abs() + eo))}
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    if dout is not None:
        gh = dout.permute(0, 2, 1, 3)
        dp = gh @ vh.transpose(-1, -2)
        dpa = gh.abs() @ vh.abs().transpose(-1, -2)
        delta = (gh * o).sum(-1, keepdim=True)
        ed = (gh.abs() * (eo + U32 * o.abs())).sum(-1, keepdim=True) + U32 * (d + 4) * (gh * o).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta)
        eds = p * (ep * (dpa + delta.abs()) + U32 * (d + 4) * dpa + ed) + U32 * 4 * ds.abs()
        su = 0.0 if dtype == torch.float32 else u
        eds2 = eds + su * (ds.abs() + eds)
        acc = U32 * 2                                                          # per summand of the products
        dv, edv = p.transpose(-1, -2) @ gh, (p * (su + ep + acc * lq)).transpose(-1, -2) @ gh.abs()
        dq, edq = scale * (ds @ kh), scale * ((eds2 + acc * lk * ds.abs()) @ kh.abs())
        dk, edk = scale * (ds.transpose(-1, -2) @ qh), scale * ((eds2 + acc * lq * ds.abs()).transpose(-1, -2) @ qh.abs())

        def shared(t):
            return back(t).reshape(b, lk, -1, g, d).sum(3)

        out["dq"] = (back(dq), back(edq + u * (dq.abs() + edq)))
        for name, t, et in (("dk", dk, edk), ("dv", dv, edv)):
            t, et = shared(t), shared(et)
            if mask is not None:
                t, et = t * mask[:, :, None, None], et * mask[:, :, None, None]
            out[name] = (t, et + u * (t.abs() + et))
        out["ds"] = (ds.sum(0), (eds + acc * (lq + lk) / 16 * ds.abs()).sum(0))
    out["o"] = (back(out["o"][0]), back(out["o"][1]))
    return out


def table_grad(ds, eds, buckets, rows):
    """Gradient of the bias table and its bound from those of the scores [H, Lq, Lk]."""
    z = lambda t: torch.zeros(rows, t.shape[0], dtype=torch.float64).index_add_(0, buckets.reshape(-1), t.reshape(t.shape[0], -1).T)  # noqa: E731
    dt = z(ds)
    return dt, z(eds) + U32 * 64 * z(ds.abs())


def check(got, value, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(value.shape)}"
    bad = ~((got - value).abs() <= bound + 1e-37)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside their bounds, worst error {(got - value).abs()[bad].max():.3e} "
                           f"(bound there {bound[bad].max():.3e}); not finite: {int((~got.isfinite()).sum())}")
