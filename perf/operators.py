"""Workloads of the token operators (`shineon_virtual_tryon_amd.ops_tokens`): dropout from a counter, per-head norms of queries and
keys with the position rotation, attention with a learned relative position bias.  Each case is one pass through one operator;
`own` selects the framework's kernels or the plain form in elementary torch operations."""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # dropout behind the innermost U-Net blocks (16 x 12 maps of 512 channels at 256 x 192 frames), batch of 4: latency
        dict(name="dropout_map_f32", op="dropout", dtype="f32", shape="4,512,16,12", p=0.5, residual=False),
        # residual branch of a token block in training: 8 clips of 4099 tokens, 1024 channels
        dict(name="dropout_tokens_bf16", op="dropout", dtype="bf16", shape="8,4099,1024", p=0.1, residual=True),
        # the same in the framework's own type, sizes that no vector width divides
        dict(name="dropout_odd_f32", op="dropout", dtype="f32", shape="3,1537,775", p=0.2, residual=True),
        # queries and keys of the 16 x 12 attention map, 8 heads of 64, trained
        dict(name="qknorm_map_f32", op="qknorm", dtype="f32", b=4, h=16, w=12, heads=8, kv=8, d=64, rot=64, train=True),
        # a long clip with shared key heads, trained
        dict(name="qknorm_seq_bf16", op="qknorm", dtype="bf16", b=2, h=1, w=8191, heads=16, kv=4, d=128, rot=128, train=True),
        # one new token per stream, far positions
        dict(name="qknorm_token_bf16", op="qknorm", dtype="bf16", b=16, h=1, w=1, heads=16, kv=4, d=128, rot=128, train=False),
        # the 16 x 12 map of the U-Net's attention, 8 heads of 64, training step: latency
        dict(name="attn_map_f32", op="attn", dtype="f32", b=4, h=16, w=12, lq=192, heads=8, kv=8, d=64, train=True, fill=1.0),
        # a 64 x 36 map (one level further up), training step
        dict(name="attn_map_bf16", op="attn", dtype="bf16", b=2, h=64, w=36, lq=2304, heads=8, kv=8, d=64, train=True, fill=1.0),
        # a ragged clip batch in the framework's own type, training step
        dict(name="attn_seq_f32", op="attn", dtype="f32", b=2, h=1, w=2049, lq=2049, heads=8, kv=8, d=64, train=True, fill=0.7),
        # long ragged clips, wide heads shared by groups of four, training step
        dict(name="attn_seq_bf16", op="attn", dtype="bf16", b=2, h=1, w=4097, lq=4097, heads=16, kv=4, d=128, train=True, fill=0.8),
        # inference over one long clip
        dict(name="attn_long_bf16", op="attn", dtype="bf16", b=1, h=1, w=8191, lq=8191, heads=16, kv=16, d=64, train=False, fill=1.0),
        # one new token per stream against a long history
        dict(name="attn_token_bf16", op="attn", dtype="bf16", b=8, h=1, w=32765, lq=1, heads=16, kv=4, d=128, train=False, fill=0.9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "qknorm", "attn", "attn"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "dropout":
        c, n = _log(rng, 1, 1500), _log(rng, 1, 8000)
        b = max(1, min(rng.randint(1, 8), 33_000_000 // (n * c)))
        shape = "%d,%d,%d,%d" % (b, c, _log(rng, 1, 128), _log(rng, 1, 96)) if rng.random() < 0.3 and c < 600 else "%d,%d,%d" % (b, n, c)
        return dict(op=op, dtype=dtype, shape=shape, p=rng.choice([0.05, 0.1, 0.2, 0.5, 0.73]), residual=rng.random() < 0.5)
    kv = rng.choice([1, 2, 4, 5, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    d = rng.choice([32, 40, 64, 64, 72, 96, 128, 128])
    b = rng.randint(1, 6)
    h, w = (1, _log(rng, 1, 8000)) if rng.random() < 0.5 else (_log(rng, 2, 72), _log(rng, 2, 48))
    train = rng.random() < 0.6
    if op == "qknorm":
        b = max(1, min(b, 39_000_000 // (h * w * (heads + kv) * d)))
        return dict(op=op, dtype=dtype, b=b, h=h, w=w, heads=heads, kv=kv, d=d, rot=rng.choice([d, d, d // 4 * 2]), train=train)
    lq = h * w
    if not train and rng.random() < 0.5:
        lq = rng.choice([1, 1, 1, 2, 5])
        h, w = 1, _log(rng, 64, 32000)
    cost = 1 if dtype == "bf16" else 8
    while b > 1 and b * heads * lq * h * w * d * cost > 2 * 16 * 4097 * 4097 * 128:
        b -= 1
    while b * heads * lq * h * w * d * cost > 2 * 16 * 4097 * 4097 * 128 and heads > kv:
        heads = kv
    if b * heads * lq * h * w * d * cost > 2 * 16 * 4097 * 4097 * 128:
        h, w = 1, w + 1000
        lq = w if lq > 5 else lq
    return dict(op=op, dtype=dtype, b=b, h=h, w=w, lq=lq, heads=heads, kv=kv, d=d, train=train, fill=rng.choice([1.0, 1.0, 0.9, 0.6, 0.3]))


def _lengths(case):
    """Visible keys of each sample: ragged below `fill`, the last of several short samples without any."""
    n, f = case["h"] * case["w"], case["fill"]
    if f == 1.0:
        return [n] * case["b"]
    lens = [max(1, int(n * min(1.0, f * (0.8 + 0.4 * i / max(1, case["b"] - 1))))) for i in range(case["b"])]
    if f < 0.5 and case["b"] > 1:
        lens[-1] = 0
    return lens


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "dropout":
        n = math.prod(int(s) for s in case["shape"].split(","))
        return {"bytes": n * e * (4 + (1 if case["residual"] else 0)), "flops": 4 * n}
    tokens = case["b"] * case["h"] * case["w"]
    if case["op"] == "qknorm":
        n = tokens * (case["heads"] + case["kv"]) * case["d"]
        return {"bytes": n * e * (5 if case["train"] else 2) + case["h"] * case["w"] * case["rot"] * 4, "flops": n * (16 if case["train"] else 6)}
    seen = sum(_lengths(case))
    fq, fk = case["b"] * case["lq"] * case["heads"] * case["d"] * e, seen * case["kv"] * case["d"] * e
    pairs = case["heads"] * case["lq"] * seen * case["d"]
    if not case["train"]:
        return {"bytes": 2 * fq + 2 * fk, "flops": 4 * pairs}
    return {"bytes": 4 * fq + 4 * fk, "flops": 14 * pairs}


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = dict(case=case, t=t)
    if case["op"] == "dropout":
        shape = [int(v) for v in case["shape"].split(",")]

        def rows():
            x = normal(*shape)
            return x.contiguous(memory_format=torch.channels_last) if x.dim() == 4 else x

        s.update(x=rows().requires_grad_(), dy=rows(), residual=rows().requires_grad_() if case["residual"] else None)
        s["rng"] = torch.tensor([seed * 1000003 + 17, 2 ** 32 - 5 + seed], dtype=torch.int64, device="cuda")
        return s
    b, h, w, heads, kv, d = (case[k] for k in ("b", "h", "w", "heads", "kv", "d"))
    n = h * w
    if case["op"] == "qknorm":
        # q | k | v side by side, as one projection leaves them
        qkv = normal(b, n, (heads + 2 * kv) * d, std=2.0)
        s["q"] = qkv[..., :heads * d].unflatten(-1, (heads, d))
        s["k"] = qkv[..., heads * d:(heads + kv) * d].unflatten(-1, (kv, d))
        s["wq"], s["wk"] = (1 + normal(d, std=0.1, dtype=torch.float32) for _ in range(2))
        r = case["rot"]
        far = 60000 if n == 1 else 0
        pos = torch.arange(far + n, dtype=torch.float64, device="cuda")
        if h == 1:
            angle = pos[:, None] * 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
        else:       # the first half of the pairs turns with the row, the second half with the column
            ny = r // 4
            freq = torch.cat([10000.0 ** (-torch.arange(m, dtype=torch.float64, device="cuda") / m) for m in (ny, r // 2 - ny) if m])
            yx = torch.stack([pos // w, pos % w], 1)
            angle = yx[:, [0] * ny + [1] * (r // 2 - ny)] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["pos"] = torch.randint(0, far + 1, (b, 1), generator=g, device="cuda") if n == 1 else None
        if case["train"]:
            s["dq"], s["dk"] = normal(b, n, heads, d), normal(b, n, kv, d)
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["wq"].requires_grad_()
            s["wk"].requires_grad_()
        return s
    lq = case["lq"]
    s["q"], s["k"], s["v"] = normal(b, lq, heads, d), normal(b, n, kv, d), normal(b, n, kv, d)
    per = 32 if h == 1 else 16
    s["table"] = normal(per if h == 1 else per * per, heads, std=0.5, dtype=torch.float32)
    s["per"], s["far"] = per, 128 if h == 1 else 32
    s["start"] = 0 if lq == n else n - lq
    s["mask"] = None
    if case["fill"] < 1.0:
        s["mask"] = torch.arange(n, device="cuda")[None, :] < torch.tensor(_lengths(case), device="cuda")[:, None]
    s["bucket"] = _axis_buckets(max(h, w), per, s["far"])
    if case["train"]:
        s["do"] = normal(b, lq, heads, d)
        for k in ("q", "k", "v", "table"):
            s[k].requires_grad_()
    if own:
        from shineon_virtual_tryon_amd import ops_tokens

        s["relative"] = ops_tokens.RelativePositions(n if h == 1 else (h, w), num_buckets=per, max_distance=s["far"], device="cuda")
    return s


def _axis_buckets(n, buckets, far):
    """Bucket of every distance -(n - 1) .. n - 1 along one axis: the sign takes half of the buckets, distances below half of those
    have one each, the others share logarithmically spaced ones up to `far`.  A distance reaches step t of the m logarithmic ones
    when dist^m exact^t >= exact^m far^t, decided in whole numbers."""
    half = buckets // 2
    exact = half // 2
    m = half - exact
    bound = np.array([next(d for d in range(exact, far + 1) if d ** m * exact ** t >= exact ** m * far ** t) for t in range(1, m)])
    dist = np.arange(-(n - 1), n)
    a = np.abs(dist)
    b = np.where(a < exact, a, exact + (a[:, None] >= bound[None, :]).sum(1))
    return torch.from_numpy(b + half * (dist > 0)).cuda()


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if case["op"] == "dropout":
        return _own_dropout(s) if own else _plain_dropout(s)
    if case["op"] == "qknorm":
        return _own_qknorm(s) if own else _plain_qknorm(s)
    return _own_attention(s) if own else _plain_attention(s)


def _own_dropout(s):
    from shineon_virtual_tryon_amd import ops_tokens

    y = ops_tokens.dropout(s["x"], s["case"]["p"], s["rng"], residual=s["residual"])
    (dx,) = torch.autograd.grad(y, [s["x"]], s["dy"])
    return {"y": y.detach(), "dx": dx}


def _own_qknorm(s):
    from shineon_virtual_tryon_amd import ops_tokens

    q, k = ops_tokens.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], positions=s["pos"], eps=1e-6)
    if not s["case"]["train"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad([q, k], [s["q"], s["k"], s["wq"], s["wk"]], [s["dq"], s["dk"]])
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _own_attention(s):
    from shineon_virtual_tryon_amd import ops_tokens

    o = ops_tokens.attention(s["q"], s["k"], s["v"], key_mask=s["mask"], relative=s["relative"], bias_table=s["table"], q_start=s["start"])
    if not s["case"]["train"]:
        return {"o": o}
    dq, dk, dv, dt = torch.autograd.grad(o, [s["q"], s["k"], s["v"], s["table"]], s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dt": dt}


# ---- plain forms
def _philox(seed, block):
    """Philox4x32-10: four 32-bit words for every 64-bit counter in `block` (as int64) under the 64-bit key `seed`."""
    lo = 0xFFFFFFFF
    c0, c1, c2, c3 = block & lo, (block >> 32) & lo, torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & lo, (seed >> 32) & lo
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & lo) ^ c1 ^ k0, p1 & lo, ((p0 >> 32) & lo) ^ c3 ^ k1, p0 & lo
        k0, k1 = (k0 + 0x9E3779B9) & lo, (k1 + 0xBB67AE85) & lo
    return torch.stack([c0, c1, c2, c3], -1)


def _rows_view(x):
    """The elements of `x` in the order the generator counts them: channels innermost for a map."""
    return x.permute(0, 2, 3, 1) if x.dim() == 4 else x


def _plain_dropout(s):
    x, p = _rows_view(s["x"].detach()), s["case"]["p"]
    n = x.numel()
    words = _philox(s["rng"][0], s["rng"][1] + torch.arange((n + 3) // 4, device="cuda")).reshape(-1)[:n]
    m = torch.where(words >= round(p * 2 ** 32), 1 / (1 - p), 0.0).to(torch.float32).reshape(x.shape)
    y = x.float() * m
    if s["residual"] is not None:
        y = y + _rows_view(s["residual"].detach()).float()
    dx = _rows_view(s["dy"]).float() * m
    back = (lambda v: v.permute(0, 3, 1, 2)) if s["x"].dim() == 4 else (lambda v: v)
    return {"y": back(y.to(s["t"])), "dx": back(dx.to(s["t"]))}


def _turn(n, cos, sin):
    h = cos.shape[-1]
    a, b = n[..., :h], n[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, n[..., 2 * h:]], -1)


def _plain_norm_turn(x, w, cos, sin):
    x = x.detach().float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return _turn(x * r * w.detach(), cos, sin)


def _plain_norm_turn_grad(x, w, cos, sin, dy):
    x = x.detach().float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    n = x * r
    dn = _turn(dy.float(), cos, -sin)
    g = dn * w.detach()
    return r * (g - n * (g * n).mean(-1, keepdim=True)), (dn * n).sum((0, 1, 2))


def _plain_qknorm(s):
    cos, sin = (s["cos"], s["sin"]) if s["pos"] is None else (s["cos"][s["pos"]], s["sin"][s["pos"]])
    cos, sin = cos[..., None, :], sin[..., None, :]
    out = {"q": _plain_norm_turn(s["q"], s["wq"], cos, sin).to(s["t"]), "k": _plain_norm_turn(s["k"], s["wk"], cos, sin).to(s["t"])}
    if s["case"]["train"]:
        dq, out["dwq"] = _plain_norm_turn_grad(s["q"], s["wq"], cos, sin, s["dq"])
        dk, out["dwk"] = _plain_norm_turn_grad(s["k"], s["wk"], cos, sin, s["dk"])
        out["dq"], out["dk"] = dq.to(s["t"]), dk.to(s["t"])
    return out


def _pair_buckets(s):
    """Bucket of every (query, key) pair."""
    c, n1 = s["case"], max(s["case"]["h"], s["case"]["w"]) - 1
    q = s["start"] + torch.arange(c["lq"], device="cuda")
    k = torch.arange(c["h"] * c["w"], device="cuda")
    bx = s["bucket"][(k % c["w"])[None, :] - (q % c["w"])[:, None] + n1]
    if c["h"] == 1:
        return bx
    return s["bucket"][(k // c["w"])[None, :] - (q // c["w"])[:, None] + n1] * s["per"] + bx


def _strip(ds, case):
    """[heads, lq, n] -> the same values with every map row widened to 2 w - 1 tokens, so that a pair's offset is the difference of two
    token numbers in a map as in a sequence."""
    h, w = case["h"], case["w"]
    if h == 1:
        return ds
    pad = torch.nn.functional.pad(ds.reshape(-1, h, w, h, w), (0, w - 1, 0, 0, 0, w - 1))
    return pad.reshape(ds.shape[0], h * (2 * w - 1), h * (2 * w - 1))


def _plain_attention(s):
    c = s["case"]
    b, heads, kv, d, lq, n = c["b"], c["heads"], c["kv"], c["d"], c["lq"], c["h"] * c["w"]
    g = heads // kv
    scale = d ** -0.5
    q = s["q"].detach().float().permute(0, 2, 1, 3).reshape(b, kv, g * lq, d)
    k = s["k"].detach().float().permute(0, 2, 1, 3).contiguous()
    v = s["v"].detach().float().permute(0, 2, 1, 3).contiguous()
    bucket = _pair_buckets(s)
    bias = s["table"].detach().t().contiguous()[:, bucket]
    a = ((q * scale) @ k.transpose(-1, -2)).reshape(b, heads, lq, n).add_(bias)
    if s["mask"] is not None:
        a = torch.where(s["mask"][:, None, None, :], a, -math.inf)
    top = a.amax(-1, keepdim=True)
    a = (a - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = a.sum(-1, keepdim=True)
    a = (a / torch.where(total == 0, 1.0, total)).reshape(b, kv, g * lq, n)
    o = a @ v
    out = {"o": o.reshape(b, heads, lq, d).permute(0, 2, 1, 3).to(s["t"]).contiguous()}
    if not c["train"]:
        return out
    do = s["do"].float().permute(0, 2, 1, 3).reshape(b, kv, g * lq, d)
    dv = a.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds = a * (ds - (do * o).sum(-1, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q) * scale
    strip = _strip(ds.reshape(b, heads, lq, n).sum(0), c)
    m = strip.shape[1]
    # row i shifted by m - 1 - i: the columns are the offsets
    diag = torch.nn.functional.pad(strip.flip(1), (0, m)).reshape(heads, -1)[:, :m * (2 * m - 1)].reshape(heads, m, 2 * m - 1).sum(1)
    of = s["bucket"]
    if c["h"] > 1:
        y, x = (torch.arange(2 * n1 - 1, device="cuda") - (n1 - 1) + max(c["h"], c["w"]) - 1 for n1 in (c["h"], c["w"]))
        of = (of[y][:, None] * s["per"] + of[x][None, :]).reshape(-1)
        off = torch.arange(2 * m - 1, device="cuda") - (m - 1) + (c["h"] - 1) * (2 * c["w"] - 1) + c["w"] - 1
        inside = (off >= 0) & (off < of.numel())
        of, diag = of[off[inside]], diag[:, inside]
    dt = torch.zeros_like(s["table"]).index_add_(0, of, diag.t().contiguous())
    back = lambda x, h: x.reshape(b, h, -1, d).permute(0, 2, 1, 3).to(s["t"]).contiguous()  # noqa: E731
    return out | {"dq": back(dq, heads), "dk": back(dk, kv), "dv": back(dv, kv), "dt": dt}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        x, dy = (_rows_view(s[k].detach()).double().cpu().numpy() for k in ("x", "dy"))
        key, first = (np.uint64(v & 0xFFFFFFFFFFFFFFFF) for v in s["rng"].tolist())
        n, low, sh = x.size, np.uint64(0xFFFFFFFF), np.uint64(32)
        ctr = first + np.arange((n + 3) // 4, dtype=np.uint64)
        w = [ctr & low, ctr >> sh, np.zeros_like(ctr), np.zeros_like(ctr)]
        ks = [int(key & low), int(key >> sh)]
        for i in range(10):
            a, b = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
            r = [np.uint64((ks[0] + i * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((ks[1] + i * 0xBB67AE85) & 0xFFFFFFFF)]
            w = [(b >> sh) ^ w[1] ^ r[0], b & low, (a >> sh) ^ w[3] ^ r[1], a & low]
        kept = (np.stack(w, 1).reshape(-1)[:n].astype(np.float64) >= np.rint(case["p"] * 2.0 ** 32)).reshape(x.shape)
        y, dx = (np.where(kept, v / (1.0 - case["p"]), 0.0) for v in (x, dy))
        if s["residual"] is not None:
            y = y + _rows_view(s["residual"].detach()).double().cpu().numpy()
        back = (lambda v: torch.from_numpy(v).permute(0, 3, 1, 2)) if s["x"].dim() == 4 else torch.from_numpy
        return {"y": back(y), "dx": back(dx)}
    if case["op"] == "qknorm":
        rows = torch.arange(case["h"] * case["w"], device="cuda")[None].expand(case["b"], -1) if s["pos"] is None else s["pos"]
        z = torch.complex(s["cos"].double(), s["sin"].double())[rows][:, :, None]
        half, out = case["rot"] // 2, {}
        for name, wname in (("q", "wq"), ("k", "wk")):
            x, w = s[name].detach().double(), s[wname].detach().double()
            norm = (x.square().sum(-1, keepdim=True) / case["d"] + 1e-6).sqrt()
            y = x / norm * w
            turned = torch.complex(y[..., :half], y[..., half:2 * half]) * z
            out[name] = torch.cat([turned.real, turned.imag, y[..., 2 * half:]], -1)
            if case["train"]:
                dy = s["d" + name].double()
                back = torch.complex(dy[..., :half], dy[..., half:2 * half]) * z.conj()
                dn = torch.cat([back.real, back.imag, dy[..., 2 * half:]], -1)
                out["dw" + name] = torch.einsum("blhd,blhd->d", dn, x / norm)
                along = (dn * w * x).sum(-1, keepdim=True)
                out["d" + name] = dn * w / norm - x * along / (case["d"] * norm ** 3)
        return out
    b, heads, kv, d, lq, h, w = (case[k] for k in ("b", "heads", "kv", "d", "lq", "h", "w"))
    n, g = h * w, heads // kv
    if b * heads * lq * n * d > 2 * 16 * 4097 * 4097 * 128 * 1.01:
        return None
    token = torch.arange(n, device="cuda")
    py, px = token // w, token % w
    far = max(h, w) - 1
    q, k, v, table = (s[m].detach().double() for m in ("q", "k", "v", "table"))
    outs = {m: torch.zeros(x.shape, dtype=torch.float64, device="cuda") for m, x in (("o", q), ("dq", q), ("dk", k), ("dv", v), ("dt", table))}
    lens = _lengths(case)
    for head in range(heads):
        shared = head // g
        diag = torch.zeros((2 * h - 1, 2 * w - 1), dtype=torch.float64, device="cuda")
        for i in range(b):
            m = lens[i]
            if m == 0:
                continue
            kk, vv = k[i, :m, shared], v[i, :m, shared]
            for at in range(0, lq, 2048):
                row = token[s["start"] + at:s["start"] + min(lq, at + 2048)]
                qq = q[i, at:at + 2048, head]
                bucket = s["bucket"][px[None, :m] - px[row][:, None] + far]
                if h > 1:
                    bucket = bucket + s["per"] * s["bucket"][py[None, :m] - py[row][:, None] + far]
                p = torch.softmax(qq @ kk.T / math.sqrt(d) + table[:, head][bucket], -1)
                outs["o"][i, at:at + 2048, head] = p @ vv
                if not case["train"]:
                    continue
                do = s["do"][i, at:at + 2048, head].double()
                dp = do @ vv.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                outs["dv"][i, :m, shared] += p.T @ do
                outs["dq"][i, at:at + 2048, head] = ds @ kk / math.sqrt(d)
                outs["dk"][i, :m, shared] += ds.T @ qq / math.sqrt(d)
                if h == 1:
                    shifted = torch.zeros((len(row), len(row) + n), dtype=torch.float64, device="cuda")
                    shifted[:, :m] = ds
                    # read with a pitch one shorter: row r moves r columns to the right, against its query's offset after the flip
                    flipped = shifted.flip(0).reshape(-1)[:len(row) * (len(row) + n - 1)].reshape(len(row), -1).sum(0)
                    first = -(int(row[-1])) + n - 1
                    diag[0, first:first + n + len(row) - 1] += flipped
                else:
                    for y in range(int(py[row[0]]), int(py[row[-1]]) + 1):
                        part = ds[(py[row] == y)]
                        xs = px[row][py[row] == y]
                        full = torch.zeros((len(xs), n), dtype=torch.float64, device="cuda")
                        full[:, :m] = part
                        wide = torch.zeros((len(xs), h, 2 * w - 1), dtype=torch.float64, device="cuda")
                        to = (torch.arange(w, device="cuda")[None, :] - xs[:, None] + w - 1)[:, None, :].expand(-1, h, -1)
                        wide.scatter_(2, to, full.reshape(len(xs), h, w))
                        diag[h - 1 - y:2 * h - 1 - y] += wide.sum(0)
        if case["train"]:
            oy, ox = (torch.arange(2 * m - 1, device="cuda") - (m - 1) + far for m in (h, w))
            flat = s["bucket"][ox][None, :].expand(2 * h - 1, -1) + (s["per"] * s["bucket"][oy][:, None] if h > 1 else 0)
            outs["dt"][:, head] = torch.zeros(table.shape[0], dtype=torch.float64, device="cuda").index_add_(0, flat.reshape(-1), diag.reshape(-1))
    return outs if case["train"] else {"o": outs["o"]}
