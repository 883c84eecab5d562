"""Autograd operators over tokens - what an attention layer with heads and positions is made of, beside the SAGAN core of ops.py:

  dropout             mask from a counter-based generator, never stored              (csrc/dropout.hip)
  qk_norm_rotary      per-head RMS norm of queries and keys + position rotation       (csrc/qkrope.hip)
  attention           softmax attention with heads shared by groups, a key mask and a learned relative position bias by buckets
                      (csrc/mha_fwd.hip, csrc/mha_bwd.hip)

Same contract as ops.py: torch supplies device memory, the current stream and the autograd tape; the arithmetic is in
libshineon_hip.so, there is no CPU fallback, everything may be captured into a hipGraph.  Two differences: operands may be float32 or
bfloat16 (sums and statistics are fp32 either way; with bfloat16 the backward pass of attention rounds probabilities and score gradients
to that type before it multiplies them with operands), and every call runs on the device of its operands, on that device's current
stream, whatever the current device is.  Gradients are first order: differentiating them again is refused."""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from .ops import _require_cuda

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _dtype(t, *others):
    """Type code of the operands; refuses CPU tensors, other types, mixed types and mixed devices."""
    _require_cuda(t)
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"float32 or bfloat16 only (got {t.dtype})")
    for o in others:
        if o.dtype != t.dtype:
            raise TypeError(f"operands of one type only (got {t.dtype} and {o.dtype})")
        if o.device != t.device:
            _require_cuda(o)
            raise ValueError(f"operands on one device only (got {t.device} and {o.device})")
    return code


def _fp32_param(t, shape, device, what):
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: float32 only (got {t.dtype})")
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what}: expected on {device}, got {t.device}")


def _launch(device, fn, what, *args):
    """fn(*args, stream) on `device`'s current stream; launches go to the current device, so that is switched when it is another."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)      # the handle alone: no Stream object (2 us, 5 - 10 in autograd's thread)
    if device.index == torch.cuda.current_device():
        err = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            err = fn(*args, stream)
    if err:
        check(err, what)


def _first_order(backward):
    """once_differentiable, at no cost where no graph of the gradients is asked for."""
    checked = once_differentiable(backward)
    return lambda ctx, *grads: (checked if torch.is_grad_enabled() else backward)(ctx, *grads)


def _places(*tensors):
    """Where operands lie, to tell in the backward pass whether the tape hands back what the forward pass's descriptor describes: saved
    tensors may come back elsewhere or with other strides (hooks, checkpoints)."""
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
def rng_state(seed, device, offset=0):
    """State of the counter-based generator: int64 {seed, offset} on the device."""
    return torch.tensor([_int64(seed), _int64(offset)], dtype=torch.int64, device=device)


def _int64(v):
    v = int(v) & 0xFFFFFFFFFFFFFFFF
    return v - (1 << 64) if v >> 63 else v


def _check_rng(rng, device):
    if rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous() or rng.device != device:
        raise ValueError(f"the generator's state is two contiguous int64 values on {device} (rng_state)")


def rng_draw(state, numel):
    """{seed, offset} for one dropout over `numel` elements; the state moves on past the counters it uses (one per four elements).
    Runs on the device, so a captured graph draws anew at every replay."""
    _require_cuda(state)
    _check_rng(state, state.device)
    out = torch.empty_like(state)
    _launch(state.device, lib().so_rng_draw, "rng_draw", state.data_ptr(), out.data_ptr(), (int(numel) + 3) // 4)
    return out


def _pitch_rows(t):
    """(rows, C, pitch) of a tensor whose elements lie in counting order - channels innermost for a 4-D map - with at most a constant
    gap behind each row; None when they do not."""
    if t.dim() == 4:
        t = t.permute(0, 2, 3, 1)
    if t.is_contiguous():
        return 1, t.numel(), t.numel()
    c = t.shape[-1]
    if t.dim() < 2 or (c > 1 and t.stride(-1) != 1):
        return None
    dims = [(s, st) for s, st in zip(t.shape[:-1], t.stride()[:-1]) if s > 1]
    if not dims or dims[-1][1] < c or any(a[1] != b[0] * b[1] for a, b in zip(dims[:-1], dims[1:])):
        return None
    return t.numel() // c, c, dims[-1][1]


def _like_rows(x):
    """An empty dense tensor of x's shape, elements in counting order."""
    if x.dim() == 4:
        n, c, h, w = x.shape
        return torch.empty((n, h, w, c), dtype=x.dtype, device=x.device).permute(0, 3, 1, 2)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _in_order(t):
    rows = _pitch_rows(t)
    if rows is None:
        t = _like_rows(t).copy_(t)
        rows = _pitch_rows(t)
    return t, rows


def _dense_in_order(t):
    return t.is_contiguous(memory_format=torch.channels_last) if t.dim() == 4 else t.is_contiguous()


def _dropout_launch(dt, x, p, rng, residual):
    n = x.numel()
    rows, c, ldx, ldr = 1, n, n, n
    if _dense_in_order(x) and (residual is None or _dense_in_order(residual)):
        y = torch.empty_like(x)
    else:
        y = _like_rows(x)
        x, (rows, c, ldx) = _in_order(x)
        if residual is not None:
            residual, (rr, rc, ldr) = _in_order(residual)
            if rr != rows:      # one of the two is dense (one row of all elements), the other has a pitch: both as rows
                if rows == 1:
                    rows, c, ldx = rr, rc, rc
                else:
                    ldr = c
    if n:
        _launch(x.device, lib().so_dropout, "dropout", dt, x.data_ptr(), ldx, None if residual is None else residual.data_ptr(), ldr,
                y.data_ptr(), c, rows, c, rng.data_ptr(), round(p * 4294967296.0), 1.0 / (1.0 - p) if p < 1.0 else 0.0)
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, dt):
        ctx.cfg = (p, dt)
        ctx.save_for_backward(rng)
        return _dropout_launch(dt, x, p, rng, residual)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        p, dt = ctx.cfg
        need_x, need_r = ctx.needs_input_grad[:2]
        return _dropout_launch(dt, dy, p, rng, None) if need_x else None, dy if need_r else None, None, None, None


def dropout(x, p, rng, residual=None):
    """residual + x * keep / (1 - p).  keep of element e (row-major; channels innermost for a 4-D map) is word e % 4 of Philox4x32-10
    with key rng[0] at counter rng[1] + e / 4, compared with p; the mask is recomputed in the backward pass.  `rng`: one draw
    (rng_draw), which must not be written to before the backward pass has run.  A dropped element counts as 0 whatever it holds;
    p = 1 drops everything."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability outside [0, 1]: {p}")
    dt = _dtype(x) if residual is None else _dtype(x, residual)
    _check_rng(rng, x.device)
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual of shape {tuple(residual.shape)} for x of shape {tuple(x.shape)}")
    return _DropoutFn.apply(x, residual, p, rng, dt)


# ------------------------------------------------------------------------------------------------
# query / key norm + rotation
# ------------------------------------------------------------------------------------------------
def rotary_table(shape, rot_dim, base=10000.0, device="cuda"):
    """(cos, sin), float32 [tokens, rot_dim / 2], angles computed in double.  shape: a length, or (H, W) for the tokens of a map in row
    order - the first rot_dim // 4 pairs then turn with the row, the others with the column."""
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even (got {rot_dim})")
    half = rot_dim // 2

    def axis(n, pairs):
        f = base ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
        return torch.arange(n, dtype=torch.float64)[:, None] * f

    if isinstance(shape, int):
        angle = axis(shape, half)
    else:
        h, w = shape
        ny = rot_dim // 4
        y, x = axis(h, ny), axis(w, half - ny)
        angle = torch.cat([y[:, None].expand(h, w, ny), x[None].expand(h, w, half - ny)], -1).reshape(h * w, half)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _heads(t, what):
    """[B, L, H, D] with contiguous channels (copied otherwise)."""
    if t.dim() != 4:
        raise ValueError(f"{what}: expected [B, L, H, D], got {tuple(t.shape)}")
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


class _QkDesc(ctypes.Structure):
    """so_qk_desc of include/shineon_hip.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "wq", "wk", "cosv", "sinv", "pos")]
                + [(n, ctypes.c_longlong) for n in ("sqb", "sql", "sqh", "skb", "skl", "skh", "P", "pos_sb", "pos_sl", "start")]
                + [(n, ctypes.c_int) for n in ("dtype", "Hq", "Hk", "pos64", "B", "L", "D", "R")] + [("eps", ctypes.c_float)])


def _qk_desc(q, k, wq, wk, cos, sin, positions, start, eps, dt):
    (b, n, hq, d), pp, p64, psb, psl = q.shape, None, 0, 0, 0
    if positions is not None:
        pp, p64, psl = positions.data_ptr(), int(positions.dtype == torch.int64), positions.stride(-1)
        psb = positions.stride(0) if positions.dim() == 2 else 0
    return _QkDesc(q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), pp, *q.stride()[:3],
                   *k.stride()[:3], cos.shape[0], psb, psl, start, dt, hq, k.shape[2], p64, b, n, d, 2 * cos.shape[1], eps)


class _QkNormRotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, start, eps, dt):
        q, k = _heads(q, "q"), _heads(k, "k")
        b, n, hq, d = q.shape
        yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        yk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        ctx.places = _places(q, k, wq, wk, cos, sin, positions)
        ctx.desc = _qk_desc(q, k, wq, wk, cos, sin, positions, start, eps, dt)
        if b and n:
            _launch(q.device, lib().so_qk_norm_rotary_fwd, "qk_norm_rotary_fwd", ctypes.addressof(ctx.desc), yq.data_ptr(), yk.data_ptr())
        return yq, yk

    @staticmethod
    @_first_order
    def backward(ctx, dyq, dyk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        x = ctx.desc
        if ctx.places != _places(q, k, wq, wk, cos, sin, positions):
            q, k = _heads(q, "q"), _heads(k, "k")
            wq, wk, cos, sin = (t.contiguous() for t in (wq, wk, cos, sin))
            x = _qk_desc(q, k, wq, wk, cos, sin, positions, x.start, x.eps, x.dtype)
        dyq, dyk = dyq.contiguous(), dyk.contiguous()
        dq, dk = torch.empty_like(dyq), torch.empty_like(dyk)
        if not (x.B and x.L):
            return dq, dk, torch.zeros_like(wq), torch.zeros_like(wk), None, None, None, None, None, None
        d, L = x.D, lib()
        n = L.so_qk_norm_rotary_ws_floats(d)
        dw, ws = (torch.empty(m, dtype=torch.float32, device=q.device) for m in ((2, d), n))      # dwq and dwk; scratch
        at = dw.data_ptr()
        _launch(q.device, L.so_qk_norm_rotary_bwd, "qk_norm_rotary_bwd", ctypes.addressof(x), dyq.data_ptr(), dyk.data_ptr(),
                dq.data_ptr(), dk.data_ptr(), at, at + 4 * d, ws.data_ptr(), n)
        return dq, dk, dw[0], dw[1], None, None, None, None, None, None


def qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions=None, start=0, eps=1e-6):
    """RMS norm over the channels of every head of q [B, L, Hq, D] and k [B, L, Hk, D] (weights [D], float32), then the rotation of
    channel pairs (i, i + R/2) by the token's row of cos / sin [P, R/2] (rotary_table); channels R .. D - 1 are not rotated.
    positions: int32 / int64, [L] or [B, L]; without it token l has position start + l.  q and k may be slices of one projection.  D
    even, at most 128.  A position outside the table makes that token's outputs NaN (its position is only known on the device).
    Returns dense (q', k')."""
    dt = _dtype(q, k)
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q [B, L, Hq, D] and k [B, L, Hk, D] expected, got {tuple(q.shape)} and {tuple(k.shape)}")
    b, n, _, d = q.shape
    if d < 2 or d % 2 or d > 128 or q.shape[2] < 1 or k.shape[2] < 1:
        raise ValueError(f"head size must be even and at most 128, at least one head each (got {tuple(q.shape)}, {tuple(k.shape)})")
    if cos.dim() != 2 or 2 * cos.shape[1] > d:
        raise ValueError(f"cos / sin of shape [P, R/2] with R <= {d} expected, got {tuple(cos.shape)}")
    _fp32_param(cos, cos.shape, q.device, "cos")
    _fp32_param(sin, cos.shape, q.device, "sin")
    if positions is None:
        if start < 0 or start + n > cos.shape[0]:
            raise ValueError(f"positions {start} .. {start + n - 1} outside a table of {cos.shape[0]} rows")
    else:
        if start:
            raise ValueError("positions and start exclude each other")
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
            raise TypeError(f"positions: int32 or int64 on {q.device}")
        if tuple(positions.shape) not in ((n,), (b, n)):
            raise ValueError(f"positions of shape ({n},) or ({b}, {n}) expected, got {tuple(positions.shape)}")
    _fp32_param(q_weight, (d,), q.device, "q_weight")
    _fp32_param(k_weight, (d,), q.device, "k_weight")
    return _QkNormRotaryFn.apply(q, k, q_weight.contiguous(), k_weight.contiguous(), cos.contiguous(), sin.contiguous(), positions,
                                 int(start), float(eps), dt)


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
class _Desc(ctypes.Structure):
    """so_mha_desc of include/shineon_hip.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "o_f32", "stats", "bias", "code", "words", "part_o", "part_ml", "dout",
                                                "dq", "dk", "dv", "delta", "strips")]
                + [(n, ctypes.c_longlong) for n in ("sqb", "sql", "sqh", "skb", "skl", "skh", "svb", "svl", "svh")]
                + [(n, ctypes.c_int) for n in ("dtype", "B", "Hq", "Hk", "Lq", "Lk", "D", "V", "code_max", "tokens", "q_start", "linear",
                                               "nwords", "width")]
                + [("scale", ctypes.c_float)])


def bucket_bounds(num_buckets, max_distance):
    """Distances at which the buckets of one direction start: one bucket per distance below half of `num_buckets`, then logarithmically
    spaced ones up to `max_distance`.  Step t of the m logarithmic ones starts at the first whole distance d with
    d >= exact (max_distance / exact)^(t / m), decided in whole numbers."""
    exact = num_buckets // 2
    m = num_buckets - exact
    bounds, d = list(range(1, exact + 1)), exact
    for t in range(1, m):
        while d ** m * exact ** t < exact ** m * max_distance ** t:
            d += 1
        bounds.append(d)
    return bounds


class RelativePositions:
    """Which pairs of tokens share an entry of a learned bias table.

    shape: a length, or (H, W) for the tokens of a map in row order.  Along one axis the signed distance key - query falls into one of
    `num_buckets` buckets: with `bidirectional` half of them for keys behind the query and half for keys in front (key > query), else
    all of them for keys at or before the query, keys after it counting as distance 0.  A map has num_buckets^2 buckets, row bucket *
    num_buckets + column bucket.  `rows` is the number of table entries per head.  Built once per shape; immutable."""

    def __init__(self, shape, num_buckets=32, max_distance=128, bidirectional=True, device="cuda"):
        h, w = (1, int(shape)) if isinstance(shape, int) else (int(shape[0]), int(shape[1]))
        if h < 1 or w < 1:
            raise ValueError(f"empty shape {shape}")
        half = num_buckets // 2 if bidirectional else num_buckets
        if half < 2 or (bidirectional and num_buckets % 2):
            raise ValueError(f"at least 2 buckets per direction, an even number for both directions (got {num_buckets})")
        if max_distance <= half // 2:
            raise ValueError(f"max_distance must exceed the {half // 2} distances that have buckets of their own (got {max_distance})")
        if h > 1 and w > 512:
            raise ValueError(f"map rows of at most 512 tokens (got {w})")
        self.shape, self.tokens, self.width = (h, w), h * w, w
        self.num_buckets, self.max_distance, self.bidirectional = num_buckets, max_distance, bidirectional
        self.linear = int(h == 1 or w == 1)      # code[t] = t
        self.code_max = (h - 1) * (2 * w - 1) + w - 1
        if 2 * self.code_max + 1 > 1 << 28:
            raise ValueError(f"shape {shape} has too many offsets")
        bounds = torch.tensor(bucket_bounds(half, max_distance), dtype=torch.int64)

        def axis(n):
            d = torch.arange(-(n - 1), n)
            if bidirectional:
                return torch.bucketize(d.abs(), bounds, right=True) + half * (d > 0)
            return torch.bucketize((-d).clamp(min=0), bounds, right=True)

        lut = axis(w) if h == 1 else (axis(h)[:, None] * num_buckets + axis(w)[None, :]).reshape(-1)
        self.rows = num_buckets if h == 1 else num_buckets * num_buckets
        token = torch.arange(self.tokens)
        code = token if h == 1 else (token // w) * (2 * w - 1) + token % w
        pad = (self.tokens + 127) // 128 * 128 + 128 - self.tokens
        code = torch.cat([code, code[-1:].expand(pad)])
        order = torch.argsort(lut, stable=True)
        start = torch.searchsorted(lut[order].contiguous(), torch.arange(self.rows + 1))
        self.device = torch.empty(0, device=device).device
        # a map's offset is (dy) (2 W - 1) + dx: every value of the range is one (dy, dx), so the lookup is dense
        self.lut, self.code, self.order, self.start = (t.to(torch.int32).to(self.device) for t in (lut, code, order, start))


def _rows16(t, what):
    """[B, L, H, D] as the kernels read it: channels contiguous, everything else a multiple of 16 bytes, rows less than 2^22 elements apart
    (128 rows within a 31-bit offset) - zero channels appended to D and a dense copy made where it is not."""
    t = _heads(t, what)
    e = 16 // t.element_size()
    d = t.shape[3]
    if d % e:
        t = torch.nn.functional.pad(t, (0, e - d % e))
    sb, sl, sh, _ = t.stride()
    if (t.data_ptr() % 16 or (sl >= 1 << 22 and t.shape[1] > 1)
            or (sb % e or sl % e or sh % e) and any(s % e for s, n in zip((sb, sl, sh), t.shape) if n > 1)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(t):
    """Strides of the first three axes; an axis of one entry counts as stride 0."""
    (b, n, h, _), (sb, sl, sh, _) = t.shape, t.stride()
    return sb if b > 1 else 0, sl if n > 1 else 0, sh if h > 1 else 0


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, mask, rel, q_start, scale, train, dt):
        d_true = q.shape[3]
        q, k, v = _rows16(q, "q"), _rows16(k, "k"), _rows16(v, "v")
        b, lq, hq, d = q.shape
        lk, hk = k.shape[1], k.shape[2]
        dev, L = q.device, lib()
        o = torch.empty((b, lq, hq, d), dtype=q.dtype, device=dev)
        ctx.d_true, ctx.rel, ctx.desc = d_true, rel, None
        if not (b and lq and lk):
            if train:
                ctx.save_for_backward(q, k, v, table)
            return o.zero_()[..., :d_true]
        x = _Desc(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr())
        (x.sqb, x.sql, x.sqh), (x.skb, x.skl, x.skh), (x.svb, x.svl, x.svh) = _strides(q), _strides(k), _strides(v)
        x.dtype, x.B, x.Hq, x.Hk, x.Lq, x.Lk, x.D, x.nwords, x.scale = dt, b, hq, hk, lq, lk, d, (lk + 63) // 64, scale
        words = bias = stats = o_f32 = None
        mp = msb = tp = lp = None
        if mask is not None:
            words = torch.empty((b, x.nwords), dtype=torch.int64, device=dev)
            x.words, mp, msb = words.data_ptr(), mask.data_ptr(), mask.stride(0)
        if table is not None:
            x.V, x.code_max, x.tokens, x.q_start, x.linear, x.width = (2 * rel.code_max + 1, rel.code_max, rel.tokens, q_start,
                                                                       rel.linear, rel.width)
            bias = torch.empty(hq * x.V + 256, dtype=torch.float32, device=dev)      # readable on both sides: 128 floats
            x.bias, x.code, tp, lp = bias.data_ptr() + 512, rel.code.data_ptr(), table.data_ptr(), rel.lut.data_ptr()
        if mp is not None or tp is not None:
            _launch(dev, L.so_mha_prep, "mha_prep", tp, lp, x.V, hq, scale, x.bias, mp, msb or 0, b, lk, x.words)
        if train:
            stats = torch.empty((2, b, hq, lq), dtype=torch.float32, device=dev)
            x.stats = stats.data_ptr()
            if dt == 1:
                o_f32 = torch.empty(o.shape, dtype=torch.float32, device=dev)
                x.o_f32 = o_f32.data_ptr()
        at = ctypes.addressof(x)
        parts = L.so_mha_parts(at)
        if parts < 0:
            check(parts, "mha_parts")
        if parts > 1:
            part = torch.empty(b * hq * lq * parts * (d + 2), dtype=torch.float32, device=dev)
            x.part_o = part.data_ptr()
            x.part_ml = x.part_o + 4 * b * hq * lq * parts * d
        _launch(dev, L.so_mha_fwd, "mha_fwd", at)
        if train:
            ctx.desc, ctx.places = x, _places(q, k, v)
            ctx.save_for_backward(q, k, v, table, o, o_f32, stats, bias, words)
        return o if d == d_true else o[..., :d_true].contiguous()

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        d_true, rel = ctx.d_true, ctx.rel
        if ctx.desc is None:
            q, k, v, table = ctx.saved_tensors
            return (*(torch.zeros_like(t[..., :d_true]) for t in (q, k, v)), None if table is None else torch.zeros_like(table),
                    None, None, None, None, None, None)
        q, k, v, table, o, o_f32, stats, bias, words = ctx.saved_tensors
        x = _Desc.from_buffer_copy(ctx.desc)      # a second backward pass of the same graph must not see this one's pointers
        if ctx.places != _places(q, k, v):
            q, k, v = _rows16(q, "q"), _rows16(k, "k"), _rows16(v, "v")
            x.q, x.k, x.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
            (x.sqb, x.sql, x.sqh), (x.skb, x.skl, x.skh), (x.svb, x.svl, x.svh) = _strides(q), _strides(k), _strides(v)
        o, o_f32, stats, bias, words = (None if t is None else t.contiguous() for t in (o, o_f32, stats, bias, words))
        x.o, x.stats = o.data_ptr(), stats.data_ptr()
        if o_f32 is not None:
            x.o_f32 = o_f32.data_ptr()
        if bias is not None:
            x.bias = bias.data_ptr() + 512
        if words is not None:
            x.words = words.data_ptr()
        b, lq, hq, d = q.shape
        dev, L = q.device, lib()
        if d != d_true:
            dout = torch.nn.functional.pad(dout, (0, d - d_true))
        dout = dout.contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        dq = torch.empty((b, lq, hq, d), dtype=q.dtype, device=dev)
        dk, dv = (torch.empty((b, x.Lk, x.Hk, d), dtype=q.dtype, device=dev) for _ in range(2))
        delta, dtable = torch.empty((b, hq, lq), dtype=torch.float32, device=dev), None
        x.dout, x.dq, x.dk, x.dv, x.delta = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr()
        at = ctypes.addressof(x)
        if table is not None and ctx.needs_input_grad[3]:
            n = L.so_mha_strip_floats(at)
            if n < 0:
                check(int(n), "mha_strip_floats")
            strips = torch.empty(n + hq * x.V, dtype=torch.float32, device=dev)      # strips | sums over offsets
            x.strips = strips.data_ptr()
            dtable = torch.empty((rel.rows, hq), dtype=torch.float32, device=dev)
        m = L.so_mha_bwd_floats(at)
        if m:
            if m < 0:
                check(int(m), "mha_bwd_floats")
            part = torch.empty(m, dtype=torch.float32, device=dev)
            x.part_o = part.data_ptr()
        _launch(dev, L.so_mha_bwd, "mha_bwd", at)
        if dtable is not None:
            _launch(dev, L.so_mha_dtable, "mha_dtable", at, rel.order.data_ptr(), rel.start.data_ptr(), rel.rows, x.strips + 4 * n,
                    dtable.data_ptr())
        if d != d_true:
            dq, dk, dv = (t[..., :d_true] for t in (dq, dk, dv))
        return dq, dk, dv, dtable, None, None, None, None, None, None


def attention(q, k, v, scale=None, key_mask=None, relative=None, bias_table=None, q_start=0):
    """softmax(scale q k^T + bias) v over the visible keys, per head.

    q [B, Lq, Hq, D]; k, v [B, Lk, Hk, D]; Hq a multiple of Hk (query heads h * Hq / Hk .. share key head h); float32 or bfloat16,
    D <= 128.  Any strides: operands whose rows do not start at multiples of 16 bytes, or whose channels are not contiguous, are copied
    first.  scale: default D^-1/2, positive.

    key_mask: bool [B, Lk], True = visible.  Hidden keys and values may hold anything (inf and NaN included) and get zero gradients; a
    sample without visible keys gives zeros.

    relative + bias_table: a RelativePositions plan and its learned table [plan.rows, Hq] (float32).  Key j against query i adds the
    entry of the bucket of token j against token q_start + i.  An entry may be -inf; finite ones beyond +-7.4e8 count as that.

    Training with a table takes scratch for the bias gradient while backward runs, per sample and head 4 bytes for every block of 128
    queries, part of the keys (1 to 8, more the fewer blocks there are) and offset that the block can meet: Lk + 127 of them in a sequence -
    Lq Lk / 32 bytes times the parts -, in a map 2 W - 1 for every map row of keys beside those of the queries, whose map rows are padded to
    multiples of 16 (so_mha_strip_floats; so_mha_bwd_floats says what the parts' sums of dq, dk and dv take besides).

    One or a few queries over long keys (a new token against what came before) are split over the keys.  Returns [B, Lq, Hq, D];
    differentiable in q, k, v and bias_table.  The order of all sums is fixed: the same inputs give the same bits, whatever wants a
    gradient.

    bfloat16: probabilities enter the product with v with all their bits, so the result is rounded once.  In the backward pass
    probabilities (for dv) and score gradients (for dq, dk) are rounded to bfloat16, half a step (2^-8 of a value) each, which adds about
    as much error to dq, dk and dv as their own rounding; the gradient of bias_table sums unrounded ones."""
    dt = _dtype(q, k, v)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q [B, Lq, Hq, D], k and v [B, Lk, Hk, D] expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"{hq} query heads cannot share {hk} key heads evenly")
    if d < 1 or d > 128:
        raise ValueError(f"head size 1 .. 128 (got {d})")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (1e-20 <= scale <= 1e20):      # the bias is kept divided by it, in fp32
        raise ValueError(f"scale must be positive, from 1e-20 to 1e20 (got {scale})")
    if key_mask is not None:
        if key_mask.dtype != torch.bool or tuple(key_mask.shape) != (b, lk) or key_mask.device != q.device:
            raise ValueError(f"key_mask: bool of shape ({b}, {lk}) on {q.device} expected, got {key_mask.dtype} {tuple(key_mask.shape)}")
        key_mask = key_mask if lk <= 1 or key_mask.stride(1) == 1 else key_mask.contiguous()
    if (relative is None) != (bias_table is None):
        raise ValueError("relative and bias_table belong together")
    if relative is not None:
        if relative.device != q.device:
            raise ValueError(f"the plan is on {relative.device}, q on {q.device}")
        if q_start < 0 or q_start + lq > relative.tokens or lk > relative.tokens:
            raise ValueError(f"queries {q_start} .. {q_start + lq - 1} and {lk} keys do not fit a plan of {relative.tokens} tokens")
        _fp32_param(bias_table, (relative.rows, hq), q.device, "bias_table")
        bias_table = bias_table.contiguous()
    elif q_start:
        raise ValueError("q_start without relative positions")
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, bias_table))
    return _AttentionFn.apply(q, k, v, bias_table, key_mask, relative, int(q_start), scale, train, dt)
