"""Token operators, host side: the generator's published vectors, bucket plans, rotation tables, refusals before any launch."""
import ctypes

import numpy as np
import pytest
import torch

import tokens_ref as ref
from shineon_virtual_tryon_amd import _lib, ops_tokens as tok


def test_oracle_generator_known_answers():
    """The published Philox4x32-10 vectors (zeros, ones, digits of pi)."""
    f = 0xFFFFFFFF
    cases = [([0] * 4, [0] * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"), ([f] * 4, [f] * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
             ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], "d16cfe09 94fdcceb 5001e420 24126ea1")]
    for ctr, key, want in cases:
        got = ref.philox4x32_full([np.array([c], np.uint64) for c in ctr], key)[0]
        assert " ".join("%08x" % int(w) for w in got) == want


@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("num,far", [(4, 3), (8, 20), (32, 128), (16, 32), (6, 100), (10, 7)])
@pytest.mark.parametrize("shape", [1, 2, 300, (3, 5), (1, 9), (9, 1), (20, 40)], ids=str)
def test_plan_buckets(shape, num, far, both):
    p = tok.RelativePositions(shape, num, far, both, device="cpu")
    n = p.tokens
    code = p.code[:n].long()
    got = p.lut.long()[code[None] - code[:, None] + p.code_max]
    assert torch.equal(got, ref.pair_buckets(shape, n, n, 0, num, far, both))
    assert (p.code[n:] == p.code[n - 1]).all() and len(p.code) >= (n + 127) // 128 * 128 + 128
    for r in range(p.rows):
        assert (p.lut[p.order[p.start[r]:p.start[r + 1]].long()] == r).all()
    assert int(p.start[-1]) == len(p.lut) == 2 * p.code_max + 1


def test_plan_refusals():
    for kw in (dict(shape=0), dict(shape=(3, 0)), dict(shape=5, num_buckets=3), dict(shape=5, num_buckets=2), dict(shape=5, num_buckets=32, max_distance=8),
               dict(shape=(2, 513)), dict(shape=1 << 29)):
        with pytest.raises(ValueError):
            tok.RelativePositions(device="cpu", **kw)
    with pytest.raises(ValueError):
        tok.rotary_table(4, 3, device="cpu")


def test_rotary_table_angles():
    cos, sin = tok.rotary_table(70000, 8, device="cpu")
    a = 69999 * 10000.0 ** (-2 / 8)
    assert abs(cos[69999, 1].item() - np.cos(a)) <= 2.0 ** -24 and abs(sin[69999, 1].item() - np.sin(a)) <= 2.0 ** -24
    cos, sin = tok.rotary_table((3, 4), 8, device="cpu")
    assert cos.shape == (12, 4)
    assert torch.equal(cos[4:8, :2], cos[4:5, :2].expand(4, 2)) and torch.equal(cos[1::4, 2:], cos[1:2, 2:].expand(3, 2))


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tok.dropout(x, 0.5, tok.rng_state(1, "cpu"))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tok.rng_draw(tok.rng_state(1, "cpu"), 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tok.qk_norm_rotary(x, x, torch.ones(8), torch.ones(8), *tok.rotary_table(2, 8, device="cpu"))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tok.attention(x, x, x)


def _desc(**kw):
    base = dict(q=256, k=256, v=256, o=256, dtype=0, B=1, Hq=4, Hk=2, Lq=8, Lk=8, D=64, nwords=1, scale=0.125, sqb=2048, sql=256, sqh=64, skb=1024,
                skl=128, skh=64, svb=1024, svl=128, svh=64)
    return tok._Desc(**{**base, **kw})


def test_c_entry_points_refuse_before_launching():
    """Wrong descriptors come back as error codes from the host side of the C ABI."""
    L = _lib.lib()
    assert L.so_mha_desc_bytes() == ctypes.sizeof(tok._Desc)
    assert L.so_mha_parts(ctypes.addressof(_desc())) >= 1
    shape, align = -2, -1
    for kw, want in ((dict(dtype=2), shape), (dict(Hq=3), shape), (dict(D=132), shape), (dict(D=0), shape), (dict(Lk=0), shape), (dict(scale=0.0), shape),
                     (dict(scale=float("nan")), shape), (dict(nwords=2), shape), (dict(D=62), align), (dict(sql=254), align), (dict(q=260), align),
                     (dict(dtype=1, D=60), align), (dict(bias=256, code=None, V=15, code_max=7, tokens=8), shape),
                     (dict(bias=256, code=256, V=15, code_max=7, tokens=8, q_start=1), shape), (dict(bias=256, code=256, V=14, code_max=7, tokens=8), shape),
                     (dict(q=None), shape)):
        assert L.so_mha_fwd(ctypes.addressof(_desc(**kw)), None) == want, kw
    assert L.so_mha_bwd(ctypes.addressof(_desc()), None) == shape          # no dout
    assert L.so_mha_strip_floats(ctypes.addressof(_desc())) == shape       # no bias
    assert L.so_mha_prep(None, None, 0, 0, 0.0, None, None, 0, 0, 0, None, None) == shape
    assert L.so_dropout(2, None, 4, None, 0, None, 4, 1, 4, None, 0, 1.0, None) == shape
    assert L.so_dropout(0, None, 3, None, 0, None, 4, 1, 4, None, 0, 1.0, None) == shape
    assert L.so_dropout(0, None, 4, None, 0, None, 4, 1, 4, None, 2 ** 32 + 1, 1.0, None) == shape
    assert L.so_dropout(0, None, 4, None, 0, None, 4, 0, 4, None, 0, 1.0, None) == 0
    assert L.so_rng_draw(None, None, 1, None) == shape
    assert L.so_qk_desc_bytes() == ctypes.sizeof(tok._QkDesc)

    def qk(**kw):
        base = dict(q=256, k=256, wq=256, wk=256, cosv=256, sinv=256, sqb=320, sql=64, sqh=64, skb=320, skl=64, skh=64, P=8, dtype=0, Hq=1, Hk=1, B=1,
                    L=5, D=64, R=64, eps=1e-6)
        return ctypes.addressof(keep.setdefault(str(kw), tok._QkDesc(**{**base, **kw})))

    keep = {}
    for kw, want in ((dict(P=4), shape), (dict(start=4), shape), (dict(start=-1), shape), (dict(D=63), shape), (dict(R=63), shape), (dict(R=66), shape),
                     (dict(D=130), shape), (dict(dtype=3), shape), (dict(Hk=0), shape), (dict(q=258), align)):
        assert L.so_qk_norm_rotary_fwd(qk(**kw), 256, 256, None) == want, kw
    assert L.so_qk_norm_rotary_bwd(qk(), 256, 256, 256, 256, 256, 256, 256, 10, None) == shape      # too little scratch


# ------------------------------------------------------------------------------------------------------------------- launches
PITCHED = {                     # name: (a slice of a wider tensor, whose pitch may exceed its number of elements)
    "two_rows": lambda: torch.zeros(2, 100)[:, :4], "projection": lambda: torch.zeros(1, 3, 24)[..., 8:16], "column": lambda: torch.zeros(5, 100)[:, 7:8],
    "map": lambda: torch.zeros(1, 40, 2, 1).contiguous(memory_format=torch.channels_last)[:, :6],
    "many_rows": lambda: torch.zeros(50, 24)[:, :8],
}


@pytest.mark.parametrize("which", ["x", "residual", "both"])
@pytest.mark.parametrize("name", sorted(PITCHED))
def test_dropout_launches_with_each_operands_own_pitch(monkeypatch, name, which):
    """Element (row, column) of every operand is at row * pitch + column, whatever the pitch and whichever operand is dense."""
    calls = []
    monkeypatch.setattr(tok, "_launch", lambda device, fn, what, *args: calls.append(args))
    part = PITCHED[name]()
    dense = tok._like_rows(part)
    x, residual = (part if which in ("x", "both") else dense), (part if which in ("residual", "both") else dense)
    assert tok._dropout_launch(0, x, 0.5, torch.zeros(2, dtype=torch.int64), residual).shape == part.shape
    ((_, xp, ldx, rp, ldr, _, ldy, rows, c, *_),) = calls
    assert (rows * c, ldy, xp, rp) == (part.numel(), c, x.data_ptr(), residual.data_ptr())
    for t, ld in ((x, ldx), (residual, ldr)):
        order = t.permute(0, 2, 3, 1) if t.dim() == 4 else t
        where = torch.arange(t.untyped_storage().size() // 4).as_strided(order.shape, order.stride(), t.storage_offset()).reshape(-1) - t.storage_offset()
        e = torch.arange(part.numel())
        assert torch.equal(e // c * ld + e % c, where)


# ------------------------------------------------------------------------------------------------------------------- modules
def test_attention_registry_and_options():
    from shineon_virtual_tryon_amd.networks.attention import ATTENTION_TYPES
    from shineon_virtual_tryon_amd.networks.attention.relative import RelativeAttention
    from shineon_virtual_tryon_amd.networks.attention.sagan import SelfAttention
    from shineon_virtual_tryon_amd.options import TrainOptions

    assert ATTENTION_TYPES["sagan"] is SelfAttention and ATTENTION_TYPES["relative"] is RelativeAttention
    base = ["--model", "tom", "--dataset", "synthetic", "--name", "t"]
    opt = TrainOptions().parse(base, interactive=False)
    assert opt.attn_type == "sagan" and not opt.use_dropout
    opt = TrainOptions().parse(base + ["--self_attn", "--attn_type", "relative", "--use_dropout"], interactive=False)
    assert opt.attn_type == "relative" and opt.use_dropout
    for channels, head in ((512, 64), (96, 48), (1336, 8), (10, 10), (2, 2)):
        m = RelativeAttention(channels)
        assert (m.head_dim, m.heads) == (head, channels // head)
    with pytest.raises(ValueError):
        RelativeAttention(7)


def test_unet_with_relative_attention_and_dropout():
    """The options add modules behind the existing ones: what is there without them keeps its names, and its values for a seed."""
    from shineon_virtual_tryon_amd.networks.attention.relative import RelativeAttention
    from shineon_virtual_tryon_amd.networks.cpvton.unet import UnetGenerator
    from shineon_virtual_tryon_amd.networks.layers import HipDropout

    def build(**kw):
        torch.manual_seed(3)
        return UnetGenerator(10, 4, 7, 2, ngf=8, norm_layer="instance", activation="gelu", **kw)

    plain, dropped = build(), build(use_dropout=True)
    drops = [m for m in dropped.modules() if isinstance(m, HipDropout)]
    assert len(drops) == 2 and all(m.p == 0.5 for m in drops) and not torch.equal(drops[0].rng_state, drops[1].rng_state)
    assert list(plain.state_dict()) == list(dropped.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(plain.state_dict().values(), dropped.state_dict().values()))
    again = [m for m in build(use_dropout=True).modules() if isinstance(m, HipDropout)]
    assert all(torch.equal(a.rng_state, b.rng_state) for a, b in zip(drops, again))
    net = build(use_self_attn=True, attn_type="relative")
    found = [n for n, m in net.named_modules() if isinstance(m, RelativeAttention)]
    sagan = build(use_self_attn=True)
    assert len(found) == 4 and set(found) < {n for n, _ in sagan.named_modules()}
    with pytest.raises(ValueError, match="attn_type"):
        build(use_self_attn=True, attn_type="none")
    with pytest.raises(ValueError):
        HipDropout(1.5)


def test_dropout_ranks_draw_different_masks(monkeypatch):
    """train.py builds the model before it joins the process group: the launcher's RANK stands for the rank then."""
    from shineon_virtual_tryon_amd.networks.layers import HipDropout

    states = []
    for rank in (None, "0", "1", "7"):
        monkeypatch.delenv("RANK", raising=False)
        if rank:
            monkeypatch.setenv("RANK", rank)
        torch.manual_seed(3)
        states.append([HipDropout(0.5, stream).rng_state.tolist() for stream in (0, 1)])
    assert states[0] == states[1]
    assert len({tuple(s) for pair in states[1:] for s in pair}) == 6


def test_dropout_modules_without_a_stream_draw_different_masks():
    """A module that is not given a stream takes one from torch's generator: others do not share its masks, the seed brings them back, and
    a module that drops nothing takes nothing."""
    from shineon_virtual_tryon_amd.networks.attention.relative import RelativeAttention
    from shineon_virtual_tryon_amd.networks.layers import HipDropout

    def build():
        torch.manual_seed(3)
        return [m.rng_state.tolist() for m in (HipDropout(0.5), HipDropout(0.5), RelativeAttention(32, dropout=0.1).dropout,
                                               RelativeAttention(32, dropout=0.1).dropout, HipDropout(0.5, 0), HipDropout(0.5, 1))]

    states = build()
    assert len({tuple(s) for s in states}) == 6 and build() == states
    torch.manual_seed(3)
    want = torch.rand(3)
    torch.manual_seed(3)
    HipDropout(0.0)
    HipDropout(0.5, 4)
    assert torch.equal(torch.rand(3), want)


def test_dropout_state_travels_between_ranks(monkeypatch):
    """A checkpoint holds rank 0's state; every rank goes on from it with its own masks."""
    from shineon_virtual_tryon_amd.networks.layers import HipDropout

    torch.manual_seed(3)
    mods = []
    for rank in ("0", "5"):
        monkeypatch.setenv("RANK", rank)
        mods.append(HipDropout(0.5, 2))
    assert mods[0].generator_state() == mods[0].rng_state.tolist() and mods[1].generator_state() == mods[0].generator_state()
    mods[0].rng_state[1] = 1234
    state, storage = mods[0].generator_state(), mods[1].rng_state.data_ptr()
    torch.manual_seed(99)
    fresh = [mods[1]]
    for rank in ("0", "5"):
        monkeypatch.setenv("RANK", rank)
        fresh.append(HipDropout(0.5, 3))
        fresh[-1].set_generator_state(state)
    seed = mods[1].rng_state[0].item()
    mods[1].set_generator_state(state)
    assert mods[1].rng_state.tolist() == [seed, 1234] == fresh[2].rng_state.tolist() and mods[1].rng_state.data_ptr() == storage
    assert fresh[1].rng_state.tolist() == state


@pytest.mark.parametrize("value,name", [(True, "sagan"), (1, "sagan"), ("sagan", "sagan"), ("relative", "relative"), (0, None), (None, None), (False, None)])
def test_unet_block_takes_any_truth_value_for_attention(value, name):
    from shineon_virtual_tryon_amd.networks.attention import ATTENTION_TYPES
    from shineon_virtual_tryon_amd.networks.cpvton.unet import UnetSkipConnectionBlock

    block = UnetSkipConnectionBlock(8, 8, innermost=True, self_attn=value)
    found = [type(m) for m in block.model if type(m) in ATTENTION_TYPES.values()]
    assert found == ([ATTENTION_TYPES[name]] * 2 if name else [])


def test_c_entry_points_refuse_null_pointers():
    """A missing descriptor or operand comes back as an error code; nothing is read and nothing is launched."""
    L, shape = _lib.lib(), -2
    for fn in (L.so_mha_parts, L.so_mha_strip_floats, L.so_mha_bwd_floats):
        assert fn(None) == shape
    assert L.so_mha_fwd(None, None) == L.so_mha_bwd(None, None) == shape
    assert L.so_mha_dtable(None, 256, 256, 1, 256, 256, None) == shape
    assert L.so_qk_norm_rotary_fwd(None, 256, 256, None) == shape
    assert L.so_qk_norm_rotary_bwd(None, 256, 256, 256, 256, 256, 256, 256, 1 << 20, None) == shape
    base = dict(q=256, k=256, wq=256, wk=256, cosv=256, sinv=256, sqb=320, sql=64, sqh=64, skb=320, skl=64, skh=64, P=8, dtype=0, Hq=1, Hk=1, B=1,
                L=5, D=64, R=64, eps=1e-6)
    for name in ("q", "k", "wq", "wk", "cosv", "sinv"):
        x = tok._QkDesc(**{**base, name: None})
        assert L.so_qk_norm_rotary_fwd(ctypes.addressof(x), 256, 256, None) == shape, name
    x = tok._QkDesc(**base)
    assert L.so_qk_norm_rotary_fwd(ctypes.addressof(x), None, 256, None) == L.so_qk_norm_rotary_fwd(ctypes.addressof(x), 256, None, None) == shape
    full = [256] * 7
    for i in range(7):
        a = [None if j == i else v for j, v in enumerate(full)]
        assert L.so_qk_norm_rotary_bwd(ctypes.addressof(x), *a, 1 << 20, None) == shape, i
    for a in ((None, 256, 256), (256, None, 256), (256, 256, None)):
        assert L.so_dropout(0, a[0], 4, None, 0, a[1], 4, 1, 4, a[2], 0, 1.0, None) == shape


def test_parts_of_the_keys_weigh_their_partial_sums():
    """Cut where blocks do not fill the chip, whole where the partial sums outgrow the caches and joining them takes what cutting gains."""
    def parts(dtype, b, n, hq, hk, d):
        return _lib.lib().so_mha_parts(ctypes.addressof(_desc(dtype=dtype, B=b, Hq=hq, Hk=hk, Lq=n, Lk=n, D=d, nwords=(n + 63) // 64)))

    assert parts(1, 2, 4097, 16, 4, 128) == 1                # 1032 blocks on 256 CUs, 67 MB a part
    assert parts(1, 4, 600, 16, 16, 128) == 1                # 304 blocks of 45 us
    assert parts(0, 2, 2049, 8, 8, 64) > 2                   # 260 blocks of 150 us: two rounds of them whole, 8 MB a part
    assert parts(1, 1, 1024, 1, 1, 64) > 2                   # 8 blocks
