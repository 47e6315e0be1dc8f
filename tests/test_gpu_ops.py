"""The step operators on the GPU against plain 64-bit forms: rotary positions,
attention with a sliding window and sinks, token sampling, and a run of them
together.

Tolerances count roundings.  ``half(dtype)`` is the largest relative error of
one rounding to the type; a result that is rounded once may be off by that
much of itself, plus what its 32-bit arithmetic adds (bounded at each test).
"""

import math

import numpy as np
import pytest
import torch

import stickykv_b200 as skv

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -24          # half a step of float32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):          # half the smallest subnormal
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, g):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def within(got, want, tol, what=""):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{((got.double() - want).abs() / tol).nan_to_num(math.inf).max().item():.3g} of the tolerance")


# -- rotary ---------------------------------------------------------------------------------

def rotary_ref(x, pos, inv, inter, scale, inverse):
    """The rotated tensor in 64 bits and the bound of its 32-bit error: cosine
    and sine are off by at most 4 ulp of 1 (the angle's rounding to 32 bits, pi
    * 2^-24, sincospi's 2 ulp and the factor's rounding: under 8 * 2^-24), the
    two products and their sum by 3 roundings."""
    r = 2 * inv.numel()
    a = pos.double().view(*pos.shape[:-1], -1, 1) * inv.double() * (-1 if inverse else 1)
    a = a.unsqueeze(-3) if a.dim() == 3 else a
    c, s = a.cos() * scale, a.sin() * scale
    y = x.double().clone()
    i = torch.arange(r, device=x.device)
    i0, i1 = (i[0::2], i[1::2]) if inter else (i[:r // 2], i[r // 2:])
    x0, x1 = y[..., i0].clone(), y[..., i1].clone()
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    e = torch.zeros_like(y)
    e[..., i0] = e[..., i1] = (x0.abs() + x1.abs()) * abs(scale) * 11 * U32
    return y, e


ROTARY = [  # B, T, Hq, Hkv, D, r, interleaved
    (1, 1, 1, 1, 2, 2, False), (1, 1, 32, 8, 64, 64, False), (4, 1, 32, 8, 64, 64, True), (2, 7, 3, 1, 128, 128, False),
    (3, 33, 14, 2, 96, 72, True), (3, 5, 4, 2, 96, 72, False), (1, 257, 2, 2, 80, 40, False), (2, 19, 5, 1, 80, 20, True),
    (2, 9, 3, 3, 50, 34, False), (2, 9, 3, 3, 50, 2, True), (1, 1000, 8, 8, 32, 32, False),
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B, T, Hq, Hkv, D, r, inter", ROTARY)
def test_rotary(B, T, Hq, Hkv, D, r, inter, dt):
    g = gen(B * T + D)
    q, k = (normal((B, T, h, D), DT[dt], g).transpose(1, 2) for h in (Hq, Hkv))
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, device="cuda")
    inv, _ = skv.rotary_frequencies(r, 500000.0, device="cuda")
    for inverse, scale in ((False, 1.0), (True, 1.25)):
        got = skv.apply_rotary(q, k, pos, inv, interleaved=inter, scale=scale, inverse=inverse)
        for x, y in zip((q, k), got):
            want, e = rotary_ref(x, pos, inv, inter, scale, inverse)
            assert y.shape == x.shape and y.stride() == x.stride()
            within(y, want, e * (1 + half(DT[dt])) + half(DT[dt]) * want.abs() + tiny(DT[dt]), f"{dt} {inverse}")
            assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("inter", [False, True])
def test_rotary_float32_counts_the_whole_angle(inter, inverse):
    """Each term of a result is off by what it is made of, small cosines and
    sines included: 2 * 2^-24 of sincospi (1 ulp), a rounding of the rest of the
    angle's share, of the product and of the sum, 6 in all with the result's
    own; the angle by four roundings of 64 bits and 2^-46."""
    g = gen(21)
    B, H, T, D = 2, 3, 700, 64
    x = normal((B, H, T, D), torch.float32, g)
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, device="cuda")
    inv, _ = skv.rotary_frequencies(D, 500000.0, device="cuda")
    a = pos.double()[:, None, :, None] * inv.double() * (-1 if inverse else 1)
    c, s, e = a.cos(), a.sin(), a.abs() * 4 * 2.0 ** -53 + 2.0 ** -46
    i = torch.arange(D, device="cuda")
    i0, i1 = (i[0::2], i[1::2]) if inter else (i[:D // 2], i[D // 2:])
    x0, x1 = x[..., i0].double(), x[..., i1].double()
    got, _ = skv.apply_rotary(x, None, pos, inv, interleaved=inter, inverse=inverse)
    for j, p, q, name in ((i0, x0 * c, -x1 * s, "first"), (i1, x1 * c, x0 * s, "second")):
        within(got[..., j], p + q, 6 * U32 * (p.abs() + q.abs()) + e * (x0.abs() + x1.abs()), name)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("inter", [False, True])
def test_rotary_in_place_on_slices_of_one_projection(dt, inter):
    """Queries and keys as views of one buffer, rotated where they are; the
    values between them stay."""
    B, T, Hq, Hkv, D = 2, 21, 6, 2, 64
    g = gen(5)
    buf = normal((B, T, Hq + 2 * Hkv, D), DT[dt], g)
    before = buf.clone()
    q, k = buf[:, :, :Hq].transpose(1, 2), buf[:, :, Hq:Hq + Hkv].transpose(1, 2)
    pos = torch.arange(100, 100 + T, device="cuda", dtype=torch.int32)
    inv, _ = skv.rotary_frequencies(D // 2, device="cuda")
    apart = skv.apply_rotary(q, k, pos, inv, interleaved=inter)
    ret = skv.apply_rotary(q, k, pos, inv, interleaved=inter, out=(q, k))
    assert ret[0] is q and ret[1] is k
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1])
    assert torch.equal(buf[:, :, Hq + Hkv:], before[:, :, Hq + Hkv:])


def test_rotary_strides_alignment_and_shapes():
    g = gen(9)
    inv, _ = skv.rotary_frequencies(32, device="cuda")
    pos = torch.tensor([[5, -7, 1 << 30]], device="cuda")
    wide = normal((2, 4, 3, 67), torch.float16, g)
    cases = {
        "odd base": wide[..., 1:33], "odd rows": wide[..., :32], "channels last but one": normal((2, 4, 32, 3), torch.float16, g).transpose(2, 3),
        "heads expanded": normal((2, 1, 3, 32), torch.float16, g).expand(2, 4, 3, 32), "contiguous": normal((2, 4, 3, 32), torch.float16, g),
    }
    for name, q in cases.items():
        got, none = skv.apply_rotary(q, None, pos, inv)
        assert none is None
        want, e = rotary_ref(q, pos, inv, False, 1.0, False)
        within(got, want, e * 1.01 + half(q.dtype) * want.abs() + tiny(q.dtype), name)
    for p in (pos[0], pos, pos.expand(2, 3), torch.stack((pos[0],) * 2, -1).t()[:1]):
        assert torch.equal(skv.apply_rotary(q, None, p, inv)[0], got)
    empty = torch.empty(0, 4, 3, 32, device="cuda", dtype=torch.float16)
    assert skv.apply_rotary(empty, empty, pos[0], inv)[0].shape == empty.shape
    nothing = torch.empty(2, 4, 0, 32, device="cuda", dtype=torch.float16)
    assert skv.apply_rotary(nothing, nothing, pos[0, :0], inv)[0].shape == nothing.shape


def test_rotary_past_32_bit_offsets():
    """A tensor of over 2^31 elements: the last tokens are the ones checked."""
    B, H, T, D = 2, 1, (1 << 24) + 37, 64
    x = torch.empty(B, H, T, D, dtype=torch.bfloat16, device="cuda")
    x[:, :, -50:] = normal((B, H, 50, D), torch.bfloat16, gen(3))
    pos = torch.arange(T, device="cuda")
    inv, _ = skv.rotary_frequencies(D, device="cuda")
    got, _ = skv.apply_rotary(x, None, pos, inv, out=(x.clone(), None))
    want, e = rotary_ref(x[:, :, -50:], pos[-50:], inv, False, 1.0, False)
    within(got[:, :, -50:], want, e * 1.01 + half(x.dtype) * want.abs())
    del x, got
    torch.cuda.empty_cache()


# -- attention with a window and sinks --------------------------------------------------------

def window_ref(q, k, v, window, sinks, starts=None, ends=None, slots=None, scaling=None):
    """Output in 64 bits, and per output the sums its error bound is made of:
    A = sum p |v|, and d, the largest error of a score in 32 bits."""
    B, Hq, T, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    scaling = D ** -0.5 if scaling is None else scaling
    dev = q.device
    zero = torch.zeros(B, dtype=torch.long, device=dev)
    st = zero if starts is None else starts.long().clamp(0, S)
    en = zero + S if ends is None else ends.long().clamp(0, S)
    first = en - T if slots is None else slots.long()
    p = (first[:, None] + torch.arange(T, device=dev))[:, :, None]
    j = torch.arange(S, device=dev)[None, None]
    st, en = st[:, None, None], en[:, None, None]
    sees = (j >= st) & (j <= p) & (p < en) & ((j - st < sinks) | (p - j < window))   # [B, T, S]
    kk = k.double().repeat_interleave(Hq // Hkv, 1)
    vv = v.double().repeat_interleave(Hq // Hkv, 1)
    used = sees.any(1)[:, None, :, None]
    kk, vv = (torch.where(used, x, torch.zeros_like(x)) for x in (kk, vv))
    a = q.double() @ kk.transpose(2, 3) * scaling
    a = a.masked_fill(~sees[:, None], -math.inf)
    pr = torch.softmax(a, -1).nan_to_num(0.0)
    out, A = pr @ vv, pr @ vv.abs()
    d = ((q.double().abs() @ kk.abs().transpose(2, 3)) * abs(scaling)).masked_fill(~sees[:, None], 0.0).amax(-1, keepdim=True)
    n = sees.sum(-1)[:, None, :, None].double()
    return out.transpose(1, 2), A.transpose(1, 2), d.transpose(1, 2), n.transpose(1, 2)


def window_tol(q, ref):
    """A score is a sum of D products in 32 bits, scaled and moved (D + 6
    roundings of at most d); the exponent's own error is 2^-21 relative; sums of
    n weights and products in 32 bits n roundings; weights are rounded once to
    the 16-bit type before the product with v, and the result once more."""
    out, A, d, n = ref
    h = half(q.dtype)
    t = 2 * ((q.shape[-1] + 6) * U32 * d + 2.0 ** -21) * A + 2 * (n + 4) * U32 * A + h * out.abs()
    return (t + (h * A if q.dtype != torch.float32 else 0.0)) * (1 + 4 * h) + tiny(q.dtype)


def check_window(q, k, v, window, sinks, **kw):
    got = skv.sink_window_attention(q, k, v, window=window, sinks=sinks, **kw)
    names = {"query_slots": "slots"}
    ref = window_ref(q, k, v, k.shape[2] if window is None else window, sinks, **{names.get(a, a): b for a, b in kw.items()})
    assert got.shape == (q.shape[0], q.shape[2], q.shape[1], q.shape[3]) and got.is_contiguous()
    within(got, ref[0], window_tol(q, ref), f"{tuple(q.shape)} over {tuple(k.shape)}, window {window}, sinks {sinks}")
    return got


def qkv(B, T, S, Hq, Hkv, D, dt, seed):
    g = gen(seed)
    q = normal((B, T, Hq, D), DT[dt], g).transpose(1, 2)
    return q, normal((B, Hkv, S, D), DT[dt], g), normal((B, Hkv, S, D), DT[dt], g)


WINDOW = [  # B, T, S, Hq, Hkv, window, sinks
    (1, 1, 1, 1, 1, 1, 0), (2, 1, 1, 4, 2, 8, 4), (1, 1, 5, 8, 1, 3, 1), (3, 1, 300, 14, 2, 64, 4), (2, 1, 2000, 32, 8, 700, 5),
    (1, 1, 4097, 8, 8, 4097, 0), (2, 1, 999, 8, 1, 1, 130), (1, 2, 130, 8, 2, 17, 3), (2, 5, 77, 28, 4, 30, 4), (1, 16, 513, 64, 8, 200, 0),
    (1, 64, 64, 4, 4, 64, 0), (2, 100, 100, 8, 2, 1, 0), (1, 127, 127, 4, 1, 32, 2), (2, 128, 128, 4, 2, 128, 4), (1, 129, 257, 8, 2, 100, 7),
    (1, 300, 1111, 8, 2, 257, 130), (2, 385, 385, 14, 2, 129, 4), (1, 700, 700, 32, 8, 90, 200), (3, 260, 260, 3, 3, 1000, 0),
]


@pytest.mark.parametrize("dt, D", [("f32", 16), ("f32", 64), ("f32", 128), ("f16", 16), ("f16", 32), ("f16", 64), ("f16", 128),
                                   ("bf16", 32), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("B, T, S, Hq, Hkv, window, sinks", WINDOW)
def test_window(B, T, S, Hq, Hkv, window, sinks, dt, D):
    q, k, v = qkv(B, T, S, Hq, Hkv, D, dt, 7 * T + S)
    check_window(q, k, v, window, sinks)


@pytest.mark.parametrize("B, T, S, Hq, Hkv, window, sinks", WINDOW)
def test_window_bf16_heads_of_16(B, T, S, Hq, Hkv, window, sinks):
    q, k, v = qkv(B, T, S, Hq, Hkv, 16, "bf16", 7 * T + S)
    check_window(q, k, v, window, sinks)


@pytest.mark.parametrize("dt, D, B, T, window", [("bf16", 64, 4, 900, 200), ("f16", 128, 2, 1111, 500), ("f16", 64, 16, 1, 900),
                                                 ("f32", 64, 3, 130, 100), ("bf16", 16, 2, 300, 77)])
def test_window_equal_calls_give_equal_bits(dt, D, B, T, window):
    q, k, v = qkv(B, T, 1200, 32, 8, D, dt, 6)
    want = skv.sink_window_attention(q, k, v, window=window, sinks=4)
    for _ in range(4):
        assert torch.equal(skv.sink_window_attention(q, k, v, window=window, sinks=4), want)


@pytest.mark.parametrize("dt, D", [("f16", 64), ("bf16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("T, S, Hq, Hkv", [(64, 64, 4, 4), (100, 100, 8, 2), (127, 127, 4, 1), (128, 128, 4, 2), (129, 257, 8, 2),
                                           (260, 260, 3, 3), (300, 1111, 8, 2), (90, 90, 100, 1), (33, 33, 128, 1)])
def test_window_batches_of_prompts(T, S, Hq, Hkv, dt, D):
    """As many blocks of two row tiles as fill the GPU once."""
    tokens = 2 * (128 // (Hq // Hkv))
    B = -(-148 // (-(-T // tokens) * Hkv))
    q, k, v = qkv(B, T, S, Hq, Hkv, D, dt, T + Hq)
    for window, sinks in ((1, 0), (17, 3), (60, 5), (100, 8), (128, 130), (None, 0)):
        check_window(q, k, v, window, sinks)
    # a cache longer than its use, tokens before heads, one row or head for all
    room = torch.full((B, Hkv, S + 23, D), math.nan, dtype=DT[dt], device="cuda")
    room[:, :, 7:7 + S] = k
    want = skv.sink_window_attention(q, k, v, window=128, sinks=9)
    assert torch.equal(want, skv.sink_window_attention(q.contiguous(), room[:, :, 7:7 + S], v.transpose(1, 2).contiguous().transpose(1, 2),
                                                       window=128, sinks=9))
    one_row, one_head = k[:1].expand_as(k), v[:, :1].expand_as(v)
    assert torch.equal(skv.sink_window_attention(q, one_row, one_head, window=128, sinks=9),
                       skv.sink_window_attention(q, one_row.contiguous(), one_head.contiguous(), window=128, sinks=9))


@pytest.mark.parametrize("dt, D", [("f32", 32), ("f16", 64), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("T", [1, 3, 150, 400])
@pytest.mark.parametrize("copies", [1, 9])
def test_window_rows_of_unlike_length(dt, D, T, copies):
    """Left and right padding, rows of no token and of one, queries before and
    behind their row; what lies in the padding is NaN or infinite and reaches no
    output, and a query that sees nothing gives zeros."""
    B, S = 6 * copies, 400
    q, k, v = qkv(B, T, S, 8, 2, D, dt, T)
    starts = torch.tensor([0, 399, 37, 400, 128, -5], dtype=torch.int32, device="cuda").repeat(copies)
    ends = torch.tensor([400, 400, 300, 400, 129, 1000], dtype=torch.int32, device="cuda").repeat(copies)
    first = torch.tensor([0, 398, 30, 0, 127, 200], dtype=torch.int32, device="cuda").repeat(copies)
    for i, bad in enumerate((math.nan, math.inf, -math.inf, math.nan, math.inf, math.nan) * copies):
        dead = torch.ones(S, dtype=torch.bool, device="cuda")
        dead[max(0, int(starts[i])):int(ends[i])] = False
        k[i, :, dead] = bad
        v[i, :, dead] = bad
    for window, sinks in ((20, 4), (None, 0), (129, 140), (1, 1)):
        for slots in (None, torch.full((B,), S - T, dtype=torch.int32, device="cuda"), first):
            got = check_window(q, k, v, window, sinks, starts=starts, ends=ends, query_slots=slots)
            assert not got[3].any()
    got = check_window(q, k, v, 20, 4, ends=torch.zeros(B, dtype=torch.int32, device="cuda"))
    assert not got.any()


@pytest.mark.parametrize("dt, D, T", [("f32", 32, 200), ("f16", 64, 200), ("bf16", 128, 333), ("f16", 128, 1), ("bf16", 64, 3)])
@pytest.mark.parametrize("rows", [1, 40])
def test_window_unseen_tokens_may_hold_anything(dt, D, T, rows):
    """Live tokens that some queries see and others do not: one that is not
    finite reaches exactly the queries that see it."""
    S, window, sinks = 333, 40, 2
    q, k, v = qkv(rows, T, S, 4, 2, D, dt, 3)
    at = [S - T, S - 60, S - 1] if T > 60 else [S - 60, S - 50]
    clean = v.clone()
    for n, j in enumerate(at):
        v[:, :, j] = (math.nan, math.inf, -math.inf)[n]
    got = skv.sink_window_attention(q, k, v, window=window, sinks=sinks)
    ref = window_ref(q, k, clean, window, sinks)
    p = torch.arange(S - T, S, device="cuda")
    hit = torch.zeros(T, dtype=torch.bool, device="cuda")
    for j in at:
        hit |= (j <= p) & ((p - j < window) | (j < sinks))
    assert not got[:, hit].isfinite().any()
    within(got[:, ~hit], ref[0][:, ~hit], window_tol(q, ref)[:, ~hit])


@pytest.mark.parametrize("dt, D, T", [("f32", 32, 200), ("f16", 16, 9), ("f16", 64, 200), ("bf16", 128, 333), ("f16", 128, 1), ("bf16", 64, 3)])
@pytest.mark.parametrize("rows", [1, 40])
def test_window_scores_of_minus_infinity(dt, D, T, rows):
    """A key whose score is -inf weighs nothing; a query of such keys alone
    gives zeros.  Without its infinite channel a key's score is -10^4 / sqrt(D)
    or below -800 and its 64-bit weight beside another key's exactly 0."""
    S, window = 333, 40
    q, k, v = qkv(rows, T, S, 4, 2, D, dt, 5)
    q[..., 0] = 1
    gone = torch.zeros(S, dtype=torch.bool, device="cuda")
    gone[::3] = True
    gone[S - 41:] = True
    gone[S - 150:S - 100] = True
    clean, low = k.clone(), k.clone()
    k[:, :, gone, 0] = -math.inf
    low[:, :, gone, 0] = -1e4
    clean[:, :, gone, 0] = 0
    p = torch.arange(S - T, S, device="cuda")[:, None]
    j = torch.arange(S, device="cuda")
    for sinks in (0, 2):
        got = skv.sink_window_attention(q, k, v, window=window, sinks=sinks)
        some = ((j <= p) & ((p - j < window) | (j < sinks)) & ~gone).any(1)
        assert (sinks == 2 or not some.all()) and not got[:, ~some].any()
        out, A, _, n = window_ref(q, low, v, window, sinks)
        d = window_ref(q, clean, v, window, sinks)[2]
        within(got[:, some], out[:, some], window_tol(q, (out, A, d, n))[:, some])


@pytest.mark.parametrize("dt, D", [("f32", 16), ("f32", 64), ("f32", 128), ("f16", 16), ("f16", 64), ("bf16", 32), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("T, rows, window", [(1, 1, 40), (1, 40, 40), (3, 1, 40), (200, 1, 40), (200, 40, 40), (333, 60, 170)])
def test_window_scores_that_are_not_finite(dt, D, T, rows, window):
    """A NaN among the scores a query sees, or one of +inf, makes its output
    NaN, as the softmax of such scores is, whatever its other scores are; the
    outputs of the other queries stay."""
    S = 333
    q, k, v = qkv(rows, T, S, 4, 2, D, dt, 11)
    ref = window_ref(q, k, v, window, 2)
    tol = window_tol(q, ref)
    one = q.clone()
    one[:, 1, T - 1, 3] = math.nan                 # every score of one query
    got = skv.sink_window_attention(one, k, v, window=window, sinks=2)
    hit = torch.zeros(rows, T, 4, dtype=torch.bool, device="cuda")
    hit[:, T - 1, 1] = True
    assert got[hit].isnan().all()
    within(got[~hit], ref[0][~hit], tol[~hit])
    # a key that is all a query sees
    bad = k.clone()
    bad[:, 0, S - 1, 0] = math.nan
    alone = window_ref(q, k, v, 1, 0)
    got = skv.sink_window_attention(q, bad, v, window=1)
    hit = torch.zeros(rows, T, 4, dtype=torch.bool, device="cuda")
    hit[:, T - 1, :2] = True                       # the heads that share kv head 0
    assert got[hit].isnan().all()
    within(got[~hit], alone[0][~hit], window_tol(q, alone)[~hit])
    # scores of +inf and of NaN that some queries see
    q[..., 0] = 1
    ref = window_ref(q, k, v, window, 2)
    tol = window_tol(q, ref)
    p = torch.arange(S - T, S, device="cuda")
    for value in (math.inf, math.nan):
        for j in (S - 1, S - 60, 1):
            bad = k.clone()
            bad[:, :, j, 0] = value
            got = skv.sink_window_attention(q, bad, v, window=window, sinks=2)
            hit = (j <= p) & ((p - j < window) | (j < 2))
            assert got[:, hit].isnan().all(), (value, j)
            within(got[:, ~hit], ref[0][:, ~hit], tol[:, ~hit], f"{value} at {j}")


@pytest.mark.parametrize("dt, D", [("f32", 16), ("f32", 128), ("f16", 32), ("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("lo, hi", [(0, 300), (0, 1), (3999, 4000), (1000, 4000), (0, 4000), (2000, 2256)])
def test_window_whole_shares_of_scores_that_are_nan(dt, D, lo, hi):
    """Decode of a row whose keys are shared out over many warps and blocks,
    some of which see NaN and nothing else."""
    q, k, v = qkv(1, 1, 4000, 4, 2, D, dt, 12)
    want = skv.sink_window_attention(q, k, v)
    k[:, 1, lo:hi] = math.nan
    got = skv.sink_window_attention(q, k, v)
    assert got[:, :, 2:].isnan().all() and torch.equal(got[:, :, :2], want[:, :, :2])


@pytest.mark.parametrize("dt, D", [("f16", 16), ("f16", 64), ("f16", 128), ("bf16", 64), ("f32", 32)])
@pytest.mark.parametrize("T, rows", [(1, 1), (1, 40), (9, 2), (333, 60)])
def test_window_weights_far_below_the_largest(dt, D, T, rows):
    """A first token that takes nearly all weight and holds zeros: the output is
    made of weights from 2^-12 to 2^-25 of the largest.  fp16 weights are scaled
    to at most 2^15, the largest to 2^7 at least, so below 2^-14 they are off by
    2^-25 / 2^7 of it at most (two terms: less), on top of the usual bound."""
    S, window = 333, 170
    q, k, v = qkv(rows, T, S, 4, 2, D, dt, 17)
    q.zero_()
    q[..., 0] = 1
    k[..., 0] = -8.5 - 8.5 * torch.rand(rows, 2, S, generator=gen(18), device="cuda")
    k[:, :, 0, 0] = 0
    v.mul_(64)
    v[:, :, 0] = 0
    got = skv.sink_window_attention(q, k, v, window=window, sinks=1, scaling=1.0)
    ref = window_ref(q, k, v, window, 1, scaling=1.0)
    size = window_ref(torch.zeros_like(q), k, v, window, 1)  # of equal weights: A is the mean of |v|
    within(got, ref[0], window_tol(q, ref) + (2.0 ** -32 * size[1] * size[3] if dt == "f16" else 0.0))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B, T", [(2, 1), (2, 40), (60, 150)])
def test_window_strides(dt, B, T):
    """Caches longer than their use, heads and tokens in any order, bases and
    rows that are not 16-byte aligned, heads shared by expansion."""
    S, Hq, Hkv, D = 200, 6, 2, 64
    q, k, v = qkv(B, T, S, Hq, Hkv, D, dt, 4)
    want = check_window(q, k, v, 50, 3)
    room = torch.full((B, Hkv, S + 57, D), math.nan, dtype=DT[dt], device="cuda")
    room[:, :, 9:9 + S] = k
    tokens_first = v.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(B, Hkv, S, D + 1, dtype=DT[dt], device="cuda")[..., 1:]
    odd.copy_(k)
    channels = v.transpose(2, 3).contiguous().transpose(2, 3)
    for kk in (room[:, :, 9:9 + S], odd):
        for vv in (tokens_first, channels):
            for qq in (q, q.contiguous(), q.transpose(2, 3).contiguous().transpose(2, 3)):
                assert torch.equal(skv.sink_window_attention(qq, kk, vv, window=50, sinks=3), want)
    one = k[:, :1].expand(B, Hkv, S, D)
    assert torch.equal(skv.sink_window_attention(q, one, one, window=50, sinks=3),
                       skv.sink_window_attention(q, one.contiguous(), one.contiguous(), window=50, sinks=3))
    place = torch.empty(B, T, Hq, D, dtype=DT[dt], device="cuda")
    assert skv.sink_window_attention(q, k, v, window=50, sinks=3, out=place) is place and torch.equal(place, want)


@pytest.mark.parametrize("dt, D", [("f32", 32), ("f16", 64), ("bf16", 128), ("f16", 32)])
@pytest.mark.parametrize("Hq, Hkv", [(128, 1), (256, 1), (260, 2), (100, 1)])
def test_window_many_heads_to_a_kv_head(dt, D, Hq, Hkv):
    """Groups of 100 to 256 query heads: as large as a tile, larger, and of no
    divisor in common with it."""
    for T, S in ((1, 200), (5, 200), (70, 70)):
        q, k, v = qkv(2, T, S, Hq, Hkv, D, dt, T)
        check_window(q, k, v, 60, 3)


@pytest.mark.parametrize("dt, D", [("bf16", 64), ("f16", 128), ("f32", 64)])
@pytest.mark.parametrize("B, T", [(1, 1), (1, 200), (1, 900), (12, 900)])
def test_window_lengths_around_tiles(dt, D, B, T):
    """First tokens and windows that end on, before and behind the borders of
    8- and 128-key tiles."""
    q, k, v = qkv(B, T, 900, 4, 1, D, dt, T)
    for sinks in (0, 1, 7, 8, 9, 127, 128, 129, 300):
        for window in (1, 2, 63, 64, 65, 127, 128, 129, 500):
            check_window(q, k, v, window, sinks)


def test_window_repeated_calls_are_checked_again():
    """Calls alike in shapes and settings: another input that asks for
    gradients, is misaligned or on the host is refused or copied all the same."""
    q, k, v = qkv(2, 1, 64, 4, 2, 64, "f16", 1)
    want = [skv.sink_window_attention(q, k, v, window=9) for _ in range(3)][-1]
    base = torch.empty(k.numel() + 1, dtype=k.dtype, device="cuda")
    odd = base[1:].view(k.shape)
    odd.copy_(k)
    assert odd.stride() == k.stride() and odd.data_ptr() % 16
    assert torch.equal(skv.sink_window_attention(q, odd, v, window=9), want)
    with pytest.raises(NotImplementedError):
        skv.sink_window_attention(q.clone().requires_grad_(), k, v, window=9)
    with pytest.raises(ValueError):
        skv.sink_window_attention(q, k.cpu(), v, window=9)
    inv, _ = skv.rotary_frequencies(64, device="cuda")
    pos = torch.arange(1, device="cuda")
    a = [skv.apply_rotary(q, k[:, :, :1], pos, inv) for _ in range(3)]
    assert all(torch.equal(x, y) for x, y in zip(a[0], a[2]))
    with pytest.raises(NotImplementedError):
        skv.apply_rotary(q.clone().requires_grad_(), k[:, :, :1], pos, inv)
    x, u = torch.randn(2, 99, device="cuda"), torch.rand(2, device="cuda")
    b = [skv.sample_tokens(x, u, top_k=5) for _ in range(3)]
    assert torch.equal(b[0], b[2])
    check_sample(x, u, top_k=6)
    with pytest.raises(NotImplementedError):
        skv.sample_tokens(x.clone().requires_grad_(), u, top_k=5)
    with pytest.raises(ValueError):
        skv.sample_tokens(x, u.cpu(), top_k=5)


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_settings_in_tensors_are_read_at_each_call(device):
    """A setting given as a 0-dim tensor counts with what it holds at the call."""
    q, k, v = qkv(2, 1, 64, 4, 2, 64, "f16", 1)
    inv, _ = skv.rotary_frequencies(64, device="cuda")
    pos = torch.arange(5, 6, device="cuda")
    x, u = normal((2, 99), torch.float32, gen(2)), torch.rand(2, generator=gen(3), device="cuda")
    attend = lambda **kw: skv.sink_window_attention(q, k, v, **kw)  # noqa: E731
    rotate = lambda **kw: skv.apply_rotary(q, None, pos, inv, **kw)[0]  # noqa: E731
    for call, name, values in ((attend, "scaling", (0.125, 0.5)), (attend, "window", (9, 30)), (rotate, "scale", (1.0, 0.75)),
                               (rotate, "inverse", (False, True)), (rotate, "interleaved", (False, True))):
        other = {"window": 20} if call is attend and name != "window" else {}
        want = [call(**{name: y}, **other) for y in values]
        assert not torch.equal(*want)
        t = torch.tensor(values[0], device=device)
        for y, w in ((values[0], want[0]), (values[1], want[1]), (values[0], want[0])):
            t.fill_(y)
            for _ in range(2):
                assert torch.equal(call(**{name: t}, **other), w), (name, y)
    few = torch.tensor(3, device=device)
    want = [attend(window=5, sinks=n) for n in (3, 11)]
    assert torch.equal(attend(window=5, sinks=few), want[0]) and torch.equal(attend(window=5, sinks=few.fill_(11)), want[1])
    top_k = np.int64(4)
    assert torch.equal(skv.sample_tokens(x, u, top_k=top_k), skv.sample_tokens(x, u, top_k=4))


def test_tangents_are_refused_of_repeated_calls():
    from torch.autograd import forward_ad
    q, k, v = qkv(2, 1, 64, 4, 2, 64, "f16", 1)
    want = [skv.sink_window_attention(q, k, v, window=9) for _ in range(2)][0]
    with forward_ad.dual_level():
        assert torch.equal(skv.sink_window_attention(q, k, v, window=9), want)
        for i in range(3):
            x = [q, k, v]
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(NotImplementedError, match="no derivative"):
                skv.sink_window_attention(*x, window=9)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T, D", [(1, 64), (30, 32), (700, 64), (700, 128)])
def test_window_of_nan_queries_takes_no_longer(T, D, dt):
    """Rows whose own scores are NaN are not done again key by key, which takes
    from 30 to 500 times as long: a call of nothing but NaN stays within five
    times the call of finite numbers (the same work, timed by the fastest of
    several)."""
    q, k, v = qkv(8, T, 4000, 32, 8, D, dt, 23)
    bad = torch.full_like(q, math.nan)

    def fastest(x):
        times = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(100000)
            a.record()
            out = skv.sink_window_attention(x, k, v, window=2000, sinks=4)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times), out

    finite, _ = fastest(q)
    nan, out = fastest(bad)
    assert out.isnan().all() and nan < 5 * finite


def test_window_past_32_bit_offsets():
    """A cache of over 2^31 elements, most of it never written; decode and a
    chunk at its far end and, with sinks, at its beginning."""
    B, Hkv, S, D = 1, 2, (1 << 24) + 1000, 64
    k, v = (torch.empty(B, Hkv, S, D, dtype=torch.float16, device="cuda") for _ in range(2))
    g = gen(8)
    for x in (k, v):
        x[:, :, -700:] = normal((B, Hkv, 700, D), torch.float16, g)
        x[:, :, :4] = normal((B, Hkv, 4, D), torch.float16, g)
    near = [torch.cat((x[:, :, :4], x[:, :, -700:]), 2) for x in (k, v)]
    for T in (1, 200, 690):
        q = normal((B, 64, T, D), torch.float16, g)
        window = min(400, 700 - T)
        got = skv.sink_window_attention(q, k, v, window=window, sinks=4)
        ref = window_ref(q, *near, window, 4)
        within(got, ref[0], window_tol(q, ref))
    del k, v
    torch.cuda.empty_cache()


def test_window_large_scores_and_lowest_values():
    """Scores far apart, and keys of the type's lowest value."""
    for dt in ("f16", "bf16", "f32"):
        for B, T in ((1, 1), (1, 200), (30, 200)):
            q, k, v = qkv(B, T, 300, 4, 2, 64, dt, 6)
            check_window(q, k, v, 70, 4, scaling=4.0)
            check_window(q, k, v, 70, 4, scaling=-0.5)
            check_window(q, k, v, 70, 4, scaling=0.0)
            low = k.clone()
            low[:, :, ::3] = torch.finfo(DT[dt]).min / 64 if dt == "f16" else -1e4
            check_window(q, low, v, 70, 4)


# -- sampling --------------------------------------------------------------------------------

def sample_ref(x, u, temperature, top_k, top_p, min_p):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0])
    if top_k > 0:
        order = order[:top_k]
    m = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp(np.where(x == m, 0.0, x - m) / np.float64(np.float32(temperature))))
    if top_p < 1:
        c = np.cumsum(w[order])
        order = order[:max(1, int(np.searchsorted(c, np.float64(np.float32(top_p)) * c[-1])) + 1)]
    order = np.sort(order[w[order] >= min(np.float64(np.float32(min_p)), 1.0)])
    c = np.cumsum(w[order])
    live = order[w[order] > 0]
    n = int(np.searchsorted(c, np.float64(np.float32(u)) * c[-1], side="right"))
    return int(order[n]) if n < len(order) else int(live[-1])


def check_sample(x, u, **kw):
    got = skv.sample_tokens(x, u, **kw)
    B = x.shape[0]
    each = [kw[n].cpu().numpy() if torch.is_tensor(kw.get(n)) else np.full(B, kw.get(n, d))
            for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))]
    want = [sample_ref(r, uu, *s) for r, uu, *s in zip(x.float().cpu().numpy(), u.cpu().numpy(), *each)]
    assert got.dtype == torch.int64 and got.tolist() == want
    return got


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [1, 2, 31, 33, 257, 1000, 1023, 4097, 32000, 50001, 128256])
def test_sample(V, dt):
    B = 5
    g = gen(V)
    for sharp in (0.3, 2.0, 6.0):
        x = normal((B, V), torch.float32, g).mul(sharp).to(DT[dt])
        for kw in (dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.95), dict(top_k=1), dict(top_k=V),
                   dict(top_p=0.9), dict(temperature=1.3, top_p=0.5, min_p=0.1), dict(min_p=0.05), dict(top_k=3000, top_p=0.999),
                   dict(top_p=1e-6), dict(temperature=1e-3), dict(temperature=50.0, top_k=700, min_p=0.9), dict(min_p=1.0)):
            u = torch.rand(B, generator=g, device="cuda")
            check_sample(x, u, **kw)


def test_sample_settings_of_each_row():
    B, V = 64, 5003
    g = gen(2)
    x = normal((B, V), torch.float32, g) * 3
    pick = lambda vals, dtype: torch.tensor(vals, dtype=dtype, device="cuda")[  # noqa: E731
        torch.randint(0, len(vals), (B,), generator=g, device="cuda")]
    kw = dict(temperature=pick([0.0, -1.0, 0.4, 1.0, 2.0, math.nan], torch.float32), top_k=pick([0, -3, 1, 40, 2000, 99999], torch.int32),
              top_p=pick([1.0, 2.0, 0.9, 0.3, 0.0, -1.0], torch.float32), min_p=pick([0.0, -1.0, 0.1, 1.0, 3.0], torch.float32))
    for dt in DT.values():
        check_sample(x.to(dt), torch.rand(B, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("dt", DT)
def test_sample_ties_and_masks(dt):
    """Equal logits are taken by index; -inf, NaN, the type's lowest value and
    +inf; empty rows; both ends of the random numbers."""
    V = 3001
    low, inf, nan = torch.finfo(DT[dt]).min, math.inf, math.nan
    rows = {
        "all equal": torch.zeros(V), "few levels": (torch.arange(V) * 7 % 3).float(), "one": torch.full((V,), -inf),
        "all -inf": torch.full((V,), -inf), "all NaN": torch.full((V,), nan), "all lowest": torch.full((V,), low),
        "lowest and zero": torch.where(torch.arange(V) % 2 == 0, 0.0, low), "NaN between": torch.where(torch.arange(V) % 2 == 0, nan, 1.0),
        "+inf twice": torch.zeros(V), "signed zeros": torch.where(torch.arange(V) % 3 == 0, -0.0, 0.0),
    }
    rows["one"][1234] = -5.0
    rows["+inf twice"][[17, 2900]] = inf
    x = torch.stack(list(rows.values())).cuda().to(DT[dt])
    for u0 in (0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24):
        u = torch.full((x.shape[0],), u0, device="cuda")
        for kw in (dict(), dict(top_k=1), dict(top_k=10), dict(top_p=0.5), dict(top_p=0.9, top_k=1000), dict(min_p=0.5), dict(temperature=0.0),
                   dict(temperature=0.7, top_p=0.25, top_k=2)):
            got = check_sample(x, u, **kw)
            assert got[3] == -1 and got[4] == -1 and got[2] == 1234 and got[8] in (17, 2900)


@pytest.mark.parametrize("dt", DT)
def test_sample_cuts_among_equals(dt):
    """Cuts that fall inside runs of equal logits, at the head of the order and
    far down, with lists that hold the run and runs that no list holds."""
    V = 20000
    g = gen(31)
    u = torch.rand(6, generator=g, device="cuda")
    x = normal((6, V), torch.float32, g)
    x[0] = x[0].round()                       # thousands of equals each
    x[1] = (x[1] * 4).round() / 4
    x[2, 1000:1300] = 5.0                     # a run of 300 above the rest
    x[3, ::7] = 6.0                           # a run of 2858 above the rest
    x[4, 1::2] = -math.inf
    x[5] = x[5].clamp(max=0.5)
    x = x.to(DT[dt])
    for kw in (dict(top_k=40), dict(top_k=299), dict(top_k=301), dict(top_k=2500), dict(top_k=3000), dict(top_k=9999), dict(top_k=15000),
               dict(top_p=0.1), dict(top_p=0.5), dict(top_p=0.97), dict(top_k=150, top_p=0.5), dict(top_k=2900, top_p=0.3),
               dict(top_k=12000, top_p=0.8, temperature=3.0), dict(temperature=0.05, top_p=0.9), dict(top_p=0.999999)):
        check_sample(x, u, **kw)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("step, levels, many", [(0.5, 16, 13), (0.25, 30, 200), (2.0, 6, 3), (0.015625, 64, 20)])
def test_sample_cuts_between_levels(step, levels, many, dt):
    """Shares of top-p one step of float32 to each side of a level's end, and
    nearest to it: 32-bit sums cannot tell which level holds the cut.  The
    vocabulary ascends, so that a random number of 0 draws the cut's level."""
    counts = [1 + many * j for j in range(levels)]
    x = torch.cat([torch.full((n,), 4.0 - step * j) for j, n in reversed(list(enumerate(counts)))])
    mass = np.cumsum([n * np.exp(-step * j) for j, n in enumerate(counts)])
    ends = (mass[:-1] / mass[-1]).astype(np.float32)
    shares = np.concatenate([np.nextafter(ends, np.float32(0)), ends, np.nextafter(ends, np.float32(1))])
    assert np.abs(shares.astype(np.float64)[:, None] - mass[:-1] / mass[-1]).min() > 1e-13  # 64-bit sums can tell
    B = len(shares)
    x = x.to(DT[dt]).cuda().expand(B, -1)
    top_p = torch.from_numpy(shares).cuda()
    for u in (torch.zeros(B, device="cuda"), torch.rand(B, generator=gen(levels), device="cuda")):
        check_sample(x, u, top_p=top_p)
        check_sample(x, u, top_p=top_p, top_k=x.shape[1] - 1)


def test_sample_extreme_scales():
    """Logits and temperatures near the ends of their types."""
    g = gen(41)
    V = 3000
    u = torch.rand(4, generator=g, device="cuda")
    for scale in (1e-30, 1e-6, 1e4, 1e30, 3e38):
        x = (torch.rand(4, V, generator=g, device="cuda") * 2 - 1) * scale
        for temperature in (1e-38, 1e-3, 1.0, 1e3, 1e38):
            for kw in (dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.7), dict(top_k=2000, min_p=0.5)):
                check_sample(x, u, temperature=temperature, **kw)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [1, 700, 50001])
def test_sample_top_p_that_keeps_one_token(V, dt):
    """Shares of nothing and of less, with and without other cuts: the first of
    the largest logits, thousands of them among the rows."""
    x = normal((9, V), torch.float32, gen(V)).to(DT[dt])
    x[1::3] = x[1::3].clamp(max=0.25)
    x[2, V // 3] = math.inf
    top_p = torch.tensor([0.0, 0.0, 0.0, -0.0, -1.0, -math.inf, 1e-45, 1e-38, 1e-30], device="cuda")
    u = torch.rand(9, generator=gen(7), device="cuda")
    for kw in (dict(), dict(top_k=5), dict(top_k=600), dict(temperature=100.0), dict(temperature=1e-30), dict(min_p=0.5)):
        got = check_sample(x, u, top_p=top_p, **kw)
        assert got.tolist() == np.argmax(x.float().cpu().numpy(), 1).tolist()


@pytest.mark.parametrize("V", [40, 1500, 50001])
def test_sample_top_k_past_the_vocabulary(V):
    """The largest and smallest whole numbers a setting holds, as "no limit"."""
    x = normal((10, V), torch.float32, gen(V))
    u = torch.rand(10, generator=gen(7), device="cuda")
    top_k = torch.tensor([V - 1, V, V + 1, 1 << 30, (1 << 30) - 1, (1 << 31) - 1, (1 << 31) - 2, -(1 << 31), -1, 0], dtype=torch.int32,
                         device="cuda")
    check_sample(x, u, top_k=top_k)
    check_sample(x, u, top_k=top_k, top_p=0.9)
    for k in ((1 << 30), (1 << 31) - 1, 1 << 40):
        assert torch.equal(skv.sample_tokens(x, u, top_k=k), skv.sample_tokens(x, u))


# largest logit, temperature, min-p (float32): the logit that weighs min-p is 0 to 10^-13 and less
MIN_P_AT_ZERO = [(2.565428, 1.1141512, 0.1), (1.3165607, 1.0935137, 0.3), (1.9748411, 1.6402706, 0.3), (3.6204104, 1.9083719, 0.15),
                 (3.3644526, 1.7734528, 0.15), (7.7067885, 1.9700264, 0.02), (7.156755, 1.8294256, 0.02), (4.9612117, 1.0773134, 0.01),
                 (6.9456964, 1.5082388, 0.01), (4.117248, 1.374705, 0.05)]


def test_sample_min_p_whose_border_is_zero():
    """Logits one part in 10^6 to each side of such a border, where a billion
    float32 numbers lie between it and an estimate of it."""
    g = gen(51)
    V = 1500
    x = normal((len(MIN_P_AT_ZERO), V), torch.float32, g)
    x = torch.where(x.abs() < 1e-6, torch.full_like(x, 1e-6), x).clamp(max=1.0)
    x[:, 100], x[:, 900] = 1e-6, -1e-6
    m, temperature, min_p = (torch.tensor(c, dtype=torch.float32, device="cuda") for c in zip(*MIN_P_AT_ZERO))
    x[:, 700] = m
    for u0 in (0.0, 0.3, 0.7, 1.0 - 2.0 ** -24):
        u = torch.full_like(m, u0)
        check_sample(x, u, temperature=temperature, min_p=min_p)
        check_sample(x, u, temperature=temperature, min_p=min_p, top_k=1200)


def test_sample_weights_are_64_bit():
    """Logits whose weights differ from min-p by 4e-15 of it and more, to either
    side: as many times what 64-bit roundings move (an exponent of 4 and an
    exponential, together under 1e-15).  The last kept token is drawn."""
    rows = []
    for m, temperature, min_p in MIN_P_AT_ZERO:
        at = np.longdouble(np.float32(m)) + np.log(np.longdouble(np.float32(min_p))) * np.longdouble(np.float32(temperature))
        for near in (0.0, at - 1e-14, at + 1e-14, at - 1e-13, at + 1e-13, at - 1e-12, at + 1e-12):
            if abs(np.longdouble(np.float32(near)) - at) > 4e-15 * temperature:
                rows.append((m, float(np.float32(near)), -20.0, temperature, min_p))
    assert len(rows) > 55
    t = torch.tensor(rows, dtype=torch.float32, device="cuda")
    u = torch.full((len(rows),), 1.0 - 2.0 ** -24, device="cuda")
    x, temperature, min_p = t[:, :3].contiguous(), t[:, 3].contiguous(), t[:, 4].contiguous()
    got = check_sample(x, u, temperature=temperature, min_p=min_p)
    assert set(got.tolist()) == {0, 1}


def test_sample_random_numbers_out_of_range_stay_in_the_vocabulary():
    x = normal((5, 1000), torch.float32, gen(5))
    u = torch.tensor([1.0, 2.0, -1.0, math.nan, math.inf], device="cuda")
    for kw in (dict(), dict(top_k=7), dict(top_p=0.9)):
        got = skv.sample_tokens(x, u, **kw)
        assert ((got >= 0) & (got < 1000)).all()


def test_sample_rows_apart_and_odd_bases():
    g = gen(12)
    for dt in DT.values():
        wide = normal((7, 2050), torch.float32, g).to(dt)
        u = torch.rand(7, generator=g, device="cuda")
        for x in (wide[:, 1:2001], wide[:, :777], wide[::2, 3:], wide.t().contiguous().t(), wide[:1].expand(7, 2050)):
            check_sample(x, u[:x.shape[0]].clone(), top_p=0.8)
            check_sample(x, u[:x.shape[0]].clone(), top_k=33)
    assert skv.sample_tokens(wide[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dt, V", [("f32", 1 << 22), ("f16", 1000003), ("bf16", 400001)])
def test_sample_large_vocabularies(dt, V):
    """Rows past what a cluster's shared memory holds, with cuts that keep few
    and that keep many, and with so many equals that no list holds them."""
    g = gen(V)
    x = normal((2, V), torch.float32, g).mul(2.0).to(DT[dt])
    u = torch.rand(2, generator=g, device="cuda")
    for kw in (dict(), dict(top_k=100, top_p=0.9), dict(top_k=70000), dict(top_p=0.7), dict(top_k=200000, top_p=0.95, min_p=1e-4)):
        check_sample(x, u, **kw)
    few = (torch.arange(V, device="cuda") % 5).to(DT[dt]).expand(2, V)
    for kw in (dict(top_p=0.8), dict(top_k=V // 2 + 3), dict(top_k=V // 2, top_p=0.93)):
        check_sample(few, u, **kw)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_sample_few_levels_of_the_largest_vocabulary(dt):
    """Half a million tokens of a block in one bin of the weights' histogram,
    of two levels and of one level with another beside it."""
    V = 1 << 22
    i = torch.arange(V, device="cuda")
    x = torch.stack(((i % 2).float(), (i % 32 == 5).float() * 0.5, (i < V // 2).float() * 3)).to(DT[dt])
    u = torch.rand(3, generator=gen(19), device="cuda")
    for kw in (dict(top_p=0.3), dict(top_p=0.8), dict(top_p=0.95, temperature=0.7), dict(top_p=0.8, top_k=V - 1000), dict(top_p=0.999999)):
        check_sample(x, u, **kw)


def test_sample_frequencies():
    """4096 evenly spaced random numbers choose each token as often as its
    probability says, to one draw at each of its two borders."""
    V, n = 50, 4096
    x = normal((1, V), torch.float32, gen(1)) * 1.5
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = skv.sample_tokens(x.expand(n, V), u.float(), temperature=0.8, top_k=20)
    w = torch.softmax(x[0].double() / np.float64(np.float32(0.8)), 0)
    keep = w >= w.sort(descending=True).values[19]
    w = torch.where(keep, w, torch.zeros_like(w))
    count = torch.bincount(got, minlength=V).double()
    assert ((count - w / w.sum() * n).abs() <= 2).all()


# -- streams, graphs and a run together ---------------------------------------------------------

def test_operators_on_another_stream_and_in_graphs_of_their_own():
    """Called on a side stream; two graphs captured apart and replayed side by
    side on two streams give what the eager calls give for their inputs."""
    g = gen(20)
    inv, _ = skv.rotary_frequencies(64, device="cuda")
    pos = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    static = []
    for i in range(2):
        q, k, v = qkv(2, 1, 3000, 8, 2, 64, "bf16", 30 + i)
        static.append(dict(q=q, k=k, v=v, x=normal((2, 9001), torch.float32, g), u=torch.rand(2, generator=g, device="cuda")))

    def step(s):
        a, _ = skv.apply_rotary(s["q"], None, pos, inv)
        o = skv.sink_window_attention(a, s["k"], s["v"], window=2500, sinks=4)
        return o, skv.sample_tokens(s["x"], s["u"], temperature=0.9, top_p=0.9), skv.sample_tokens(s["x"], s["u"], top_k=40)

    side = torch.cuda.Stream()
    graphs, outs = [], []
    for s in static:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    for trial in range(3):
        for s in static:
            for name in ("q", "k", "v"):
                s[name].copy_(normal(s[name].shape, torch.bfloat16, g))
            s["x"].normal_(generator=g)
        want = [step(s) for s in static]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(a, b) for a, b in zip(w, o))


def test_a_decode_loop_of_all_three():
    """A tiny one-layer model decodes over a preallocated cache: rotary, append,
    window attention, logits, sampling.  Each step's attention and token are
    checked against the 64-bit forms on the step's own inputs, and the loop
    replayed from one graph gives the same tokens."""
    B, Hq, Hkv, D, V, S, window, sinks = 3, 8, 2, 64, 501, 64, 10, 2
    g = gen(77)
    dtype = torch.bfloat16
    E = normal((V, Hq * D), dtype, g)
    Wq, Wk, Wv = (normal((Hq * D, h * D), dtype, g) * 0.05 for h in (Hq, Hkv, Hkv))
    inv, scale = skv.rotary_frequencies(D // 2, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32},
                                        device="cuda")
    uniforms = torch.rand(40, B, generator=g, device="cuda")
    k, v = (torch.full((B, Hkv, S, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    tok, n, u = torch.zeros(B, dtype=torch.long, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, device="cuda")
    seen = {}

    def step():
        h = E[tok]
        q, kn, vn = ((h @ W).view(B, 1, -1, D).transpose(1, 2) for W in (Wq, Wk, Wv))
        pos = n.long()[:, None]
        q, kn = skv.apply_rotary(q, kn, pos, inv, scale=scale)
        at = pos.view(B, 1, 1, 1).expand(B, Hkv, 1, D)
        k.scatter_(2, at, kn)
        v.scatter_(2, at, vn)
        n.add_(1)
        o = skv.sink_window_attention(q, k, v, window=window, sinks=sinks, ends=n)
        logits = (o.reshape(B, -1) @ E.t()) * 0.05
        seen.update(q=q, o=o, logits=logits)
        tok.copy_(skv.sample_tokens(logits, u, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01))

    def run(one):
        tok.zero_(), n.zero_(), k.fill_(math.nan), v.fill_(math.nan)
        got = []
        for i in range(40):
            u.copy_(uniforms[i])
            one()
            got.append(tok.tolist())
        return got

    def checked():
        step()
        ref = window_ref(seen["q"], k, v, window, sinks, ends=n)
        within(seen["o"], ref[0], window_tol(seen["q"], ref))
        x = seen["logits"].float().cpu().numpy()
        assert tok.tolist() == [sample_ref(r, uu, 0.9, 40, 0.95, 0.01) for r, uu in zip(x, u.cpu().numpy())]

    with torch.no_grad():
        want = run(checked)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        assert run(graph.replay) == want
