"""Corners of K8 (visible scores of minus infinity, infinite values of little weight, many small weights) and of K7 (NaN bit
patterns). Bars as in test_norm_w4_window_gpu."""
import math

import pytest
import torch

import gpu_harness as G
from cubert_b200 import kernels
from test_norm_w4_window_gpu import (HALF_STEP, SMALLEST, TYPES, attention64, check_window, gen, matvec, norm_bar, normal, pack, rms_norm, step,
                                     window64, window_attention, window_inputs, within)

pytestmark = pytest.mark.gpu
INF = float("inf")


# ============================================================================ K8: visible scores of minus infinity

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad", [0, 1])                          # 1: rows that only the general loads can read
@pytest.mark.parametrize("seq,dim", [(5, 64), (45, 64), (45, 128), (300, 64), (300, 128), (300, 40), (45, 256)])
def test_rows_that_see_only_scores_of_minus_infinity_are_nan(seq, dim, pad, t):
    """softmax of nothing but minus infinity is 0 / 0; zeros are for rows that see no key at all."""
    batch, heads, before = 3, 2, 3
    q, k, v, _ = window_inputs(seq + dim, batch, seq, heads, heads, dim, None, t, pad)
    q.abs_().add_(0.125)
    m = torch.ones((batch, seq), dtype=torch.int8, device="cuda")
    low = [0, 1] if seq == 5 else list(range(10, 20))            # sequence 0: these keys, and so some rows see nothing else
    k[low, 0::dim] = -INF
    m[0, low[0]] = 0                                             # a masked one does not count as seen
    k[seq:2 * seq, 0::dim] = -INF                                # sequence 1: every key
    m[2, seq // 2:] = 0                                          # sequence 2: rows that see nothing
    args = (batch, seq, heads, heads, dim, before, 0, 0, dim ** -0.5)
    got = window_attention(q, k, v, m, *args, t).view(batch, seq, heads * dim)
    ref = tuple(a.view(batch, seq, heads * dim) for a in window64(q, k, v, m, *args))
    nan = torch.zeros((batch, seq), dtype=torch.bool, device="cuda")
    kept = [j for j in low if j != low[0]]
    for i in range(seq):
        seen = [j for j in range(max(0, i - before), i + 1) if j != low[0]]
        nan[0, i] = bool(seen) and all(j in kept for j in seen)
    nan[1] = True
    assert nan[0].any() and not nan[0].all()
    assert torch.equal(torch.isnan(got), nan[:, :, None].expand_as(got))
    check_window(got[~nan], tuple(a[~nan] for a in ref), t)
    none = [0] if seq == 5 else []                               # row 0 of sequence 0 sees its masked self alone
    assert all(bool((got[0, i] == 0).all()) for i in none) and bool((got[2, seq // 2 + before:] == 0).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_whole_sequences_of_minus_infinity_are_nan(dim, t):
    """Without a window and a mask, where every row sees every key."""
    q, k, v, _ = window_inputs(dim, 1, 512, 2, 2, dim, None, t)
    q.abs_().add_(0.125)
    k[:, 0::dim] = -INF
    assert torch.isnan(window_attention(q, k, v, None, 1, 512, 2, 2, dim, 1000, 1000, 0, 0.125, t)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,window", [(2, 2, 64, 40), (8, 2, 128, 300), (16, 1, 64, 1000), (3, 1, 32, 17), (2, 1, 5, 33), (2, 2, 256, 40)])
def test_steps_that_see_only_scores_of_minus_infinity_are_nan(heads, kv_heads, dim, window, t):
    """A cache that overflowed must not come out as a plausible context. Stream 1 keeps every third key."""
    batch, sinks = 3, 2
    slots, g = window + sinks, gen(window)
    q, k, v = normal(g, batch, heads * dim, t=t).abs_().add_(0.125), normal(g, batch, kv_heads * dim, t=t), normal(g, batch, kv_heads * dim, t=t)
    kc, vc = normal(g, batch, kv_heads, slots, dim, t=t), normal(g, batch, kv_heads, slots, dim, t=t)
    k[0, 0::dim] = kc[0, :, :, 0] = -INF
    low = torch.arange(slots, device="cuda") % 3 != 0
    kc[1, :, low, 0] = -INF
    pos = torch.tensor([5 * slots, 7 * slots + 1, slots // 2], dtype=torch.int32, device="cuda")
    ctx = torch.zeros((batch, heads * dim), dtype=q.dtype, device="cuda")
    step(q, k, v, pos, batch, heads, kv_heads, dim, window, sinks, dim ** -0.5, kc, vc, ctx, t)
    assert torch.isnan(ctx[0]).all()
    seen = torch.ones((batch, slots), dtype=torch.bool, device="cuda")
    seen[2, slots // 2 + 1:] = False
    share = heads // kv_heads
    ref = attention64(q.reshape(batch, heads, 1, dim).double(), kc.double().repeat_interleave(share, 1), vc.double().repeat_interleave(share, 1),
                      seen[:, None, None, :], dim ** -0.5, dim)
    check_window(ctx[1:], tuple(a[1:] for a in ref), t)


# ============================================================================ K8: infinite values of little weight

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,window,batch", [(2, 2, 64, 40, 2), (8, 2, 128, 300, 2), (16, 1, 64, 1000, 2), (32, 2, 128, 500, 2),
                                                             (2, 2, 64, 3000, 2), (4, 4, 64, 200, 120), (3, 1, 32, 17, 2), (2, 1, 5, 33, 2)])
def test_step_infinite_value_whose_weight_binary16_cannot_hold(heads, kv_heads, dim, window, batch, t):
    """A weight of 2^-40 times infinity is infinity, in its own column alone; a NaN value is NaN there."""
    sinks = 1
    slots, g = window + sinks, gen(window + heads)
    q, k, v = normal(g, batch, heads * dim, t=t), normal(g, batch, kv_heads * dim, t=t), normal(g, batch, kv_heads * dim, t=t)
    kc, vc = normal(g, batch, kv_heads, slots, dim, t=t), normal(g, batch, kv_heads, slots, dim, t=t)
    scale = 1.0 / dim
    q.view(batch, heads, dim)[:, :, 0] = 4.0
    kc[:, :, :, 0], k.view(batch, kv_heads, dim)[:, :, 0] = 2.0, 2.0
    far = [3, slots - 2]                                         # their scores lie 28 below the others': a weight of 2^-40
    for j in far:
        kc[:, :, j] = 0
        kc[:, :, j, 0] = 2.0 - 7.0 * dim
    pos = torch.full((batch,), 10 * slots, dtype=torch.int32, device="cuda")
    at = sinks + (10 * slots - sinks) % window
    assert at not in far
    args = (batch, heads, kv_heads, dim, window, sinks, scale)
    kc[:, :, at], vc[:, :, at] = k.view(batch, kv_heads, dim), v.view(batch, kv_heads, dim)
    share = heads // kv_heads
    vc[:, :, far, 1], vc[0, :, far[1], 2] = 0, 0
    ref = attention64(q.reshape(batch, heads, 1, dim).double(), kc.double().repeat_interleave(share, 1), vc.double().repeat_interleave(share, 1),
                      torch.ones((batch, 1, 1, slots), dtype=torch.bool, device="cuda"), scale, dim)
    vc[:, :, far[0], 1] = INF
    vc[0, :, far[1], 2] = float("nan")
    ctx = torch.zeros((batch, heads * dim), dtype=q.dtype, device="cuda")
    step(q, k, v, pos, *args, kc, vc, ctx, t)
    got, odd = ctx.view(batch, heads, dim), torch.zeros((batch, heads, dim), dtype=torch.bool, device="cuda")
    assert bool((got[:, :, 1] == INF).all()) and torch.isnan(got[0, :, 2]).all()
    odd[:, :, 1] = True
    odd[0, :, 2] = True
    odd = odd.view(batch, -1)
    assert torch.isfinite(ctx[~odd]).all()
    check_window(ctx.masked_fill(odd, 0), tuple(a.masked_fill(odd, 0) for a in ref), t)


# ============================================================================ K8: many small weights

def small_weight_bar(want, count):
    # Weights of binary16 products are held 2^7 below the largest at the least, so one of them is off by 2^-32 of the largest or by
    # 2^-11 of itself; then the result, the sums (2^-23 for each 16 products) and the exponentials (arguments of up to 30: 2^-17).
    return count * 2.0 ** -32 + want * (2 * 2.0 ** -11 + (count / 16 + 64) * 2.0 ** -23 + 2.0 ** -16) + 2.0 ** -25


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_many_small_weights_are_not_lost(dim, t):
    """One key far above all others, whose value is 0; the others weigh 2^-25.5 each and together 2^-10 of a row."""
    seq = 40000
    q, k, v = (torch.zeros((seq, dim), dtype=G.TORCH_DTYPE[t], device="cuda") for _ in range(3))
    q[:, 0], k[0, 0], v[1:] = 4.0, 25.5 * math.log(2) / 4, 1.0
    got = window_attention(q, k, v, None, 1, seq, 1, 1, dim, seq, 0, 0, 1.0, t).double()
    w = math.exp(-4.0 * float(k[0, 0]))
    others = torch.arange(seq, dtype=torch.float64, device="cuda")
    want = (others * w / (1 + others * w))[:, None].expand_as(got)
    within(got, want, small_weight_bar(want, others[:, None]))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (4, 2, 128)])
def test_many_small_weights_of_a_step_are_not_lost(heads, kv_heads, dim, t):
    batch, slots = 440 // kv_heads, 20000
    dt = G.TORCH_DTYPE[t]
    kc, vc = torch.zeros((batch, kv_heads, slots, dim), dtype=dt, device="cuda"), torch.ones((batch, kv_heads, slots, dim), dtype=dt, device="cuda")
    q, k, v = torch.zeros((batch, heads * dim), dtype=dt, device="cuda"), torch.zeros((batch, kv_heads * dim), dtype=dt, device="cuda"), None
    v = torch.ones_like(k)
    q[:, 0::dim] = 4.0
    kc[:, :, 100, 0] = 25.5 * math.log(2) / 4
    vc[:, :, 100] = 0
    pos = torch.full((batch,), 3 * slots, dtype=torch.int32, device="cuda")
    ctx = torch.zeros((batch, heads * dim), dtype=dt, device="cuda")
    step(q, k, v, pos, batch, heads, kv_heads, dim, slots, 0, 1.0, kc, vc, ctx, t)
    w = (slots - 1) * math.exp(-4.0 * float(kc[0, 0, 100, 0]))
    want = torch.full_like(ctx, w / (1 + w), dtype=torch.float64)
    within(ctx, want, small_weight_bar(want, slots))


# ============================================================================ K7

@pytest.mark.parametrize("rows,k,n", [(1, 128, 16), (3, 1000, 77), (20, 300, 40)])
def test_w4_matvec_every_nan_stays_nan(rows, k, n):
    """A float32 is a NaN by any of its 23 bits, the low 16 among them."""
    g = gen(k)
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand((-(-k // 64), n), generator=g, device="cuda") + 0.5
    packed, x = pack(codes), normal(g, rows, k)
    clean = matvec(x, packed, scales, 64, n, None, "f32")
    for bits in (0x7f800001, 0xff800001 - 2 ** 32, 0x7f80ffff, 0x7fc00000, 0x7fffffff, -1):
        y = x.clone()
        y.view(torch.int32)[0, k // 2] = bits
        got = matvec(y, packed, scales, 64, n, None, "f32")
        assert torch.isnan(got[0]).all() and torch.equal(got[1:], clean[1:]), hex(bits)


# ============================================================================ K8: give-ups

@pytest.mark.parametrize("dim", [64, 128])
def test_window_attention_gives_up_no_wait(dim):
    """NaN rows from the inputs are not give-ups, and nothing else should be there to count."""
    before = kernels.window_give_ups()
    q, k, v, m = window_inputs(dim, 4, 2000, 6, 3, dim, "holes", "f16")
    args = (4, 2000, 6, 3, dim, 300, 20, 2, dim ** -0.5)
    check_window(window_attention(q, k, v, m, *args, "f16"), window64(q, k, v, m, *args), "f16")
    k[100] = float("nan")
    m[0, 100] = 1
    assert torch.isnan(window_attention(q, k, v, m, *args, "f16")).any()
    assert kernels.window_give_ups() == before == 0


# ============================================================================ K8: which kernel runs

@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (40, 2, 1), (128, 4, 2), (72, 3, 3)])
def test_binary16_sequences_on_16_byte_boundaries_run_on_the_tensor_cores(dim, heads, kv_heads):
    """Only there are weights rounded to binary16. Rows that start 2 bytes later go by the float32 pipes: the same up to what is rounded,
    but not bit by bit, which it would be if both took that way."""
    batch, seq = 2, 300
    q, k, v, m = window_inputs(dim, batch, seq, heads, kv_heads, dim, "holes", "f16")
    parts = [a.contiguous() for a in (q, k, v)]
    shifted = []
    for a in parts:
        room = torch.zeros(a.numel() + 8, dtype=a.dtype, device="cuda")
        shifted.append(room[1:1 + a.numel()].view(a.shape).copy_(a))
    assert all(a.data_ptr() % 16 == 0 for a in parts) and all(a.data_ptr() % 16 == 2 for a in shifted)
    args = (batch, seq, heads, kv_heads, dim, 70, 11, 2, dim ** -0.5)
    ctx, bar, pv, tiny = window64(*parts, m, *args)
    fast, slow = window_attention(*parts, m, *args, "f16"), window_attention(*shifted, m, *args, "f16")
    check_window(slow, (ctx, bar, pv, tiny), "f16")
    # both within the bar of the float32 steps; the weights' rounding on one side; the results' on both
    within(fast, slow.double(), 2 * bar + 2.0 ** -11 * pv * (1 + 2.0 ** -6) + tiny + 2 * (2.0 ** -11 * ctx.abs() + 2.0 ** -25) * (1 + 2.0 ** -8))
    assert not torch.equal(fast, slow)
    assert torch.equal(slow, window_attention(*shifted, m, *args, "f16"))


# ============================================================================ the same data by every path

def by_every_start(a):
    """`a` on a 16-byte boundary, and one element further."""
    out = []
    for shift in (0, 1):
        room = torch.zeros(a.numel() + 16, dtype=a.dtype, device="cuda")
        out.append(room[shift:shift + a.numel()].view(a.shape).copy_(a))
    return out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,ch", [(5, 64), (9, 1024), (3, 8192), (2, 16384)])
def test_rms_norm_by_every_path_agrees(rows, ch, t):
    """The sums of squares are added in another order: their error (as norm_bar has it) on both sides, and a rounding on both."""
    g = gen(rows + ch)
    x, gamma = normal(g, rows, ch, t=t), 1 + normal(g, ch, std=0.3, t=t)
    (xa, xb), (ga, gb) = by_every_start(x), by_every_start(gamma)
    (sum_a, a), (sum_b, b) = rms_norm(xa, None, ga, 1e-6, t), rms_norm(xb, None, gb, 1e-6, t)
    assert torch.equal(sum_a, sum_b)
    within(b, a, 2 * (HALF_STEP[t] + norm_bar(ch)) * a.double().abs() * (1 + 2.0 ** -8) + 2 * SMALLEST[t])
    for group in (0, 128):
        (_, ca, sa), (_, cb, sb) = rms_norm(xa, None, ga, 1e-6, t, e4m3=group), rms_norm(xb, None, gb, 1e-6, t, e4m3=group)
        within(sb, sa, 2 * (norm_bar(ch) + 2.0 ** -22) * sa.double().abs())
        # half a step of a code (2^-4, 2^-10 near 0) on both sides, and the values' own difference
        within(cb.float(), ca.float(), ca.double().abs() * (2 * 2.0 ** -4 * (1 + 2.0 ** -3) + 4 * norm_bar(ch)) + 2 * 2.0 ** -10 * (1 + 2.0 ** -8))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,window", [(2, 2, 64, 40), (8, 2, 128, 700), (3, 1, 32, 17)])
def test_steps_by_every_path_agree(heads, kv_heads, dim, window, t):
    batch, sinks = 3, 2
    slots, g = window + sinks, gen(window)
    q, k, v = normal(g, batch, heads * dim, t=t), normal(g, batch, kv_heads * dim, t=t), normal(g, batch, kv_heads * dim, t=t)
    caches = normal(g, batch, kv_heads, slots, dim, t=t), normal(g, batch, kv_heads, slots, dim, t=t)
    pos = torch.tensor([slots // 2, 3 * slots, -1], dtype=torch.int32, device="cuda")
    got = []
    for kc, vc in zip(*(by_every_start(c) for c in caches)):
        ctx = torch.zeros((batch, heads * dim), dtype=q.dtype, device="cuda")
        step(q, k, v, pos, batch, heads, kv_heads, dim, window, sinks, dim ** -0.5, kc, vc, ctx, t)
        got.append((ctx, kc, vc))
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2])
    seen = torch.ones((batch, slots), dtype=torch.bool, device="cuda")
    seen[0, slots // 2 + 1:] = False
    share = heads // kv_heads
    ctx, bar, pv, tiny = attention64(q.reshape(batch, heads, 1, dim).double(), got[0][1].double().repeat_interleave(share, 1),
                                     got[0][2].double().repeat_interleave(share, 1), seen[:, None, None, :], dim ** -0.5, dim)
    bar = 2 * bar + 2 * (HALF_STEP[t] * ctx.abs() + SMALLEST[t]) * (1 + 2.0 ** -8)
    if t == "f16":                                               # weights rounded on one side
        bar = bar + 2.0 ** -11 * pv * (1 + 2.0 ** -6) + tiny
    within(got[1][0][:2], got[0][0][:2].double(), bar[:2])


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (40, 2, 1), (128, 4, 2), (72, 3, 3)])
@pytest.mark.parametrize("shift,pad", [(1, 0), (0, 1), (8, 4), (2, 6)])
def test_tensor_core_sequences_into_a_context_of_any_alignment(dim, heads, kv_heads, shift, pad):
    """Operands on 16-byte boundaries, a context that starts or whose rows start elsewhere: the same bits, and nothing beside them."""
    batch, seq = 2, 300
    q, k, v, m = window_inputs(dim, batch, seq, heads, kv_heads, dim, "holes", "f16")
    q, k, v = (a.contiguous() for a in (q, k, v))
    args = (batch, seq, heads, kv_heads, dim, 70, 11, 2, dim ** -0.5)
    want = window_attention(q, k, v, m, *args, "f16")
    wide = heads * dim + pad
    room = torch.full((batch * seq * wide + 16,), 3.0, dtype=torch.float16, device="cuda")
    ctx = room[shift:shift + batch * seq * wide].view(batch * seq, wide)
    window_attention(q, k, v, m, *args, "f16", ctx=ctx[:, :heads * dim])
    assert torch.equal(ctx[:, :heads * dim], want) and bool((ctx[:, heads * dim:] == 3).all())
    assert bool((room[:shift] == 3).all() and (room[shift + batch * seq * wide:] == 3).all())


# ============================================================================ K8: bits of a weight

@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (16, 1, 64), (32, 2, 128)])
def test_step_weights_keep_22_bits(heads, kv_heads, dim):
    """Few keys whose values nearly cancel: the context is small beside its terms, and so is its own rounding beside that of a weight
    held in 11 bits. Scores are one product each."""
    batch, slots, g = 64, 6, gen(dim + heads)
    q = torch.zeros((batch, heads * dim), dtype=torch.float16, device="cuda")
    q[:, 0::dim] = 1.0
    k, v = torch.zeros((batch, kv_heads * dim), dtype=torch.float16, device="cuda"), normal(g, batch, kv_heads * dim, t="f16")
    kc, vc = torch.zeros((batch, kv_heads, slots, dim), dtype=torch.float16, device="cuda"), normal(g, batch, kv_heads, slots, dim, t="f16")
    kc[..., 0] = torch.rand((batch, kv_heads, slots), generator=g, device="cuda").half()
    pos = torch.full((batch,), 4 * slots + 1, dtype=torch.int32, device="cuda")
    ctx = torch.zeros((batch, heads * dim), dtype=torch.float16, device="cuda")
    step(q, k, v, pos, batch, heads, kv_heads, dim, slots, 0, 1.0, kc, vc, ctx, "f16")
    share = heads // kv_heads
    want, bar, pv, _ = attention64(q.reshape(batch, heads, 1, dim).double(), kc.double().repeat_interleave(share, 1),
                                   vc.double().repeat_interleave(share, 1), torch.ones((batch, 1, 1, slots), dtype=torch.bool, device="cuda"), 1.0, dim)
    # two binary16 parts of a weight: half a step of the second is 2^-22 of it at most; then the result's rounding
    within(ctx, want, bar + 2.0 ** -22 * pv + 2.0 ** -11 * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -25)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad", [0, 1])
def test_long_rows_of_minus_infinity_and_of_nothing(pad, t):
    """Three keys of 9000: one whose score is minus infinity, then one that is not."""
    seq, dim = 9000, 64
    q, k, v, _ = window_inputs(17, 1, seq, 1, 1, dim, None, t, pad)
    q.abs_().add_(0.125)
    k[5, 0] = -INF
    m = torch.zeros((1, seq), dtype=torch.int8, device="cuda")
    m[0, [5, 4600, 8901]] = 1
    got = window_attention(q, k, v, m, 1, seq, 1, 1, dim, seq, 0, 0, dim ** -0.5, t)
    assert bool((got[:5] == 0).all()) and torch.isnan(got[5:4600]).all()
    assert torch.equal(got[4600:8901], v[4600:4601].expand(4301, dim))
    s = q[8901:].double() @ k[[4600, 8901]].double().t() * dim ** -0.5
    want, pv = torch.softmax(s, 1) @ v[[4600, 8901]].double(), torch.softmax(s, 1) @ v[[4600, 8901]].double().abs()
    # scores of up to 64 (72 steps of float32), the exponential, then weights and result in binary16 at the most
    half = 2.0 ** -11 if t == "f16" else 2.0 ** -24
    within(got[8901:], want, pv * (2 * 64 * 72 * 2.0 ** -23 + 2.0 ** -18 + half * (1 + 2.0 ** -6)) + half * want.abs() + 2.0 ** -25)
