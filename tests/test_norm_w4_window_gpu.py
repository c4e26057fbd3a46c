"""K6 (residual + RMS norm), K7 (products with 4-bit weights) and K8 (sliding-window attention) against plain
float64 forms of the same definitions, and a decoding layer made of the three.

Bars, in units of what can be rounded: half a step is 2^-24 (float32), 2^-11 (binary16) or 2^-4 (e4m3) of a value;
binary16 and e4m3 numbers below their normal range are off by up to 2^-25 and 2^-10. A float32 sum of n terms is off
by at most n 2^-24 of the sum of their magnitudes, a sum on the tensor cores by 2^-23 per product it takes in (their
additions may cut instead of round).
"""
import math
import os
import random
import subprocess
import sys

import numpy as np
import pytest
import torch

import gpu_harness as G
from cubert_b200 import kernels

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16"]
F8 = torch.float8_e4m3fn
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
SMALLEST = {"f32": 0.0, "f16": 2.0 ** -25}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0, t="f32"):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(G.TORCH_DTYPE[t])


def within(got, want, bound, what=""):
    """|got - want| <= bound, elementwise, in float64; NaN exactly where `want` is NaN."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    bad = ~((got - want).abs() <= bound) & ~torch.isnan(want)
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError("%s: %d of %d outside the bound; first at %s: got %r want %r" % (
            what, int(bad.sum()), bad.numel(), at, got[tuple(at)].item(), want[tuple(at)].item()))


def banded(t):
    """A copy of `t` between two bands of a sentinel, and a check that the bands still hold it. The copy's alignment is t's."""
    raw = torch.empty(t.numel() * t.element_size() + 512, dtype=torch.uint8, device="cuda").fill_(0x5A)
    body = raw[256:256 + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    body.copy_(t)
    return body, lambda: bool((raw[:256] == 0x5A).all() and (raw[256 + t.numel() * t.element_size():] == 0x5A).all())


# ============================================================================ K6

def rms_norm(x, r, gamma, eps, t, sum_=True, e4m3=None, total=None, out=None):
    rows, ch = x.shape
    total = torch.empty_like(x) if total is None and sum_ else total
    if e4m3 is None:
        out = torch.empty_like(x) if out is None else out
        kernels.check(G.fn("residual_rms_norm", t)(G.ptr(x), G.ptr(r), G.ptr(gamma), rows, ch, eps, G.ptr(total), G.ptr(out), G.stream()))
        return total, out
    codes = torch.full((rows, ch), 0x55, dtype=torch.uint8, device="cuda").view(F8)
    scales = torch.full((rows, -(-ch // e4m3) if e4m3 else 1), -1.0, device="cuda")
    kernels.check(G.fn("residual_rms_norm_e4m3", t)(G.ptr(x), G.ptr(r), G.ptr(gamma), rows, ch, eps, e4m3, G.ptr(total), G.ptr(codes),
                                                    G.ptr(scales), G.stream()))
    return total, codes, scales


def norm64(x, r, gamma, eps):
    t = x.double() + (0 if r is None else r.double())
    return t, t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * gamma.double()


def norm_bar(ch):
    # t once; the mean of squares: chains of at most ch / 32 additions and a tree, halved by the root; root, quotient, two products
    return (ch / 64 + 12) * 2.0 ** -24


NORM_SHAPES = [(1, 1), (3, 7), (1, 768), (2, 8), (5, 1024), (33, 1004), (129, 128), (4, 4096), (2, 8192), (3, 8200), (7, 130), (1, 20011),
               (700, 64), (2500, 256), (301, 2048), (6, 5120)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,ch", NORM_SHAPES)
def test_rms_norm(rows, ch, residual, t):
    g = gen(rows * 10007 + ch)
    x, gamma = normal(g, rows, ch, t=t), 1 + normal(g, ch, std=0.3, t=t)
    r = normal(g, rows, ch, std=3.0, t=t) if residual else None
    total, out = rms_norm(x, r, gamma, 1e-6, t)
    t64, y64 = norm64(x, r, gamma, 1e-6)
    within(total, t64, HALF_STEP[t] * t64.abs() + SMALLEST[t], "sum")
    within(out, y64, (HALF_STEP[t] + norm_bar(ch)) * y64.abs() * (1 + 2.0 ** -8) + SMALLEST[t], "out")
    _, again = rms_norm(x, r, gamma, 1e-6, t, sum_=False)      # without the sum: the same output
    assert torch.equal(again, out)
    total2, out2 = rms_norm(x.clone(), r, gamma, 1e-6, t, total=(xc := x.clone()))  # sum in a buffer that starts as x
    assert torch.equal(total2, total) and torch.equal(out2, out) and total2 is xc


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("rows,ch", NORM_SHAPES)
def test_rms_norm_e4m3(rows, ch, group, t):
    g = gen(rows * 31 + ch + group)
    x, gamma, r = normal(g, rows, ch, t=t), 1 + normal(g, ch, std=0.3, t=t), normal(g, rows, ch, t=t)
    x[0] = 0
    r[0] = 0                                                    # a row of zeros: scale 0, codes 0
    total, codes, scales = rms_norm(x, r, gamma, 1e-6, t, e4m3=group)
    t64, y64 = norm64(x, r, gamma, 1e-6)
    within(total, t64, HALF_STEP[t] * t64.abs() + SMALLEST[t], "sum")
    want = torch.stack([p.abs().amax(1) / 448 for p in y64.split(group or ch, 1)], 1)
    bar = norm_bar(ch)
    within(scales, want, (bar + 2.0 ** -22) * want, "scales")
    assert float(scales[0].abs().max()) == 0 and float(codes[0].float().abs().max()) == 0
    v = y64 / want.repeat_interleave(group or ch, 1)[:, :ch].clamp(min=1e-300)
    within(codes.float(), v, v.abs() * (2.0 ** -4 * (1 + 2.0 ** -10) + 2 * bar) + 2.0 ** -10 * (1 + 2.0 ** -10), "codes")
    assert float(codes[1:].float().abs().max() if rows > 1 else 448) == 448


@pytest.mark.parametrize("t", TYPES)
def test_rms_norm_in_place_and_unaligned(t):
    g = gen(5)
    for rows, ch, shift in ((37, 768, 0), (37, 768, 1), (5, 1001, 3)):
        raw = normal(g, 2, rows * ch + 8, t=t)
        x, r = raw[0, shift:shift + rows * ch].view(rows, ch), raw[1, shift:shift + rows * ch].view(rows, ch)
        gamma = normal(g, ch + 8, t=t)[shift:shift + ch]
        total, out = rms_norm(x, r, gamma, 1e-5, t)
        xs, rs = x.clone(), r.clone()
        rms_norm(x, r, gamma, 1e-5, t, total=r, out=x)          # the residual stream and the row updated where they are
        assert torch.equal(r, total) and torch.equal(x, out)
        x.copy_(xs), r.copy_(rs)
        rms_norm(x, r, gamma, 1e-5, t, total=x, out=r)
        assert torch.equal(x, total) and torch.equal(r, out)


@pytest.mark.parametrize("t", TYPES)
def test_rms_norm_not_finite_rows_stay_in_their_rows(t):
    g = gen(6)
    for ch in (768, 777):
        x, gamma = normal(g, 6, ch, t=t), normal(g, ch, t=t)
        x[1, 5], x[3, 700] = float("nan"), float("inf")
        total, out = rms_norm(x, None, gamma, 1e-6, t)
        _, y64 = norm64(x, None, gamma, 1e-6)
        within(out, y64, (HALF_STEP[t] + norm_bar(ch)) * y64.abs() * (1 + 2.0 ** -8) + SMALLEST[t])
        assert torch.equal(torch.isnan(total), torch.isnan(x))
        _, codes, scales = rms_norm(x, None, gamma, 1e-6, t, e4m3=128)
        nan = torch.isnan(codes.float())
        assert nan[1].all() and torch.isnan(scales[1]).all()                                   # a NaN spoils its row
        assert nan[3, 640:768].all() and torch.isnan(scales[3, 5:6]).all() and not nan[3, :640].any()   # an infinity its block: 0 elsewhere
        assert not nan[[0, 2, 4, 5]].any() and not torch.isnan(scales[[0, 2, 4, 5]]).any()


@pytest.mark.parametrize("t", TYPES)
def test_rms_norm_stays_inside_its_buffers(t):
    g = gen(7)
    for rows, ch in ((1, 768), (3, 1004), (65, 1024), (9, 77)):
        x, gamma = normal(g, rows, ch, t=t), normal(g, ch, t=t)
        for e4m3 in (None, 0, 128):
            bx, ok_x = banded(x)
            total, ok_total = banded(x)
            if e4m3 is None:
                out, ok_out = banded(x)
                rms_norm(bx, None, gamma, 1e-6, t, total=total, out=out)
            else:
                codes, ok_out = banded(torch.zeros((rows, ch), dtype=torch.uint8, device="cuda"))
                scales, ok_s = banded(torch.zeros((rows, -(-ch // 128) if e4m3 else 1), device="cuda"))
                kernels.check(G.fn("residual_rms_norm_e4m3", t)(G.ptr(bx), None, G.ptr(gamma), rows, ch, 1e-6, e4m3, G.ptr(total),
                                                                G.ptr(codes), G.ptr(scales), G.stream()))
                assert ok_s()
            assert ok_x() and ok_total() and ok_out() and torch.equal(bx, x)


# ============================================================================ K7

def pack(codes):
    n, k = codes.shape
    packed = torch.full((kernels.load().cubk_w4_packed_bytes(n, k),), 0x33, dtype=torch.uint8, device="cuda")
    kernels.check(kernels.load().cubk_w4_pack(G.ptr(codes), n, k, G.ptr(packed), G.stream()))
    return packed


def unpack(packed, n, k):
    """The documented layout read back on the host, one address formula per element."""
    p = packed.cpu().numpy()
    kb = -(-k // 128)
    rows, cols = np.arange(-(-n // 16) * 16)[:, None], np.arange(kb * 128)[None, :]
    c = cols % 128
    word = ((rows // 16) * kb + cols // 128) * 256 + (rows % 16) * 16 + 4 * (c % 32 // 8) + c // 32
    bit = (c % 2) * 16 + 4 * (c % 8 // 2)
    return ((p.view("<u4")[word] >> bit.astype(np.uint32)) & 15).astype(np.int64) - 8


def matvec(x, packed, scales, group, n, bias, t, xs=None, code_group=0, out=None):
    rows, k = x.shape
    out = torch.full((rows, n), float("nan"), dtype=G.TORCH_DTYPE[t], device="cuda") if out is None else out
    if xs is None:
        kernels.check(G.fn("w4_matvec", t)(G.ptr(x), rows, k, G.ptr(packed), G.ptr(scales), group, n, G.ptr(bias), G.ptr(out), G.stream()))
    else:
        kernels.check(G.fn("w4_matvec_e4m3", t)(G.ptr(x), G.ptr(xs), code_group, rows, k, G.ptr(packed), G.ptr(scales), group, n, G.ptr(bias),
                                                G.ptr(out), G.stream()))
    return out


def check_matvec(got, x64, codes, scales, group, bias, t, what=""):
    k = codes.shape[1]
    w = codes.double() * scales.double().repeat_interleave(group, 0)[:k].t()
    want = x64 @ w.t() + (0 if bias is None else bias.double())
    size = x64.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    # products of 16 columns, three for float32; then scales, joins of the warps, bias
    bar = (3 * math.ceil(k / 16) + 24) * 2.0 ** -23
    within(got, want, HALF_STEP[t] * want.abs() + SMALLEST[t] + bar * size, what)
    if t == "f32" and want.numel() > 100:
        # the same errors as a random walk: sqrt(3 k / 16) 2^-23 of a result, and slack of two
        rms = float((got.double() - want).square().mean().sqrt() / want.square().mean().sqrt())
        assert rms <= 2 * math.sqrt(3 * k / 16 + 24) * 2.0 ** -23, rms


W4_SHAPES = [(1, 128, 16), (1, 768, 2304), (8, 1024, 1000), (3, 1000, 777), (2, 1, 1), (5, 37, 17), (9, 512, 100), (16, 4096, 64), (17, 768, 33),
             (33, 200, 50), (64, 1024, 256), (70, 640, 48), (1, 8192, 96), (4, 2056, 4096), (130, 96, 16),
             (24, 6144, 139), (64, 3272, 1201), (16, 8192, 2500), (40, 12300, 800), (2401, 64, 40)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,k,n", W4_SHAPES)
def test_w4_matvec(rows, k, n, group, t):
    g = gen(rows + 7 * k + 13 * n + group)
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = (torch.rand((-(-k // group), n), generator=g, device="cuda") * 0.1 + 0.01).to(G.TORCH_DTYPE[t])
    packed = pack(codes)
    x = normal(g, rows, k, t=t)
    bias = normal(g, n, t=t)
    check_matvec(matvec(x, packed, scales, group, n, bias, t), x.double(), codes, scales, group, bias, t)
    one = matvec(x, packed, scales, group, n, None, t)
    check_matvec(one, x.double(), codes, scales, group, None, t)
    assert torch.equal(one, matvec(x, packed, scales, group, n, None, t))      # the same bits every time


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("code_group", [0, 128])
@pytest.mark.parametrize("rows,k,n", W4_SHAPES)
def test_w4_matvec_e4m3(rows, k, n, code_group, t):
    g = gen(rows + 7 * k + 13 * n + code_group)
    group = (32, 64, 128)[(rows + k) % 3]
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = (torch.rand((-(-k // group), n), generator=g, device="cuda") * 0.1 + 0.01).to(G.TORCH_DTYPE[t])
    x = normal(g, rows, k, std=60).to(F8)
    xs = torch.rand((rows, -(-k // 128) if code_group else 1), generator=g, device="cuda") * 0.01
    x64 = x.float().double() * xs.double().repeat_interleave(code_group or k, 1)[:, :k]
    check_matvec(matvec(x, pack(codes), scales, group, n, None, t, xs, code_group), x64, codes, scales, group, None, t)


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (100, 1000), (33, 640)])
def test_w4_pack_and_quantize_write_the_documented_layout(n, k):
    g = gen(n + k)
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    got = unpack(pack(codes), n, k)
    assert np.array_equal(got[:n, :k], codes.cpu().numpy()) and not got[n:].any() and not got[:, k:].any()
    for t in TYPES:
        for group in (32, 64, 128):
            w = normal(g, n, k, std=0.02, t=t)
            w[:, : min(k, group)] = 0                            # a group of zeros
            if n > 2:
                w[1] = 0
            packed = torch.empty(kernels.load().cubk_w4_packed_bytes(n, k), dtype=torch.uint8, device="cuda")
            scales = torch.full((-(-k // group), n), float("nan"), dtype=w.dtype, device="cuda")
            kernels.check(G.fn("w4_quantize", t)(G.ptr(w), n, k, group, G.ptr(packed), G.ptr(scales), G.stream()))
            top = torch.stack([p.float().abs().amax(1) for p in w.split(group, 1)])
            want = (top / torch.full_like(top, 7)).to(w.dtype)   # a quotient: torch multiplies by 1 / 7 for a plain number
            assert torch.equal(scales, want)
            s = want.double().repeat_interleave(group, 0)[:k].t()
            q = unpack(packed, n, k)
            assert not q[n:].any() and not q[:, k:].any()
            q = torch.from_numpy(q[:n, :k]).cuda().double()
            # half a code, and where the scale was rounded down the largest weight may lie half a step past code 7
            assert bool(((q * s - w.double()).abs() <= s * (0.5 + 7.5 * HALF_STEP[t] + 2.0 ** -20)).all())


@pytest.mark.parametrize("t", TYPES)
def test_w4_matvec_not_finite_rows_and_buffers(t):
    g = gen(11)
    n, k, rows = 53, 300, 9
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = (torch.rand((-(-k // 64), n), generator=g, device="cuda") + 0.5).to(G.TORCH_DTYPE[t])
    packed = pack(codes)
    x = normal(g, rows, k, t=t)
    clean = matvec(x, packed, scales, 64, n, None, t)
    x[4, 17] = float("nan")
    x[8, 299] = float("inf")
    bx, ok_x = banded(x)
    out, ok_out = banded(torch.zeros((rows, n), dtype=x.dtype, device="cuda"))
    bp, ok_p = banded(packed)
    matvec(bx, bp, scales, 64, n, None, t, out=out)
    keep = [r for r in range(rows) if r not in (4, 8)]
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[4]).all()
    zero = codes[:, 299] == 0
    assert torch.isnan(out[8][zero]).all() and not torch.isfinite(out[8]).any()
    assert ok_x() and ok_out() and ok_p()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_quantize_keeps_nan_and_infinities(group, t):
    """A weight that is not finite must not come out as a plausible code: its group's products are NaN, the others what they were."""
    g = gen(group)
    n, k, rows = 37, 300, 3
    w = normal(g, n, k, std=0.02, t=t)
    x = normal(g, rows, k, t=t)
    hit = {(2, 5): float("nan"), (17, 299): float("inf"), (36, 130): float("-inf"), (20, 0): float("nan")}

    def quantized():
        packed = torch.empty(kernels.load().cubk_w4_packed_bytes(n, k), dtype=torch.uint8, device="cuda")
        scales = torch.zeros((-(-k // group), n), dtype=w.dtype, device="cuda")
        kernels.check(G.fn("w4_quantize", t)(G.ptr(w), n, k, group, G.ptr(packed), G.ptr(scales), G.stream()))
        return packed, scales

    packed, scales = quantized()
    clean, clean_codes = matvec(x, packed, scales, group, n, None, t), unpack(packed, n, k)[:n, :k]
    for (r, c), v in hit.items():
        w[r, c] = v
    packed, got = quantized()
    codes = unpack(packed, n, k)[:n, :k]
    same = np.ones((n, k), bool)
    for (r, c), v in hit.items():
        first = c // group * group
        assert not torch.isfinite(got[c // group, r]) and torch.isnan(got[c // group, r]).item() == math.isnan(v)
        assert not codes[r, first:first + group].any()
        got[c // group, r] = scales[c // group, r]
        same[r, first:first + group] = False
    assert torch.equal(got, scales) and np.array_equal(codes[same], clean_codes[same])
    packed, scales = quantized()
    out = matvec(x, packed, scales, group, n, None, t)
    rest = [r for r in range(n) if r not in {r for r, _ in hit}]
    assert torch.isnan(out[:, sorted({r for r, _ in hit})]).all() and torch.equal(out[:, rest], clean[:, rest])


# ============================================================================ K8

def window_attention(q, k, v, mask, batch, seq, heads, kv_heads, dim, before, after, sinks, scale, t, ctx=None):
    if ctx is None:
        ctx = torch.full((batch * seq, heads * dim), float("nan"), dtype=q.dtype, device="cuda")
    kernels.check(G.fn("window_attention", t)(G.ptr(q), G.ptr(k), G.ptr(v), q.stride(0), k.stride(0), G.ptr(mask), batch, seq, heads, kv_heads,
                                              dim, before, after, sinks, scale, G.ptr(ctx), ctx.stride(0), G.stream()))
    return ctx


def window64(q, k, v, mask, batch, seq, heads, kv_heads, dim, before, after, sinks, scale):
    """(context, bound of its error for float32 storage, sum of p |v|, visible keys), float64."""
    q = q.reshape(batch, seq, heads, dim).permute(0, 2, 1, 3).double()
    k = k.reshape(batch, seq, kv_heads, dim).permute(0, 2, 1, 3).double().repeat_interleave(heads // kv_heads, 1)
    v = v.reshape(batch, seq, kv_heads, dim).permute(0, 2, 1, 3).double().repeat_interleave(heads // kv_heads, 1)
    i = torch.arange(seq, device="cuda")
    seen = (i[None, :] <= i[:, None] + after) & ((i[None, :] >= i[:, None] - before) | (i[None, :] < sinks))
    seen = seen[None].expand(batch, seq, seq)
    if mask is not None:
        seen = seen & (mask != 0)[:, None, :]
    return attention64(q, k, v, seen[:, None], scale, dim)


def attention64(q, k, v, seen, scale, dim):
    s = q @ k.transpose(2, 3) * scale
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(3, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(s))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    finite_v = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
    ctx = p @ finite_v
    pv = p @ finite_v.abs()
    count = seen.sum(3, keepdim=True).double()
    qk = torch.nan_to_num(q.abs(), nan=0.0, posinf=0.0) @ torch.nan_to_num(k.abs(), nan=0.0, posinf=0.0).transpose(2, 3)
    delta = torch.where(seen, qk, torch.zeros_like(qk)).amax(3, keepdim=True) * abs(scale) * (dim + 8) * 2.0 ** -23
    # a weight: its score's error, two steps of the exponential and of its argument; then the sums over the visible keys
    eps = 2 * (delta + 2.0 ** -20 + (count + 16) * 2.0 ** -23)
    def rows(a):
        return a.permute(0, 2, 1, 3).reshape(a.shape[0] * a.shape[2], -1)
    vtop = finite_v.abs().amax()
    return rows(ctx), rows(eps * pv), rows(pv), rows((count * 2.0 ** -25 * vtop).expand_as(pv))


def check_window(got, ref, t, what=""):
    ctx, bar, pv, tiny = ref
    if t == "f16":   # weights rounded to binary16 (below their normal range: 2^-25 of the largest each), and the result
        bar = bar + 2.0 ** -11 * pv * (1 + 2.0 ** -6) + tiny + 2.0 ** -11 * ctx.abs() + 2.0 ** -25
    else:
        bar = bar + 2.0 ** -24 * ctx.abs() + 1e-37
    within(got, ctx, bar, what)


# batch, seq, heads, kv_heads, dim, before, after, sinks, mask
WINDOWS = [
    (1, 1, 1, 1, 64, 0, 0, 0, None),
    (2, 5, 3, 1, 64, 2, 0, 1, None),
    (2, 33, 4, 4, 32, 7, 3, 0, "holes"),
    (1, 127, 2, 2, 64, 0, 0, 2, None),
    (2, 128, 4, 2, 64, 1000, 1000, 0, "prefix"),
    (1, 129, 6, 2, 128, 64, 64, 4, "holes"),
    (3, 200, 4, 1, 64, 50, 0, 4, "prefix"),
    (1, 300, 2, 2, 128, 2000000000, 2000000000, 0, None),
    (2, 333, 2, 1, 64, 17, 200, 150, "holes"),
    (1, 515, 8, 2, 128, 300, 0, 17, None),
    (2, 640, 3, 3, 64, 128, 127, 1, "prefix"),
    (1, 1000, 2, 2, 64, 255, 0, 500, "holes"),
    (1, 1537, 4, 4, 32, 300, 100, 4, None),
    (2, 70, 2, 2, 5, 10, 10, 1, "holes"),
    (1, 40, 2, 1, 256, 9, 0, 2, None),
    (2, 64, 2, 2, 96, 16, 16, 1, "prefix"),
    (1, 2049, 2, 1, 64, 700, 0, 4, None),
    (1, 1, 2, 2, 128, 5, 5, 5, "none kept"),
    (3, 6, 4, 2, 64, 2, 1, 1, "holes"),
    (70, 7, 4, 2, 128, 4, 0, 2, "prefix"),
    (5, 12, 3, 1, 64, 5, 2, 3, "holes"),
    (300, 12, 2, 2, 32, 100, 0, 0, "prefix"),
    (2, 13, 6, 3, 128, 6, 6, 1, "holes"),
    (1000, 2, 12, 12, 64, 1, 0, 0, "prefix"),
    (2, 260, 2, 2, 64, 40, 3, 0, "none kept"),
]


def window_inputs(seed, batch, seq, heads, kv_heads, dim, mask, t, pad=0):
    g = gen(seed)
    qkv = normal(g, batch * seq, (heads + 2 * kv_heads) * dim + pad, t=t)
    q, k, v = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv_heads) * dim], qkv[:, (heads + kv_heads) * dim:(heads + 2 * kv_heads) * dim]
    m = None
    if mask == "prefix":
        m = (torch.arange(seq, device="cuda")[None] < torch.randint(1, seq + 1, (batch, 1), generator=g, device="cuda")).to(torch.int8)
    elif mask == "holes":
        m = (torch.rand((batch, seq), generator=g, device="cuda") < 0.5).to(torch.int8)
        m[0, : seq // 2] = 0
    elif mask == "none kept":
        m = torch.zeros((batch, seq), dtype=torch.int8, device="cuda")
    if m is not None:
        m = m * 3                                                 # any non-zero byte keeps a key
    return q, k, v, m


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,seq,heads,kv_heads,dim,before,after,sinks,mask", WINDOWS)
def test_window_attention(batch, seq, heads, kv_heads, dim, before, after, sinks, mask, t):
    q, k, v, m = window_inputs(seq + heads, batch, seq, heads, kv_heads, dim, mask, t)
    args = (batch, seq, heads, kv_heads, dim, before, after, sinks, dim ** -0.5)
    got = window_attention(q, k, v, m, *args, t)
    check_window(got, window64(q, k, v, m, *args), t)
    assert torch.equal(got, window_attention(q, k, v, m, *args, t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad,dim", [(0, 64), (1, 64), (2, 64), (8, 64), (8, 128), (3, 32), (4, 128)])
def test_window_attention_strides_and_alignment(pad, dim, t):
    """Rows further apart than they are long (odd distances too), each operand from its own tensor, a strided context
    whose gaps keep their contents."""
    batch, seq, heads, kv_heads = 2, 150, 4, 2
    q, _, _, m = window_inputs(3, batch, seq, heads, kv_heads, dim, "holes", t, pad)
    _, k, v, _ = window_inputs(4, batch, seq, heads, kv_heads, dim, None, t, pad)
    args = (batch, seq, heads, kv_heads, dim, 60, 20, 3, 0.3)
    wide = torch.full((batch * seq, heads * dim + pad), 3.0, dtype=q.dtype, device="cuda")
    got = window_attention(q, k, v, m, *args, t, ctx=wide[:, :heads * dim])
    check_window(got, window64(q, k, v, m, *args), t)
    assert bool((wide[:, heads * dim:] == 3).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128, 48])
def test_window_attention_keys_out_of_sight_may_hold_anything(dim, t):
    """NaN and infinities in masked keys and values, and in visible-to-others ones: only the queries that see them notice."""
    batch, seq, heads = 2, 400, 2
    q, k, v, m = window_inputs(9, batch, seq, heads, heads, dim, "holes", t)
    q, k, v = q.clone(), k.clone(), v.clone()
    args = (batch, seq, heads, heads, dim, 33, 9, 2, 0.2)
    ref = window64(q, k, v, m, *args)
    check_window(window_attention(q, k, v, m, *args, t), ref, t)
    off = (m == 0).reshape(-1)
    k[off], v[off] = float("nan"), float("inf")
    v[off.nonzero()[::3, 0]] = float("nan")
    check_window(window_attention(q, k, v, m, *args, t), ref, t, "masked keys")
    # a kept key in the middle of sequence 1: rows 300 - 9 .. 300 + 33 see it
    m[1, 300] = 1
    ref = window64(q, k, v, m, *args)
    v[seq + 300] = float("nan")
    k[seq + 300] = 0
    got = window_attention(q, k, v, m, *args, t)
    sees = torch.zeros(batch * seq, dtype=torch.bool, device="cuda")
    sees[seq + 291:seq + 334] = True
    assert torch.isnan(got[sees]).all()
    check_window(got[~sees], tuple(a[~sees] for a in ref), t, "rows that do not see the key")
    k[seq + 300] = float("nan")
    got = window_attention(q, k, v, m, *args, t)
    assert torch.isnan(got[sees]).all()
    check_window(got[~sees], tuple(a[~sees] for a in ref), t, "NaN keys")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("seq,dim", [(16, 64), (256, 64), (1296, 64), (1296, 128), (1300, 128), (1301, 64)])
@pytest.mark.parametrize("before,after,sinks", [(101, 7, 3), (300, 0, 140), (5000, 5000, 0)])
def test_window_attention_masks_of_any_alignment_and_byte(seq, dim, before, after, sinks, t):
    """Any byte but 0 keeps a key, wherever the mask starts; long runs of masked keys between."""
    batch, heads = 2, 2
    q, k, v, _ = window_inputs(seq + dim, batch, seq, heads, heads, dim, None, t)
    g = gen(seq)
    values = torch.tensor([0, 1, -1, -128, 127, 64, 2, 0], dtype=torch.int8, device="cuda")
    m = values[torch.randint(0, 8, (batch, seq), generator=g, device="cuda")]
    m[1, 200:700] = 0
    args = (batch, seq, heads, heads, dim, before, after, sinks, dim ** -0.5)
    got = None
    for shift in (0, 1, 4, 8, 16):
        room = torch.full((batch * seq + 64,), 77, dtype=torch.int8, device="cuda")
        here = room[shift:shift + batch * seq].view(batch, seq)
        here.copy_(m)
        out = window_attention(q, k, v, here, *args, t)
        if got is None:
            check_window(out, window64(q, k, v, m, *args), t)
        assert got is None or torch.equal(out, got)
        got = out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim,kv_heads", [(64, 12), (128, 6), (128, 12)])
def test_window_attention_not_finite_values_among_many_items(dim, kv_heads, t):
    """One column of one kept value is NaN in every other sequence, and padding holds anything: rows that see the key have NaN in that
    column alone, the others and the other sequences what they had, however many items a block works through."""
    batch, seq, heads = 4, 1300, 12
    q, k, v, m = window_inputs(77 + dim, batch, seq, heads, kv_heads, dim, None, t)
    q, k, v = q.clone(), k.clone(), v.clone()
    m = torch.ones((batch, seq), dtype=torch.int8, device="cuda")
    for b, length in enumerate((1300, 1211, 640, 77)):
        m[b, length:] = 0
    args = (batch, seq, heads, kv_heads, dim, 200, 0, 3, dim ** -0.5)
    off = (m == 0).reshape(-1)
    k[off], v[off] = 0, 0
    clean = window_attention(q, k, v, m, *args, t)
    k[off], v[off] = float("nan"), float("inf")
    assert torch.equal(clean, window_attention(q, k, v, m, *args, t))
    hit = {1: 600, 3: 50}
    for b, j in hit.items():
        v[b * seq + j, dim - 3::dim] = 0
    ref = window64(q, k, v, m, *args)
    for b, j in hit.items():
        v[b * seq + j, dim - 3::dim] = float("nan")
    got = window_attention(q, k, v, m, *args, t)
    nan = torch.zeros((batch, seq, heads, dim), dtype=torch.bool, device="cuda")
    for b, j in hit.items():
        nan[b, j:j + 201, :, dim - 3] = True
    nan = nan.reshape(batch * seq, heads * dim)
    assert torch.equal(torch.isnan(got), nan)
    check_window(got.masked_fill(nan, 0), tuple(a.masked_fill(nan, 0) for a in ref), t)
    same = torch.ones((batch, seq), dtype=torch.bool, device="cuda")
    same[1, 600 // 128 * 128:] = False
    same[3] = False
    assert torch.equal(got[same.reshape(-1)], clean[same.reshape(-1)])


@pytest.mark.parametrize("dim", [64, 128])
def test_window_attention_long_rows_computed_again_leave_the_others_alone(dim):
    """A NaN in a value that every later token sees: many long rows are computed again, and no wait for them runs out."""
    batch, seq, heads, key = 2, 40000, 2, 100
    g = gen(dim)
    q, k, v = (normal(g, batch * seq, heads * dim, t="f16") for _ in range(3))
    args = (batch, seq, heads, heads, dim, seq, 0, 0, dim ** -0.5)
    clean = window_attention(q, k, v, None, *args, "f16")
    v[key, 3::dim] = float("nan")
    got = window_attention(q, k, v, None, *args, "f16")
    nan = torch.zeros((batch, seq, heads, dim), dtype=torch.bool, device="cuda")
    nan[0, key:, :, 3] = True
    assert torch.equal(torch.isnan(got).view(batch, seq, heads, dim), nan)
    assert torch.equal(got[seq:], clean[seq:])
    v[key, 3::dim] = 0
    for i in (0, 50, 99, 100, 101, 127, 128, 5000, 20011, 39999):
        for h in range(heads):
            at = slice(h * dim, (h + 1) * dim)
            qd, kd, vd = q[i, at].double(), k[:i + 1, at].double(), v[:i + 1, at].double()
            p = torch.softmax(kd @ qd * dim ** -0.5, 0)
            want, pv = p @ vd, p @ vd.abs()
            # float32 scores (dim sums, the exponential) move a weight and the sum by twice this; weights and result rounded to binary16
            scores = 2 * (dim + 8) * 2.0 ** -23 * float((kd.abs() @ qd.abs()).max() * dim ** -0.5) + 2.0 ** -20
            bar = pv * (scores + 2.0 ** -11 * (1 + 2.0 ** -6)) + 2.0 ** -25 * (vd.abs().sum(0) + 1) + 2.0 ** -11 * want.abs()
            row = got[i, at].double()
            if i >= key:
                row[3], want[3] = 0, 0
            within(row, want, bar, "row %d of head %d" % (i, h))


@pytest.mark.parametrize("t", TYPES)
def test_window_attention_large_scores(t):
    """Scores of some thousands: the running maximum moves far; the largest weight wins."""
    q, k, v, m = window_inputs(21, 1, 700, 2, 2, 64, None, t)
    args = (1, 700, 2, 2, 64, 300, 300, 1, 40.0)
    check_window(window_attention(q, k, v, m, *args, t), window64(q, k, v, m, *args), t)
    args = (1, 700, 2, 2, 64, 300, 300, 1, 0.0)                  # every visible key weighs the same
    check_window(window_attention(q, k, v, m, *args, t), window64(q, k, v, m, *args), t)
    args = (1, 700, 2, 2, 64, 300, 300, 1, -0.125)
    check_window(window_attention(q, k, v, m, *args, t), window64(q, k, v, m, *args), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim,seq", [(64, 130), (128, 257), (32, 64), (40, 70)])
def test_window_attention_stays_inside_its_buffers(dim, seq, t):
    batch, heads, kv_heads = 2, 4, 2
    q, k, v, m = window_inputs(2, batch, seq, heads, kv_heads, dim, "holes", t)
    args = (batch, seq, heads, kv_heads, dim, 50, 11, 3, 0.2)
    want = window_attention(q, k, v, m, *args, t)
    parts = [banded(a.contiguous()) for a in (q, k, v, m)]
    ctx, ok = banded(torch.zeros_like(want))
    window_attention(*[p for p, _ in parts], *args, t, ctx=ctx)
    assert torch.equal(ctx, want) and ok() and all(good() for _, good in parts)
    assert all(torch.equal(p, a) for (p, _), a in zip(parts, (q, k, v, m)))


def step(q, k, v, pos, batch, heads, kv_heads, dim, window, sinks, scale, kc, vc, ctx, t):
    kernels.check(G.fn("window_attention_step", t)(G.ptr(q), G.ptr(k), G.ptr(v), q.stride(0), k.stride(0), G.ptr(pos), batch, heads, kv_heads, dim,
                                                   window, sinks, scale, G.ptr(kc), G.ptr(vc), G.ptr(ctx), ctx.stride(0), G.stream()))


def fill(k, v, lengths, batch, seq, kv_heads, dim, window, sinks, kc, vc, t):
    kernels.check(G.fn("window_cache_fill", t)(G.ptr(k), G.ptr(v), k.stride(0), G.ptr(lengths), batch, seq, kv_heads, dim, window, sinks,
                                               G.ptr(kc), G.ptr(vc), G.stream()))


# batch, heads, kv_heads, dim, window, sinks
STEPS = [(1, 1, 1, 64, 1, 0), (3, 4, 4, 64, 7, 2), (5, 8, 2, 128, 100, 4), (2, 6, 2, 64, 511, 1), (9, 12, 12, 64, 64, 0), (2, 32, 8, 128, 1020, 4),
         (1, 16, 1, 128, 3000, 17), (4, 3, 1, 5, 33, 1), (2, 4, 2, 256, 40, 3), (2, 40, 2, 64, 260, 0), (7, 2, 1, 32, 129, 1), (1, 8, 8, 64, 5000, 4),
         (40, 4, 2, 64, 300, 4), (2, 14, 2, 96, 130, 2)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,heads,kv_heads,dim,window,sinks", STEPS)
def test_window_attention_step(batch, heads, kv_heads, dim, window, sinks, t):
    g = gen(batch + heads + window)
    slots = window + sinks
    scale = dim ** -0.5
    choices = [0, 1, slots // 2, slots - 1, slots, slots + 1, 3 * slots + 5, sinks, max(sinks - 1, 0), 2 ** 31 - 1, -1, -2 ** 31]
    for turn in range(3):
        pos = torch.tensor([choices[(turn * 5 + i) % len(choices)] for i in range(batch)], dtype=torch.int32, device="cuda")
        qkv = normal(g, batch, (heads + 2 * kv_heads) * dim, t=t)
        q, k, v = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv_heads) * dim], qkv[:, (heads + kv_heads) * dim:]
        kc, vc = normal(g, batch, kv_heads, slots, dim, t=t), normal(g, batch, kv_heads, slots, dim, t=t)
        want_k, want_v = kc.clone(), vc.clone()
        seen = torch.zeros((batch, slots), dtype=torch.bool, device="cuda")
        for b, p in enumerate(pos.tolist()):
            if p >= 0:
                at = p if p < sinks else sinks + (p - sinks) % window
                n = min(p + 1, slots)
                want_k[b, :, at], want_v[b, :, at] = k[b].reshape(kv_heads, dim), v[b].reshape(kv_heads, dim)
                seen[b, :n] = True
                kc[b, :, n:], vc[b, :, n:] = float("nan"), float("inf")        # slots nothing has reached
                want_k[b, :, n:], want_v[b, :, n:] = float("nan"), float("inf")
                kc[b, :, at] = float("nan")                                    # the slot the new token takes over
                vc[b, :, at] = float("nan")
        share = heads // kv_heads
        clean = [torch.nan_to_num(a.double(), nan=0.0, posinf=0.0).repeat_interleave(share, 1) for a in (want_k, want_v)]
        ref = attention64(q.reshape(batch, heads, 1, dim).double(), *clean, seen[:, None, None, :], scale, dim)
        kb, ok_k = banded(kc)
        vb, ok_v = banded(vc)
        ctx, ok_c = banded(torch.full((batch, heads * dim), 5.0, dtype=q.dtype, device="cuda"))
        step(q, k, v, pos, batch, heads, kv_heads, dim, window, sinks, scale, kb, vb, ctx, t)
        live = pos >= 0
        check_window(ctx[live], tuple(a[live] for a in ref), t)
        assert bool((ctx[~live] == 5).all())
        assert torch.equal(torch.nan_to_num(kb, nan=-7.0), torch.nan_to_num(want_k, nan=-7.0))
        assert torch.equal(torch.nan_to_num(vb, nan=-7.0), torch.nan_to_num(want_v, nan=-7.0))
        assert ok_k() and ok_v() and ok_c()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads,window,sinks", [(64, 4, 2, 20, 3), (128, 8, 2, 70, 4), (48, 2, 2, 9, 0)])
def test_prompt_then_steps_equals_the_whole_sequence(dim, heads, kv_heads, window, sinks, t):
    """Prompts of ragged lengths, their caches filled, then one token at a time: every row as the causal form gives it."""
    batch, seq = 3, 150
    q, k, v, _ = window_inputs(12, batch, seq, heads, kv_heads, dim, None, t)
    args = (batch, seq, heads, kv_heads, dim, window - 1, 0, sinks, dim ** -0.5)
    ref = window64(q, k, v, None, *args)
    check_window(window_attention(q, k, v, None, *args, t), ref, t)
    lengths = torch.tensor([1, 60, 133], dtype=torch.int32, device="cuda")
    shape = (batch, kv_heads, window + sinks, dim)
    kc, vc = torch.full(shape, float("nan"), dtype=q.dtype, device="cuda"), torch.full(shape, float("nan"), dtype=q.dtype, device="cuda")
    fill(k, v, lengths, batch, seq, kv_heads, dim, window, sinks, kc, vc, t)
    pos = lengths.clone()
    for _ in range(90):
        rows = torch.arange(batch, device="cuda") * seq + pos.clamp(max=seq - 1)
        at = torch.where(pos < seq, pos, torch.full_like(pos, -1))
        ctx = torch.full((batch, heads * dim), float("nan"), dtype=q.dtype, device="cuda")
        step(q[rows], k[rows], v[rows], at, batch, heads, kv_heads, dim, window, sinks, dim ** -0.5, kc, vc, ctx, t)
        live = at >= 0
        check_window(ctx[live], tuple(a[rows][live] for a in ref), t)
        pos = pos + 1


@pytest.mark.parametrize("t", TYPES)
def test_cache_fill_writes_the_named_slots_only(t):
    batch, seq, kv_heads, dim = 4, 50, 2, 24
    _, k, v, _ = window_inputs(13, batch, seq, kv_heads, kv_heads, dim, None, t)
    for window, sinks, lengths in ((7, 2, [0, 1, 30, 50]), (100, 4, [3, 50, 60, -5]), (1, 0, [1, 2, 3, 49]), (20, 60, [50, 10, 0, 7])):
        slots = window + sinks
        kc, vc = normal(gen(1), batch, kv_heads, slots, dim, t=t), normal(gen(2), batch, kv_heads, slots, dim, t=t)
        want_k, want_v = kc.clone(), vc.clone()
        for b, n in enumerate(lengths):
            for j in range(min(max(n, 0), seq)):                 # in order: a later token takes its slot over
                at = j if j < sinks else sinks + (j - sinks) % window
                want_k[b, :, at], want_v[b, :, at] = k[b * seq + j].reshape(kv_heads, dim), v[b * seq + j].reshape(kv_heads, dim)
        kb, ok_k = banded(kc)
        vb, ok_v = banded(vc)
        fill(k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"), batch, seq, kv_heads, dim, window, sinks, kb, vb, t)
        assert torch.equal(kb, want_k) and torch.equal(vb, want_v) and ok_k() and ok_v()
    kc, vc = torch.zeros((batch, kv_heads, seq, dim), dtype=k.dtype, device="cuda"), torch.zeros((batch, kv_heads, seq, dim), dtype=k.dtype, device="cuda")
    fill(k, v, None, batch, seq, kv_heads, dim, seq, 0, kc, vc, t)
    assert torch.equal(kc, k.reshape(batch, seq, kv_heads, dim).permute(0, 2, 1, 3))
    assert torch.equal(vc, v.reshape(batch, seq, kv_heads, dim).permute(0, 2, 1, 3))


@pytest.mark.parametrize("seed", range(48))
def test_window_attention_of_random_shapes(seed):
    r = random.Random(seed)
    t = TYPES[seed % 2]
    dim = r.choice([8, 16, 24, 32, 40, 64, 64, 72, 96, 128, 128, 50])
    kv_heads = r.choice([1, 2, 3])
    heads = kv_heads * r.choice([1, 2, 3, 4])
    seq = r.choice([1, 2, 15, 16, 17, 63, 64, 65, 79, 81, 127, 128, 129, 255, 257, 300, 511, 700])
    batch = r.choice([1, 2, 3])
    before, after = r.choice([0, 1, 15, 16, 17, 100, 127, 128, 1000]), r.choice([0, 0, 1, 15, 64, 128, 1000])
    sinks = r.choice([0, 1, 4, 15, 16, 17, 33, 129, 300])
    q, k, v, m = window_inputs(seed, batch, seq, heads, kv_heads, dim, r.choice([None, "prefix", "holes"]), t, r.choice([0, 0, 8]))
    args = (batch, seq, heads, kv_heads, dim, before, after, sinks, r.choice([dim ** -0.5, 1.0, 0.01]))
    check_window(window_attention(q, k, v, m, *args, t), window64(q, k, v, m, *args), t, str((args, m is not None)))


@pytest.mark.parametrize("t", TYPES)
def test_window_attention_step_beyond_32_bit_offsets(t):
    """A cache of more than 2^31 elements: the last stream's last head is where it should be."""
    batch, heads, kv_heads, dim, window, sinks = 3, 4, 2, 128, 2900000, 4
    slots = window + sinks
    assert batch * kv_heads * slots * dim > 2 ** 31
    dt = G.TORCH_DTYPE[t]
    kc, vc = torch.zeros((batch, kv_heads, slots, dim), dtype=dt, device="cuda"), torch.zeros((batch, kv_heads, slots, dim), dtype=dt, device="cuda")
    g = gen(4)
    pos = torch.tensor([-1, 3, 10 * slots + 7], dtype=torch.int32, device="cuda")
    at = sinks + (10 * slots + 7 - sinks) % window
    kc[2, 1, -500:], vc[2, 1, -500:] = normal(g, 500, dim, t=t), normal(g, 500, dim, t=t)
    kc[2, :, :, 0] = -8.0                                        # the other slots count for little
    kc[2, 1, -500:, 0] = 8.0
    qkv = normal(g, batch, (heads + 2 * kv_heads) * dim, t=t)
    q, k, v = (a.clone() for a in (qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv_heads) * dim], qkv[:, (heads + kv_heads) * dim:]))
    q[2].view(heads, dim)[:, 0] = 8.0
    k[2].view(kv_heads, dim)[:, 0] = 8.0
    ctx = torch.zeros((batch, heads * dim), dtype=dt, device="cuda")
    step(q, k, v, pos, batch, heads, kv_heads, dim, window, sinks, dim ** -0.5, kc, vc, ctx, t)
    assert torch.equal(kc[2, :, at], k[2].view(kv_heads, dim)) and torch.equal(vc[2, 1, at], v[2].view(kv_heads, dim)[1])
    # scores away from the last 500 slots are exactly -64 / sqrt(128): their weights are counted, not listed
    s = torch.cat((kc[2, 1, -500:], kc[2, 1, at:at + 1])).double() @ q[2].view(heads, dim)[2:].double().t() * dim ** -0.5      # [501, 2]
    others = slots - 501
    top = s.amax(0)
    w = torch.exp(s - top)
    total = w.sum(0) + others * torch.exp(-64 * dim ** -0.5 - top)
    want = (w.t() @ torch.cat((vc[2, 1, -500:], vc[2, 1, at:at + 1])).double()) / total[:, None]
    got = ctx[2].view(heads, dim)[2:].double()
    # weights and values of the few that count, as in check_window; the sums take in 2.9 million equal terms
    bar = (2.0 ** -10 if t == "f16" else 2.0 ** -16) * (w.t() @ torch.cat((vc[2, 1, -500:], vc[2, 1, at:at + 1])).double().abs() / total[:, None])
    assert at < slots - 500 and bool(((got - want).abs() <= bar + 1e-6).all())
    assert float(ctx[0].abs().max()) == 0 and torch.isfinite(ctx.float()).all()


# ============================================================================ together, streams, graphs

class Layer:
    """One decoding layer without positions: norm (8 bits) -> 4-bit q | k | v -> attention step -> 4-bit output -> norm."""

    def __init__(self, t, batch, heads, kv_heads, dim, window, sinks, seed=3):
        g = gen(seed)
        self.t, self.batch, self.heads, self.kv_heads, self.dim, self.window, self.sinks = t, batch, heads, kv_heads, dim, window, sinks
        self.hidden, self.wide = heads * dim, (heads + 2 * kv_heads) * dim
        dt = G.TORCH_DTYPE[t]
        self.g1, self.g2 = 1 + normal(g, self.hidden, std=0.1, t=t), 1 + normal(g, self.hidden, std=0.1, t=t)
        self.w_qkv, self.w_out = normal(g, self.wide, self.hidden, std=0.05, t=t), normal(g, self.hidden, self.hidden, std=0.05, t=t)
        self.packs = []
        for w in (self.w_qkv, self.w_out):
            packed = torch.empty(kernels.load().cubk_w4_packed_bytes(*w.shape), dtype=torch.uint8, device="cuda")
            scales = torch.empty((w.shape[1] // 64, w.shape[0]), dtype=dt, device="cuda")
            kernels.check(G.fn("w4_quantize", t)(G.ptr(w), *w.shape, 64, G.ptr(packed), G.ptr(scales), G.stream()))
            self.packs.append((packed, scales))
        self.x, self.res = torch.zeros((batch, self.hidden), dtype=dt, device="cuda"), torch.zeros((batch, self.hidden), dtype=dt, device="cuda")
        self.pos = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.codes, self.code_scales = torch.empty((batch, self.hidden), dtype=F8, device="cuda"), torch.empty((batch, self.hidden // 128), device="cuda")
        self.qkv = torch.empty((batch, self.wide), dtype=dt, device="cuda")
        self.kc = torch.zeros((batch, kv_heads, window + sinks, dim), dtype=dt, device="cuda")
        self.vc = torch.zeros_like(self.kc)
        self.ctx, self.proj = torch.zeros((batch, self.hidden), dtype=dt, device="cuda"), torch.empty((batch, self.hidden), dtype=dt, device="cuda")
        self.out = torch.empty((batch, self.hidden), dtype=dt, device="cuda")

    def run(self):
        t, b = self.t, self.batch
        kernels.check(G.fn("residual_rms_norm_e4m3", t)(G.ptr(self.x), G.ptr(self.res), G.ptr(self.g1), b, self.hidden, 1e-6, 128, G.ptr(self.res),
                                                        G.ptr(self.codes), G.ptr(self.code_scales), G.stream()))
        matvec(self.codes, *self.packs[0], 64, self.wide, None, t, self.code_scales, 128, out=self.qkv)
        n, kv = self.hidden, self.kv_heads * self.dim
        step(self.qkv[:, :n], self.qkv[:, n:n + kv], self.qkv[:, n + kv:], self.pos, b, self.heads, self.kv_heads, self.dim, self.window, self.sinks,
             self.dim ** -0.5, self.kc, self.vc, self.ctx, t)
        matvec(self.ctx, *self.packs[1], 64, self.hidden, None, t, out=self.proj)
        rms_norm(self.proj, self.res, self.g2, 1e-6, t, total=self.res, out=self.out)


@pytest.mark.parametrize("t", TYPES)
def test_a_decoding_layer_of_the_three(t):
    """Each operator gets what the one before it wrote; each is held to its own bar on the inputs it got."""
    m = Layer(t, 5, 8, 2, 64, 12, 2)
    keys, values = [[] for _ in range(5)], [[] for _ in range(5)]
    for turn in range(30):
        m.x.copy_(normal(gen(100 + turn), 5, m.hidden, t=t))
        m.pos.fill_(turn)
        before = m.res.clone()
        m.run()
        t64, y64 = norm64(m.x, before, m.g1, 1e-6)
        scale = torch.stack([p.abs().amax(1) for p in y64.split(128, 1)], 1) / 448
        v = y64 / scale.repeat_interleave(128, 1)
        within(m.codes.float(), v, v.abs() * (2.0 ** -4 * (1 + 2.0 ** -10) + 2 * norm_bar(m.hidden)) + 2.0 ** -10 * (1 + 2.0 ** -10))
        x64 = m.codes.float().double() * m.code_scales.double().repeat_interleave(128, 1)
        q_codes = torch.from_numpy(unpack(m.packs[0][0], m.wide, m.hidden)).cuda()
        check_matvec(m.qkv, x64, q_codes, m.packs[0][1], 64, None, t)
        n, kv = m.hidden, m.kv_heads * m.dim
        for b in range(5):
            keys[b].append(m.qkv[b, n:n + kv].clone())
            values[b].append(m.qkv[b, n + kv:].clone())
        seen = [j for j in range(turn + 1) if j < m.sinks or j > turn - m.window]
        k = torch.stack([torch.stack([keys[b][j] for j in seen]) for b in range(5)]).view(5, -1, m.kv_heads, m.dim).permute(0, 2, 1, 3)
        vv = torch.stack([torch.stack([values[b][j] for j in seen]) for b in range(5)]).view(5, -1, m.kv_heads, m.dim).permute(0, 2, 1, 3)
        ref = attention64(m.qkv[:, :n].reshape(5, m.heads, 1, m.dim).double(), k.double().repeat_interleave(4, 1), vv.double().repeat_interleave(4, 1),
                          torch.ones((5, 1, 1, len(seen)), dtype=torch.bool, device="cuda"), m.dim ** -0.5, m.dim)
        check_window(m.ctx, ref, t)
        check_matvec(m.proj, m.ctx.double(), torch.from_numpy(unpack(m.packs[1][0], n, n)).cuda(), m.packs[1][1], 64, None, t)


@pytest.mark.parametrize("t", TYPES)
def test_captured_layers_share_nothing_and_replay(t):
    """Two captured layers replayed in turn and at once on two streams give what eager calls give, as positions advance."""
    eager, caught = [Layer(t, 3, 4, 2, 64, 40, 2, seed=s) for s in (1, 2)], [Layer(t, 3, 4, 2, 64, 40, 2, seed=s) for s in (1, 2)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for m, s in zip(caught, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            m.run()
            s.synchronize()
            with torch.cuda.graph(graph, stream=s):
                m.run()
        graphs.append(graph)
    for m in caught:
        m.res.zero_(), m.kc.zero_(), m.vc.zero_()
    torch.cuda.synchronize()
    for turn in range(60):
        for i in range(2):
            for m in (eager[i], caught[i]):
                m.x.copy_(normal(gen(7 * turn + i), 3, m.hidden, t=t))
                m.pos.copy_(torch.tensor([turn, 2 * turn, -1 if turn % 3 else turn], dtype=torch.int32))
            eager[i].run()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for name in ("out", "res", "kc", "vc"):
                assert torch.equal(getattr(eager[i], name), getattr(caught[i], name)), (turn, i, name)
    del graphs


FIRST_CALLS = """
import sys, torch
sys.path.insert(0, %r)
sys.path.insert(0, %r)
import test_norm_w4_window_gpu as M
torch.cuda.init()
g = M.gen(1)
work = []
for t in M.TYPES:
    for dim in (64, 128, 48, 5):
        q, k, v, m = M.window_inputs(dim, 2, 200, 4, 2, dim, "holes", t)
        args = (2, 200, 4, 2, dim, 40, 9, 3, 0.2)
        ctx = torch.zeros((400, 4 * dim), dtype=q.dtype, device="cuda")
        work.append((lambda q=q, k=k, v=v, m=m, args=args, t=t, ctx=ctx: M.window_attention(q, k, v, m, *args, t, ctx=ctx), ctx))
        kc, vc = torch.zeros((3, 2, 70, dim), dtype=q.dtype, device="cuda"), torch.zeros((3, 2, 70, dim), dtype=q.dtype, device="cuda")
        c2, pos = torch.zeros((3, 4 * dim), dtype=q.dtype, device="cuda"), torch.tensor([5, 69, 700], dtype=torch.int32, device="cuda")
        work.append((lambda q=q, k=k, v=v, kc=kc, vc=vc, c2=c2, pos=pos, dim=dim, t=t: M.step(q[:3], k[:3], v[:3], pos, 3, 4, 2, dim, 66, 4, 0.2, kc, vc, c2, t), c2))
    for n, k in ((40, 300), (2000, 1024)):
        for rows in (1, 12, 40):
            packed = M.pack(torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8))
            scales, x = M.normal(g, -(-k // 64), n, t=t), M.normal(g, rows, k, t=t)
            out = torch.zeros((rows, n), dtype=x.dtype, device="cuda")
            work.append((lambda x=x, packed=packed, scales=scales, n=n, t=t, out=out: M.matvec(x, packed, scales, 64, n, None, t, out=out), out))
    for ch in (64, 1024, 1001, 9000):
        x = M.normal(g, 7, ch, t=t)
        total, out = torch.zeros_like(x), torch.zeros_like(x)
        work.append((lambda x=x, total=total, out=out, t=t: M.rms_norm(x, None, x[0], 1e-6, t, total=total, out=out), out))
torch.cuda.synchronize()
s = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=s):       # the process's first call of each kernel
    for f, _ in work:
        f()
for _, out in work:
    out.zero_()
graph.replay()
torch.cuda.synchronize()
caught = [out.clone() for _, out in work]
for f, _ in work:
    f()
torch.cuda.synchronize()
assert all(torch.equal(a, out) for a, (_, out) in zip(caught, work))
assert all(bool((a != 0).any()) for a in caught)
del graph
print("FIRST CALLS CAPTURED")
"""


def test_first_calls_of_a_process_may_be_captured():
    here = os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS % (here, os.path.dirname(here))], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                         text=True, timeout=300)
    assert run.returncode == 0 and "FIRST CALLS CAPTURED" in run.stdout, run.stdout[-3000:]
