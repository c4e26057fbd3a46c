"""Cases of the root-mean-square norm, the products with 4-bit weights and the sliding-window attention.

Each case is one call a serving program makes: the plain forms below are the definitions in elementary torch operations,
the other branch calls the kernel library through its ctypes binding.
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the norm of one token between two layers of a decoding step: latency
        {"name": "norm_token_f16", "op": "norm", "t": "f16", "rows": 1, "channels": 1024, "residual": True, "out": "same"},
        # a batch of 256 x 128 tokens at hidden 1024, output for an 8-bit product with one scale per token
        {"name": "norm_batch_e4m3_f16", "op": "norm", "t": "f16", "rows": 32768, "channels": 1024, "residual": True, "out": "row"},
        # float32 storage, odd rows, a row length that no vector width but four divides, scales per 128 columns (the last block short)
        {"name": "norm_odd_e4m3_f32", "op": "norm", "t": "f32", "rows": 5001, "channels": 1004, "residual": False, "out": "block"},
        # one token through a query/key/value projection of hidden 768
        {"name": "matvec_token_f16", "op": "matvec", "t": "f16", "x": "same", "rows": 1, "k": 768, "n": 2304, "group": 128, "bias": True},
        # sixteen rows against a vocabulary of 30522: weights larger than most of L2
        {"name": "matvec_vocab_f16", "op": "matvec", "t": "f16", "x": "same", "rows": 16, "k": 4096, "n": 30522, "group": 128, "bias": False},
        # the 8-bit rows the norm writes into a feed-forward product, a few tokens
        {"name": "matvec_e4m3_f16", "op": "matvec", "t": "f16", "x": "row", "rows": 5, "k": 4096, "n": 11008, "group": 64, "bias": True},
        # float32 storage, a reduction length that is not a multiple of the group, small groups
        {"name": "matvec_odd_f32", "op": "matvec", "t": "f32", "x": "same", "rows": 3, "k": 1000, "n": 21128, "group": 32, "bias": True},
        # long documents in an encoder: symmetric window, the first token seen by all, ragged lengths, heads of BERT-large
        {"name": "window_encoder_f16", "op": "window", "t": "f16", "batch": 4, "seq": 4096, "heads": 16, "kv_heads": 16, "dim": 64,
         "before": 256, "after": 256, "sinks": 1, "mask": "prefix"},
        # one long prompt of a decoder with shared key/value heads
        {"name": "window_prompt_f16", "op": "window", "t": "f16", "batch": 1, "seq": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "before": 2047, "after": 0, "sinks": 4, "mask": "none"},
        # float32 storage, odd length, keys masked anywhere (some rows see nothing)
        {"name": "window_odd_f32", "op": "window", "t": "f32", "batch": 3, "seq": 777, "heads": 12, "kv_heads": 12, "dim": 64,
         "before": 100, "after": 30, "sinks": 2, "mask": "holes"},
        # single tokens of many streams over their ring caches
        {"name": "step_streams_f16", "op": "step", "t": "f16", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "window": 2044, "sinks": 4},
        # a single token of one stream, float32: latency
        {"name": "step_one_f32", "op": "step", "t": "f32", "batch": 1, "heads": 12, "kv_heads": 12, "dim": 64, "window": 511, "sinks": 1},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "matvec", "window", "step"])
    t = rng.choice(["f16", "f16", "f32"])
    if op == "norm":
        channels = _log(rng, 8, 8192)
        rows = _log(rng, 1, max(1, min(40000, (1 << 24) // channels)))
        if rng.random() < 0.5:
            channels = (channels + 7) // 8 * 8
        return {"op": op, "t": t, "rows": rows, "channels": channels, "residual": rng.random() < 0.7, "out": rng.choice(["same", "row", "block"])}
    if op == "matvec":
        k = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            k = (k + 63) // 64 * 64
        n = _log(rng, 16, min(32768, (1 << 26) // k))
        return {"op": op, "t": t, "x": rng.choice(["same", "same", "row", "block"]), "rows": rng.choice([1, 1, 2, 3, 4, 7, 8, 11, 16, 24, 33, 64]),
                "k": k, "n": n, "group": rng.choice([32, 64, 128]), "bias": rng.random() < 0.5}
    dim = rng.choice([32, 64, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    if op == "window":
        seq = _log(rng, 1, 4096)
        batch = rng.randint(1, max(1, min(16, (1 << 25) // (seq * max(seq, 64)))))
        causal = rng.random() < 0.5
        return {"op": op, "t": t, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "before": _log(rng, 1, 2048) - 1, "after": 0 if causal else _log(rng, 1, 1024), "sinks": rng.choice([0, 1, 4, 17]),
                "mask": rng.choice(["none", "prefix", "holes"])}
    window = _log(rng, 1, 4096)
    return {"op": op, "t": t, "batch": rng.randint(1, max(1, min(48, (1 << 16) // (window + 64)))), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": rng.choice([0, 1, 4, 17])}


# ------------------------------------------------------------------------------------------------ inputs

def _pack(codes):
    """int8 codes [n, k] in -8..7 -> the kernel library's packed bytes: tiles of 16 rows x 128 columns; per row and tile 16 words,
    word 4 t + j holding columns 32 j + 8 t .. + 7, even columns in its low half and odd ones in its high half."""
    n, k = codes.shape
    nt, kt = -(-n // 16), -(-k // 128)
    full = torch.zeros((nt * 16, kt * 128), dtype=torch.int32, device=codes.device)
    full[:n, :k] = codes
    v = (full + 8).view(nt, 16, kt, 4, 4, 4, 2)                  # tile, row, block, j, t, pair, parity
    v = v.permute(0, 2, 1, 4, 3, 6, 5).reshape(nt, kt, 16, 16, 4, 2)   # tile, block, row, word 4 t + j, then nibbles two by two
    return (v[..., 0] | (v[..., 1] << 4)).to(torch.uint8).contiguous()


def _unpack(packed, n, k):
    """The codes [n, k] of the packed bytes, as float32."""
    nt, kt = packed.shape[:2]
    v = torch.stack((packed & 15, packed >> 4), dim=-1).view(nt, kt, 16, 4, 4, 2, 4)  # tile, block, row, t, j, parity, pair
    v = v.permute(0, 2, 1, 4, 3, 6, 5).reshape(nt * 16, kt * 128)
    return v[:n, :k].float() - 8.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["t"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        rows, ch = case["rows"], case["channels"]
        s["x"] = normal(rows, ch)
        s["r"] = normal(rows, ch, std=2.0) if case["residual"] else None
        s["g"] = 1 + normal(ch, std=0.1)
    elif case["op"] == "matvec":
        rows, k, n = case["rows"], case["k"], case["n"]
        x = normal(rows, k, dtype=torch.float32)
        if case["x"] == "same":
            s["x"], s["xs"] = x.to(t), None
        else:
            block = k if case["x"] == "row" else 128
            nb = -(-k // block)
            top = torch.zeros((rows, nb * block), device="cuda")
            top[:, :k] = x.abs()
            s["xs"] = top.view(rows, nb, block).amax(2) / 448
            s["x"] = (x / s["xs"].repeat_interleave(block, 1)[:, :k]).to(F8)
        s["w"] = _pack(torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8))
        s["ws"] = (torch.rand((-(-k // case["group"]), n), generator=g, device="cuda") * 0.004 + 0.001).to(t)
        s["b"] = normal(n, std=0.1) if case["bias"] else None
    elif case["op"] == "window":
        rows = case["batch"] * case["seq"]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        qkv = normal(rows, (h + 2 * hk) * d)                    # one projection's output: query | key | value heads
        s["q"], s["k"], s["v"] = qkv[:, :h * d], qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:]
        s["m"] = None
        if case["mask"] == "prefix":
            lengths = torch.randint(max(1, case["seq"] // 16), case["seq"] + 1, (case["batch"], 1), generator=g, device="cuda")
            s["m"] = (torch.arange(case["seq"], device="cuda") < lengths).to(torch.int8)
        elif case["mask"] == "holes":
            s["m"] = (torch.rand((case["batch"], case["seq"]), generator=g, device="cuda") < 0.6).to(torch.int8)
            s["m"][0, : case["seq"] // 2] = 0                   # whole windows without a kept key
    else:
        b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        slots = case["window"] + case["sinks"]
        qkv = normal(b, (h + 2 * hk) * d)
        s["q"], s["k"], s["v"] = qkv[:, :h * d], qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:]
        s["kc"], s["vc"] = normal(b, hk, slots, d), normal(b, hk, slots, d)
        # most streams are far past their window, every fifth is still filling it, one in seven rows of a larger batch is idle
        pos = torch.randint(slots, 100 * slots + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        short = torch.randint(0, slots, (b,), generator=g, device="cuda", dtype=torch.int32)
        i = torch.arange(b, device="cuda")
        pos = torch.where(i % 5 == 3, short, pos)
        s["pos"] = torch.where(i % 7 == 5, torch.full_like(pos, -1), pos)
        s["ctx"] = torch.zeros((b, h * d), dtype=t, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_norm(s):
    t = s["x"].float()
    if s["r"] is not None:
        t = t + s["r"].float()
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * s["g"].float()
    if s["out"] == "same":
        return [t.to(s["x"].dtype), y.to(s["x"].dtype)]
    rows, ch = y.shape
    block = ch if s["out"] == "row" else 128
    nb = -(-ch // block)
    z = torch.nn.functional.pad(y, (0, nb * block - ch)).view(rows, nb, block)
    scale = z.abs().amax(2, keepdim=True) / 448
    codes = torch.where(scale > 0, z / scale, torch.zeros_like(z)).view(rows, nb * block)[:, :ch].to(F8)
    return [t.to(s["x"].dtype), codes, scale.view(rows, nb)]


def _plain_matvec(s):
    n, k = s["n"], s["k"]
    x = s["x"].float()
    if s["xs"] is not None:
        x = x * s["xs"].repeat_interleave(k if s["xs"].shape[1] == 1 else 128, 1)[:, :k]
    w = _unpack(s["w"], n, k) * s["ws"].float().repeat_interleave(s["group"], 0)[:k].t()
    out = x @ w.t()
    if s["b"] is not None:
        out = out + s["b"].float()
    return out.to(TYPES[s["t"]])


def _plain_window(s):
    b, n, h, hk, d = s["batch"], s["seq"], s["heads"], s["kv_heads"], s["dim"]
    q = s["q"].reshape(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).float()
    k = s["k"].reshape(b, n, hk, 1, d).permute(0, 2, 3, 4, 1).float()
    v = s["v"].reshape(b, n, hk, 1, d).permute(0, 2, 3, 1, 4).float()
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
    seen = ((j <= i + s["after"]) & ((j >= i - s["before"]) | (j < s["sinks"])))[None]
    if s["m"] is not None:
        seen = seen & (s["m"] != 0)[:, None, :]
    seen = seen[:, None, None]
    p = torch.matmul(q, k).mul_(d ** -0.5).masked_fill_(~seen, -math.inf)
    top = p.amax(4, keepdim=True)
    p = p.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = p.sum(4, keepdim=True)
    ctx = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return ctx.permute(0, 3, 1, 2, 4).reshape(b * n, h * d).to(s["q"].dtype)


def _plain_step(s):
    b, h, hk, d, w, sinks = s["batch"], s["heads"], s["kv_heads"], s["dim"], s["window"], s["sinks"]
    pos = s["pos"].long()
    live = pos >= 0
    slot = torch.where(pos < sinks, pos, sinks + (pos - sinks) % w)
    here = ((torch.arange(w + sinks, device="cuda")[None] == slot[:, None]) & live[:, None])[:, None, :, None]
    s["kc"].copy_(torch.where(here, s["k"].reshape(b, hk, 1, d), s["kc"]))
    s["vc"].copy_(torch.where(here, s["v"].reshape(b, hk, 1, d), s["vc"]))
    q = s["q"].reshape(b, hk, h // hk, d).float()
    p = torch.matmul(q, s["kc"].float().transpose(2, 3)) * d ** -0.5
    p = p.masked_fill((torch.arange(w + sinks, device="cuda")[None] > pos.clamp(min=0)[:, None])[:, None, None], -math.inf)
    p = (p - p.amax(3, keepdim=True)).exp()
    ctx = torch.matmul(p, s["vc"].float()) / p.sum(3, keepdim=True)
    s["ctx"].copy_(torch.where(live[:, None], ctx.reshape(b, h * d).to(s["ctx"].dtype), s["ctx"]))
    return [s["ctx"], s["kc"], s["vc"]]


# ------------------------------------------------------------------------------------------------ the framework's calls

def _call(name, s, *args):
    from cubert_b200 import kernels
    p = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    kernels.check(getattr(kernels.load(), "cubk_%s_%s" % (name, s["t"]))(*p, torch.cuda.current_stream().cuda_stream))


def _own_norm(s):
    rows, ch = s["rows"], s["channels"]
    total = torch.empty_like(s["x"])
    if s["out"] == "same":
        y = torch.empty_like(s["x"])
        _call("residual_rms_norm", s, s["x"], s["r"], s["g"], rows, ch, EPS, total, y)
        return [total, y]
    group = 0 if s["out"] == "row" else 128
    codes = torch.empty((rows, ch), dtype=F8, device="cuda")
    scales = torch.empty((rows, 1 if group == 0 else -(-ch // group)), dtype=torch.float32, device="cuda")
    _call("residual_rms_norm_e4m3", s, s["x"], s["r"], s["g"], rows, ch, EPS, group, total, codes, scales)
    return [total, codes, scales]


def _own_matvec(s):
    out = torch.empty((s["rows"], s["n"]), dtype=TYPES[s["t"]], device="cuda")
    if s["xs"] is None:
        _call("w4_matvec", s, s["x"], s["rows"], s["k"], s["w"], s["ws"], s["group"], s["n"], s["b"], out)
    else:
        _call("w4_matvec_e4m3", s, s["x"], s["xs"], 0 if s["xs"].shape[1] == 1 else 128, s["rows"], s["k"], s["w"], s["ws"], s["group"], s["n"], s["b"], out)
    return out


def _own_window(s):
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    ctx = torch.empty((s["batch"] * s["seq"], h * d), dtype=s["q"].dtype, device="cuda")
    _call("window_attention", s, s["q"], s["k"], s["v"], s["q"].stride(0), s["k"].stride(0), s["m"], s["batch"], s["seq"], h, hk, d,
          s["before"], s["after"], s["sinks"], d ** -0.5, ctx, h * d)
    return ctx


def _own_step(s):
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    _call("window_attention_step", s, s["q"], s["k"], s["v"], s["q"].stride(0), s["k"].stride(0), s["pos"], s["batch"], h, hk, d,
          s["window"], s["sinks"], d ** -0.5, s["kc"], s["vc"], s["ctx"], h * d)
    return [s["ctx"], s["kc"], s["vc"]]


def run(state):
    if own:
        return {"norm": _own_norm, "matvec": _own_matvec, "window": _own_window, "step": _own_step}[state["op"]](state)
    return {"norm": _plain_norm, "matvec": _plain_matvec, "window": _plain_window, "step": _plain_step}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ 64-bit values

def exact(case, seed):
    """The definitions in float64, one row group / head at a time. For 8-bit codes the value that is rounded: y / scale."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        t = s["x"].double() + (0 if s["r"] is None else s["r"].double())
        y = t / torch.sqrt(t.pow(2).sum(1, keepdim=True) / case["channels"] + EPS) * s["g"].double()
        if case["out"] == "same":
            return [t, y]
        codes, scales = [], []
        for part in y.split(case["channels"] if case["out"] == "row" else 128, 1):
            scale = part.abs().max(1, keepdim=True).values / 448
            scales.append(scale)
            codes.append(part / scale.clamp(min=1e-300))
        return [t, torch.cat(codes, 1), torch.cat(scales, 1)]
    if case["op"] == "matvec":
        n, k, x = case["n"], case["k"], s["x"].double()
        if s["xs"] is not None:
            block = k if case["x"] == "row" else 128
            x = torch.cat([part * s["xs"][:, i:i + 1].double() for i, part in enumerate(x.split(block, 1))], 1)
        out = torch.zeros((case["rows"], n), dtype=torch.float64, device="cuda")
        for c in range(k):                                       # column c of the weights: word, half and nibble looked up one by one
            blk, j, t, e = c // 128, c % 128 // 32, c % 32 // 8, c % 8
            nib = (4 * t + j) * 8 + (e % 2) * 4 + e // 2
            byte = s["w"][:, blk].reshape(-1, 64)[:n, nib // 2].long()
            code = (byte >> 4 if nib % 2 else byte & 15) - 8
            out += x[:, c:c + 1] * (code.double() * s["ws"][c // case["group"]].double())[None]
        return out if s["b"] is None else out + s["b"].double()
    d, ratio = case["dim"], case["heads"] // case["kv_heads"]
    if case["op"] == "window":
        n = case["seq"]
        i = torch.arange(n, device="cuda")
        far = i[None, :] - i[:, None]                            # key minus query
        ctx = torch.zeros((case["batch"], n, case["heads"], d), dtype=torch.float64, device="cuda")
        q = s["q"].reshape(case["batch"], n, -1, d)
        k, v = s["k"].reshape(case["batch"], n, -1, d), s["v"].reshape(case["batch"], n, -1, d)
        for b in range(case["batch"]):
            hidden = (far > case["after"]) | ((far < -case["before"]) & (i >= case["sinks"])[None, :])
            if s["m"] is not None:
                hidden |= (s["m"][b] == 0)[None, :]
            empty = hidden.all(1)
            for h in range(case["heads"]):
                w = q[b, :, h].double() @ k[b, :, h // ratio].double().t() / math.sqrt(d)
                w[hidden] = -1e300
                w = torch.softmax(w, 1)
                w[empty] = 0
                ctx[b, :, h] = w @ v[b, :, h // ratio].double()
        return ctx.reshape(case["batch"] * n, -1)
    ctx, kc, vc = s["ctx"].double(), s["kc"].double(), s["vc"].double()
    for b, p in enumerate(s["pos"].tolist()):
        if p < 0:
            continue
        at = p if p < case["sinks"] else case["sinks"] + (p - case["sinks"]) % case["window"]
        seen = min(p + 1, case["sinks"] + case["window"])
        kc[b, :, at] = s["k"][b].reshape(-1, d).double()
        vc[b, :, at] = s["v"][b].reshape(-1, d).double()
        for h in range(case["heads"]):
            w = torch.softmax(kc[b, h // ratio, :seen] @ s["q"][b, h * d:(h + 1) * d].double() / math.sqrt(d), 0)
            ctx[b, h * d:(h + 1) * d] = w @ vc[b, h // ratio, :seen]
    return [ctx, kc, vc]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = 2 if case["t"] == "f16" else 4
    if case["op"] == "norm":
        rows, ch = case["rows"], case["channels"]
        out = e * ch if case["out"] == "same" else ch + 4 * (1 if case["out"] == "row" else -(-ch // 128))
        return {"bytes": rows * (ch * e * (3 if case["residual"] else 2) + out) + ch * e, "flops": 6.0 * rows * ch}
    if case["op"] == "matvec":
        rows, k, n = case["rows"], case["k"], case["n"]
        x = e * k if case["x"] == "same" else k + 4 * (1 if case["x"] == "row" else -(-k // 128))
        return {"bytes": n * k / 2 + -(-k // case["group"]) * n * e + rows * (x + n * e) + (n * e if case["bias"] else 0), "flops": 2.0 * rows * n * k}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "window":
        n, bf, af, sk = case["seq"], case["before"], case["after"], case["sinks"]
        pairs = 0
        for i in range(n):
            lo, hi = max(0, i - bf), min(n - 1, i + af)
            pairs += hi - lo + 1 + min(sk, lo)
        kept = {"none": 1.0, "prefix": 0.53, "holes": 0.5}[case["mask"]]   # the mean share of kept keys
        return {"bytes": case["batch"] * n * (e * d * (2 * h + 2 * hk * kept) + (0 if case["mask"] == "none" else 1)),
                "flops": 4.0 * d * h * case["batch"] * pairs * kept}
    slots = case["window"] + case["sinks"]
    b = case["batch"]
    live = b - len(range(5, b, 7))
    seen = sum((0.5 if i % 5 == 3 else 1.0) * slots for i in range(b) if i % 7 != 5)
    return {"bytes": e * d * (2 * hk * seen + live * (2 * h + 4 * hk)) + 4 * b, "flops": 4.0 * d * h * seen}
