"""The operators of a decoder's step on the kernel ABI, as measurable cases.

  norm     thb_rmsnorm_fwd: the residual's addition, root-mean-square norm, and its result in 16 or 32 bits, in 8, or both
  gemv     thb_gemv_q4_fwd: 4-bit weights with group scales on up to eight rows
  append   thb_kv_append_fwd: keys and values into a paged cache, keys and queries rotated by their positions on the way
  attend   thb_paged_attn_fwd: attention of one new token a sequence over the paged cache

`own` false: the plain forms in elementary torch operations; true: the calls that a program makes of libthnets.so.  A program
fills an operator's descriptor once and keeps it, as it keeps its weights: so does a state, from its first pass on.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
E4M3_MAX = 448.0
MOST_BYTES = 1.0e9          # no drawn case moves more than the largest listed one
MOST_GEMV = 130e6           # weights (values) of a drawn matrix


def _norm(name, dtype, rows, c, res, out):
    return dict(name=name, op="norm", dtype=dtype, rows=rows, c=c, res=res, out=out)


def _gemv(name, dtype, n, k, m, group, zeros, x8=False):
    return dict(name=name, op="gemv", dtype=dtype, n=n, k=k, m=m, group=group, zeros=zeros, x8=x8)


def _append(name, dtype, tokens, seqs, q_heads, heads, dim, rot, interleaved, page, far):
    return dict(name=name, op="append", dtype=dtype, tokens=tokens, seqs=seqs, q_heads=q_heads, heads=heads, dim=dim, rot=rot,
                interleaved=interleaved, page=page, far=far)


def _attend(name, dtype, rows, most, least, q_heads, heads, dim, page, window, by_head):
    return dict(name=name, op="attend", dtype=dtype, rows=rows, most=most, least=least, q_heads=q_heads, heads=heads, dim=dim,
                page=page, window=window, by_head=by_head)


def listed():
    return [
        # one token of a decoder of 4096 channels: residual in, codes for the 4-bit product out; nothing but latency
        _norm("norm_bf16_1_e4m3", "bf16", 1, 4096, True, "q"),
        # a prompt of eight thousand tokens in half precision
        _norm("norm_fp16_8192", "fp16", 8192, 4096, True, "y"),
        # full precision, rows of an odd number of vectors, both results
        _norm("norm_fp32_777_odd", "fp32", 777, 1004, False, "yq"),
        # a square projection for one token: the smallest product that a decoder has many of
        _gemv("gemv_fp16_1", "fp16", 1, 4096, 4096, 128, False),
        # the first fully connected layer of AlexNet-OWT, eight rows at a time, with zero points
        _gemv("gemv_bf16_8_g64", "bf16", 8, 9216, 4096, 64, True),
        # a vocabulary's scores for four tokens from the norm's 8-bit codes, rows that no tile divides
        _gemv("gemv_e4m3_4_g32_odd", "fp16", 4, 4096, 32003, 32, True, x8=True),
        # VGG-16's first fully connected layer in full precision on three pictures
        _gemv("gemv_fp32_3", "fp32", 3, 25088, 4096, 128, False),
        # a token of each of sixteen conversations, far into them
        _append("append_bf16_16", "bf16", 16, 16, 32, 8, 128, 128, False, 16, 100000),
        # four prompts of two thousand tokens each, half of every head rotated in neighbouring pairs
        _append("append_fp16_8192", "fp16", 8192, 4, 32, 8, 128, 64, True, 64, 0),
        # one conversation of four thousand tokens: few rows, so the length has to be split
        _attend("attend_fp16_1", "fp16", 1, 4096, 4096, 32, 8, 128, 16, 0, False),
        # full precision, heads of 80 without sharing, odd lengths and pages, a window that cuts them
        _attend("attend_fp32_5_odd", "fp32", 5, 3001, 0, 12, 12, 80, 24, 2500, True),
        # long documents, eight at a time
        _attend("attend_bf16_8_long", "bf16", 8, 32768, 20000, 32, 8, 128, 64, 0, False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "gemv", "append", "attend"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if op == "norm":
        c = _log(rng, 60, 16384)
        rows = _log(rng, 1, max(2, min(20000, 200_000_000 // (c * 4))))
        case = _norm("", dtype, rows, c, rng.random() < 0.7, rng.choice(("y", "q", "yq")))
    elif op == "gemv":
        k = _log(rng, 64, 25088)
        m = _log(rng, 16, min(130000, MOST_GEMV / k))
        case = _gemv("", dtype, rng.randint(1, 8), k, m, rng.choice((32, 64, 128)), rng.random() < 0.5,
                     dtype != "fp32" and rng.random() < 0.4)
    elif op == "append":
        heads, dim = rng.choice((1, 2, 4, 8, 12)), rng.choice((64, 80, 96, 128, 256))
        tokens = _log(rng, 1, 8192)
        seqs = tokens if tokens <= 64 and rng.random() < 0.5 else rng.randint(1, min(8, tokens))
        rot = rng.choice((dim, dim // 2, dim // 4 // 2 * 2))
        case = _append("", dtype, tokens, seqs, heads * rng.choice((1, 2, 4)), heads, dim, rot, rng.random() < 0.5,
                       rng.choice((16, 24, 32, 64, 128)), rng.choice((0, 1000, 100000)))
    else:
        heads, dim = rng.choice((1, 2, 4, 8, 12)), rng.choice((64, 80, 96, 128, 256))
        rows = _log(rng, 1, 96)
        cap = MOST_BYTES / (rows * heads * dim * 2.0 * SIZE[dtype])
        most = _log(rng, 1, max(2, min(60000, cap)))
        least = rng.choice((0, most // 2, most))
        case = _attend("", dtype, rows, most, least, heads * rng.choice((1, 3, 4, 8, 16)), heads, dim, rng.choice((16, 24, 32, 64, 128)),
                       0 if rng.random() < 0.7 else _log(rng, 1, max(2, most)), rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs

def _up(v, m):
    return (v + m - 1) // m * m


def _frequencies(rot, base, factor):
    """Radians a position of each pair; `factor`: positions pressed together for contexts longer than a model was made for."""
    i = torch.arange(max(rot // 2, 1), dtype=torch.float64)
    return (base ** (-2.0 * i / max(rot, 1)) / factor).cuda()


def _pages(g, seqs, a_seq, spare):
    """A table of pages in no order, `a_seq` of each of `seqs` sequences, from a pool with `spare` more; the table and the pool's size."""
    pool = seqs * a_seq + spare
    return torch.randperm(pool, generator=g, device="cuda")[: seqs * a_seq].reshape(seqs, a_seq).to(torch.int32).contiguous(), pool


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    vec = 16 // SIZE[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        s["has_res"] = case["res"]
        rows, c, ld = case["rows"], case["c"], _up(case["c"], vec)
        # a residual stream's few large channels among many small ones
        spread = torch.exp(0.8 * randn(c))
        s["x"] = torch.zeros(rows, ld, device="cuda", dtype=dt)
        s["x"][:, :c] = randn(rows, c) * 0.3
        s["res"] = torch.zeros_like(s["x"])
        s["res"][:, :c] = randn(rows, c) * spread
        s["gain"] = (1.0 + 0.2 * randn(c)).contiguous()
        s["sum"], s["y"] = torch.zeros_like(s["x"]), torch.zeros_like(s["x"])
        s["q"] = torch.zeros(rows, _up(c, 16), device="cuda", dtype=torch.float8_e4m3fn)
        s["q_scale"] = torch.zeros(rows, device="cuda")
    elif case["op"] == "gemv":
        n, k, m, group = case["n"], case["k"], case["m"], case["group"]
        groups = (k + group - 1) // group
        s["w"] = torch.randint(0, 256, (m, _up(k, 32) // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["wscale"] = (torch.exp(0.3 * randn(m, groups)) / (4.6 * math.sqrt(k))).to(torch.float16)
        s["wzero"] = torch.randint(5, 11, (m, groups), generator=g, device="cuda", dtype=torch.uint8)
        s["shift"] = 0.1 * randn(m)
        x = randn(n, k) * torch.exp(0.5 * randn(k))
        s["x"] = torch.zeros(n, _up(k, 16), device="cuda", dtype=torch.float8_e4m3fn if case["x8"] else dt)
        s["x_scale"] = (x.abs().amax(1) / E4M3_MAX).contiguous()
        s["x"][:, :k] = (x / s["x_scale"][:, None]).to(s["x"].dtype) if case["x8"] else x.to(dt)
        s["y"] = torch.zeros(n, _up(m, vec), device="cuda", dtype=dt)
    elif case["op"] == "append":
        tokens, seqs, heads, dim, page = case["tokens"], case["seqs"], case["heads"], case["dim"], case["page"]
        at = torch.arange(tokens, device="cuda")
        s["seq"] = (at % seqs).to(torch.int32)
        turn = at // seqs
        before = torch.randint(0, page, (seqs,), generator=g, device="cuda")
        s["pos"] = (case["far"] + before[s["seq"].long()] + turn).to(torch.int32)
        last = case["far"] + page + (tokens + seqs - 1) // seqs
        # pages before the first one written belong to the conversation's past: the table names them, the pool need not hold more
        first = case["far"] // page
        table, pool = _pages(g, seqs, last // page + 1 - first, 3)
        s["table"] = torch.zeros(seqs, last // page + 1, device="cuda", dtype=torch.int32)
        s["table"][:, first:] = table
        s["pool"] = pool
        s["qkv"] = randn(tokens, (case["q_heads"] + 2 * heads) * dim).to(dt)
        s["freq"] = _frequencies(case["rot"], 500000.0, 1.0 if case["far"] < 50000 else 4.0)
        s["q_out"] = torch.zeros(tokens, case["q_heads"] * dim, device="cuda", dtype=dt)
        s["k"] = torch.zeros(pool, page, heads, dim, device="cuda", dtype=dt)
        s["v"] = torch.zeros_like(s["k"])
    else:
        rows, heads, dim, page, most = case["rows"], case["heads"], case["dim"], case["page"], case["most"]
        a_seq = (most + page - 1) // page
        s["table"], s["pool"] = _pages(g, rows, a_seq, 5)
        shape = (s["pool"], heads, page, dim) if case["by_head"] else (s["pool"], page, heads, dim)
        s["k"] = randn(*shape).to(dt)
        s["v"] = randn(*shape).to(dt)
        s["len"] = torch.randint(case["least"], most + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["len"][rows // 2] = most
        s["q"] = (1.5 * randn(rows, case["q_heads"] * dim)).to(dt)
        s["y"] = torch.zeros(rows, case["q_heads"] * dim, device="cuda", dtype=dt)
    return s


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n = case["rows"] * case["c"]
        b = n * size * (3 if case["res"] else 1) + 4 * case["c"]
        b += n * size * ("y" in case["out"]) + (n + 4 * case["rows"]) * ("q" in case["out"])
        return {"bytes": b, "flops": 5 * n}
    if case["op"] == "gemv":
        n, k, m = case["n"], case["k"], case["m"]
        groups = (k + case["group"] - 1) // case["group"]
        x = n * (k + 4) if case["x8"] else n * k * size
        return {"bytes": m * ((k + 1) // 2 + groups * (3 if case["zeros"] else 2) + 4) + x + n * m * size, "flops": 2.0 * n * m * k}
    if case["op"] == "append":
        n = case["tokens"] * (case["q_heads"] + 2 * case["heads"]) * case["dim"]
        return {"bytes": 2 * n * size + case["tokens"] * 8, "flops": 3.0 * case["tokens"] * (case["q_heads"] + case["heads"]) * case["rot"]}
    mean = (case["least"] + case["most"]) / 2.0
    if case["window"]:
        mean = min(mean, case["window"])
    tokens = (case["rows"] - 1) * mean + (min(case["most"], case["window"]) if case["window"] else case["most"])
    b = 2 * tokens * case["heads"] * case["dim"] * size + 2 * case["rows"] * case["q_heads"] * case["dim"] * size
    return {"bytes": b, "flops": 4.0 * tokens * case["q_heads"] * case["dim"]}


# ----------------------------------------------------------------------------------------------------------- plain forms

def _plain_norm(s):
    c = s["c"]
    wide = torch.float64 if "q" in s["out"] else torch.float32  # a code next to a border takes 64 bits to tell
    t = s["x"][:, :c].to(wide)
    out = {}
    if s["has_res"]:
        t = t + s["res"][:, :c].to(wide)
        out["sum"] = t.to(s["x"].dtype)
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-5) * s["gain"].to(wide)
    if "y" in s["out"]:
        out["y"] = y.to(s["x"].dtype)
    if "q" in s["out"]:
        scale = y.abs().amax(1, keepdim=True) / E4M3_MAX
        out["q"] = (y / scale).float().to(torch.float8_e4m3fn)
        out["q_scale"] = scale[:, 0].float()
    return out


def _plain_gemv(s):
    k, group = s["k"], s["group"]
    w = torch.stack((s["w"] & 15, s["w"] >> 4), 2).reshape(s["m"], -1)[:, :k].float()
    zero = s["wzero"].float() if s["zeros"] else torch.full_like(s["wzero"], 8, dtype=torch.float32)
    w -= zero.repeat_interleave(group, 1)[:, :k]
    w *= s["wscale"].float().repeat_interleave(group, 1)[:, :k]
    x = s["x"][:, :k].float()
    if s["x8"]:
        x = x * s["x_scale"][:, None]
    return (x @ w.T + s["shift"]).to(s["y"].dtype)


def _rotated(s, x, heads):
    """x: [tokens, heads, dim] in 32 bits."""
    rot, dim = s["rot"], s["dim"]
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(-1, heads, rot)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_append(s):
    hq, h, dim, page = s["q_heads"], s["heads"], s["dim"], s["page"]
    q, k, v = torch.split(s["qkv"].reshape(-1, hq + 2 * h, dim), (hq, h, h), 1)
    pos, seq = s["pos"].long(), s["seq"].long()
    at = s["table"].long()[seq, pos // page], pos % page
    s["k"][at] = _rotated(s, k.float(), h).to(k.dtype)
    s["v"][at] = v
    s["q_out"].copy_(_rotated(s, q.float(), hq).reshape(-1, hq * dim))
    return s["q_out"], s["k"], s["v"]


def _plain_attend(s):
    rows, h, dim, page, most = s["rows"], s["heads"], s["dim"], s["page"], s["most"]
    at = torch.arange(most, device="cuda")
    pages, inside = s["table"].long()[:, at // page], at % page
    if s["by_head"]:
        k, v = (s[n].permute(0, 2, 1, 3)[pages, inside] for n in "kv")
    else:
        k, v = (s[n][pages, inside] for n in "kv")
    length = s["len"][:, None]
    seen = at < length
    if s["window"]:
        seen = seen & (at >= length - s["window"])
    q = s["q"].float().reshape(rows, h, -1, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1).float()) / math.sqrt(dim)
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(3, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    y = torch.matmul(p, v.permute(0, 2, 1, 3).float()) / p.sum(3, keepdim=True).clamp(min=1e-30)
    return y.reshape(rows, -1).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------- the framework's calls

@functools.lru_cache(None)
def _library():
    from thnets_b200 import kernels_abi

    return kernels_abi, kernels_abi.load()


def _plan(s):
    """The descriptor of a state's operator, the entry point and the arguments that stay the same."""
    K, lib = _library()
    code = {"fp32": K.THB_F32, "fp16": K.THB_F16, "bf16": K.THB_BF16}[s["dtype"]]
    p = lambda name: s[name].data_ptr()  # noqa: E731
    if s["op"] == "norm":
        c = s["c"]
        d = K.RmsNormDesc(dtype=code, C=c, rows=s["rows"], x_ld=s["x"].stride(0), res_ld=s["x"].stride(0), sum_ld=s["x"].stride(0),
                          y_ld=s["x"].stride(0), q_ld=s["q"].stride(0), gain=p("gain"), eps=1e-5)
        res, y, q = s["has_res"], "y" in s["out"], "q" in s["out"]
        out = {}
        if res:
            out["sum"] = s["sum"][:, :c]
        if y:
            out["y"] = s["y"][:, :c]
        if q:
            out["q"], out["q_scale"] = s["q"][:, :c], s["q_scale"]
        args = (p("x"), p("res") if res else None, p("sum") if res else None, p("y") if y else None, p("q") if q else None,
                p("q_scale") if q else None)
        return lib.thb_rmsnorm_fwd, (C.byref(d),) + args, out, (d,)
    if s["op"] == "gemv":
        d = K.GemvQ4Desc(dtype=code, N=s["n"], K=s["k"], M=s["m"], group=s["group"], x_ld=s["x"].stride(0), y_ld=s["y"].stride(0),
                         w_ld=s["w"].stride(0), s_ld=s["wscale"].stride(0), z_ld=s["wzero"].stride(0), w=p("w"), wscale=p("wscale"),
                         wscale_dtype=K.THB_F16, wzero=p("wzero") if s["zeros"] else None, shift=p("shift"))
        return lib.thb_gemv_q4_fwd, (C.byref(d), p("x"), p("x_scale") if s["x8"] else None, p("y")), s["y"][:, : s["m"]], (d,)
    page_first = not s.get("by_head")
    h, dim, page = s["heads"], s["dim"], s["page"]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = K.KvCache(dtype=code, heads=h, dim=dim, pages=s["pool"], page_len=page, page_stride=page * h * dim,
                      token_stride=h * dim if page_first else dim, head_stride=dim if page_first else page * dim, k=p("k"), v=p("v"),
                      table=p("table"), table_ld=s["table"].stride(0), sequences=s["table"].shape[0], status=status.data_ptr())
    if s["op"] == "append":
        hq, ld, size = s["q_heads"], s["qkv"].stride(0), SIZE[s["dtype"]]
        d = K.KvAppendDesc(cache=cache, rope=K.Rope(dim=s["rot"], interleaved=int(s["interleaved"]), freq=p("freq"), magnitude=1.0),
                           tokens=s["tokens"], pos=p("pos"), seq=p("seq"), k_ld=ld, v_ld=ld, q_ld=ld, q_out_ld=hq * dim, q_heads=hq)
        args = (p("qkv") + hq * dim * size, p("qkv") + (hq + h) * dim * size, p("qkv"), p("q_out"))
        return lib.thb_kv_append_fwd, (C.byref(d),) + args, (s["q_out"], s["k"], s["v"]), (d, status)
    d = K.PagedAttnDesc(cache=cache, rows=s["rows"], q_heads=s["q_heads"], q_ld=s["q"].stride(0), y_ld=s["y"].stride(0), len=p("len"),
                        max_len=s["most"], window=s["window"], scale=1.0 / math.sqrt(dim))
    need = lib.thb_paged_attn_scratch(C.byref(d))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    d.scratch, d.scratch_bytes = scratch.data_ptr(), need
    return lib.thb_paged_attn_fwd, (C.byref(d), p("q"), p("y")), s["y"], (d, status, scratch)


PLAIN = {"norm": _plain_norm, "gemv": _plain_gemv, "append": _plain_append, "attend": _plain_attend}


def run(s):
    if not own:
        return PLAIN[s["op"]](s)
    if "plan" not in s:
        s["plan"] = _plan(s)
    call, args, out, _ = s["plan"]
    rc = call(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError("%s: status %d" % (s["op"], rc))
    return out


# ------------------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "norm":
        c = case["c"]
        total = s["x"].to(f64)[:, :c]
        out = {}
        if case["res"]:
            total = total + s["res"].to(f64)[:, :c]
            out["sum"] = total
        power = torch.einsum("rc,rc->r", total, total) / c
        y = torch.einsum("rc,c,r->rc", total, s["gain"].to(f64), 1.0 / torch.sqrt(power + 1e-5))
        if "y" in case["out"]:
            out["y"] = y
        if "q" in case["out"]:
            largest = torch.maximum(y.max(1).values, -y.min(1).values)
            out["q"] = (y * (E4M3_MAX / largest)[:, None]).to(torch.float8_e4m3fn).to(f64)
            out["q_scale"] = largest / E4M3_MAX
        return out
    if case["op"] == "gemv":
        k, m, group = case["k"], case["m"], case["group"]
        x = s["x"].to(f64)[:, :k]
        if case["x8"]:
            x = x * s["x_scale"].to(f64)[:, None]
        y = s["shift"].to(f64).repeat(case["n"], 1)
        for g in range((k + group - 1) // group):  # a group's columns at a time
            a, b = g * group, min(k, (g + 1) * group)
            column = torch.arange(a, b, device="cuda")
            codes = (s["w"][:, column // 2] >> (4 * (column % 2)).to(torch.uint8)) & 15
            centre = s["wzero"][:, g, None].to(f64) if case["zeros"] else 8.0
            y += (x[:, a:b] @ (codes.to(f64) - centre).T) * s["wscale"][:, g].to(f64)
        return y
    dim, h, page = case["dim"], case["heads"], case["page"]
    if case["op"] == "append":
        hq, rot = case["q_heads"], case["rot"]
        rows = s["qkv"].to(f64).reshape(case["tokens"], hq + 2 * h, dim)
        half = max(rot // 2, 0)
        i = torch.arange(half, device="cuda")
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        turn = torch.polar(torch.ones(case["tokens"], half, dtype=f64, device="cuda"), s["pos"].to(f64)[:, None] * s["freq"][:half])
        z = torch.complex(rows[:, : hq + h, first], rows[:, : hq + h, second]) * turn[:, None, :]
        rows[:, : hq + h, first], rows[:, : hq + h, second] = z.real, z.imag
        k, v = torch.zeros(s["k"].shape, dtype=f64, device="cuda"), torch.zeros(s["k"].shape, dtype=f64, device="cuda")
        place = torch.gather(s["table"].long()[s["seq"].long()], 1, (s["pos"].long() // page)[:, None])[:, 0] * page + s["pos"].long() % page
        k.view(-1, h, dim).index_copy_(0, place, rows[:, hq : hq + h])
        v.view(-1, h, dim).index_copy_(0, place, rows[:, hq + h :])
        return rows[:, :hq].reshape(case["tokens"], -1), k, v
    y = torch.zeros(case["rows"], case["q_heads"], dim, dtype=f64, device="cuda")
    share = case["q_heads"] // h
    for r, length in enumerate(s["len"].tolist()):
        start = max(0, length - case["window"]) if case["window"] else 0
        if start >= length:
            continue
        pages = s["table"][r].long()[: (length + page - 1) // page]
        for j in range(h):
            if case["by_head"]:
                k, v = (s[n][pages, j].reshape(-1, dim)[start:length].to(f64) for n in "kv")
            else:
                k, v = (s[n][pages][:, :, j].reshape(-1, dim)[start:length].to(f64) for n in "kv")
            q = s["q"].to(f64).reshape(case["rows"], -1, dim)[r, j * share : (j + 1) * share]
            y[r, j * share : (j + 1) * share] = torch.softmax(q @ k.T * dim ** -0.5, 1) @ v
    return y.reshape(case["rows"], -1)
