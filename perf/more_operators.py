"""The operators of projections in 8-bit floating point (e4m3) with a scale for
each block of 128 (bf16 beside rows, f32 beside weights as checkpoints hold them), as cases that can be timed and checked: the quantizer of rows,
the RMSNorm with the residual's addition whose output is in 8 bits, the product,
the gated product whose result is in 8 bits again, and both products over the
groups of a mixture of experts.

A case is a dict of plain values. prepare() makes what a program has in hand
(inputs, weights, a plan), run() is one pass: the plain form in elementary
torch operations where `own` is false, the library's calls where it is true.
exact() is each operator's definition in 64 bits.

Codes are returned as float8 tensors, their scales beside them.
"""
import math
import os
import sys
import zlib

import numpy as np
import torch

# True: run() calls the library. False: run() computes the plain form.
own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HID, FFN, CAP = 3840, 10240, 2560      # the image model's widths and the encoder's
F8 = torch.float8_e4m3fn
MOST = 448.0                           # the largest e4m3 value
TINY = 2.0 ** -100                     # a block's largest value counts as this at least
EPS = 1e-6


# ---- the cases -----------------------------------------------------------------
def listed():
    return [
        # eight prompts' next tokens: attention's rows before the o projection
        {"name": "quantize_8x3840", "op": "quantize", "rows": 8, "D": HID},
        # the same over two images of 1024 x 1024 with their captions
        {"name": "quantize_8704x3840", "op": "quantize", "rows": 8704, "D": HID},
        # one prompt's next token: the residual joined and the next norm
        {"name": "norm_1x2560_add", "op": "norm", "rows": 1, "D": CAP, "add": True, "y": False},
        # a prompt of odd length into a layer whose router reads the bf16 norm
        {"name": "norm_203x2048_y", "op": "norm", "rows": 203, "D": 2048, "add": False, "y": True},
        # two images' rows: the residual joined and the next norm
        {"name": "norm_8704x3840_add", "op": "norm", "rows": 8704, "D": HID, "add": True,
         "y": False},
        # one next token through a projection: the weights are read once
        {"name": "lin_1_3840x3840", "op": "lin", "M": 1, "N": HID, "K": HID, "bias": False},
        # a caption of odd length, a biased projection out of the wide layer
        {"name": "lin_203_2560x10240_bias", "op": "lin", "M": 203, "N": CAP, "K": FFN,
         "bias": True},
        # two images' rows out of the feed-forward
        {"name": "lin_8704_3840x10240", "op": "lin", "M": 8704, "N": HID, "K": FFN, "bias": False},
        # eight next tokens through gate and up
        {"name": "swiglu_8_10240x3840", "op": "swiglu", "M": 8, "N": FFN, "K": HID},
        # an image of 1024 x 1024 with its caption through gate and up
        {"name": "swiglu_4352_10240x3840", "op": "swiglu", "M": 4352, "N": FFN, "K": HID},
        # the next tokens of eight prompts through the experts' gate and up
        {"name": "experts_swiglu_8x8_of_64", "op": "experts_swiglu", "tokens": 8, "k": 8,
         "experts": 64, "N": 1024, "K": 2048},
        # a long batch through the experts' down product
        {"name": "experts_lin_4352x8_of_64", "op": "experts_lin", "tokens": 4352, "k": 8,
         "experts": 64, "N": 2048, "K": 1024},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "norm", "lin", "lin", "lin", "swiglu", "swiglu",
                     "experts_swiglu", "experts_lin"])
    if op in ("quantize", "norm"):
        c = {"op": op, "rows": _log(rng, 1, 8704), "D": 16 * _log(rng, 8, 512)}
        if op == "norm":
            c["add"], c["y"] = rng.random() < 0.6, rng.random() < 0.4
        while c["rows"] * c["D"] > 8704 * HID:
            c["rows"] //= 2
        return c
    if op in ("lin", "swiglu"):
        N, K = rng.choice([(HID, HID), (FFN, HID), (HID, FFN), (CAP, CAP),
                           (16 * _log(rng, 4, 640), 16 * _log(rng, 8, 640))])
        M, wide = _log(rng, 1, 8704), N * (2 if op == "swiglu" else 1)
        M = max(1, min(M, 8704 * FFN * HID // (wide * K)))
        c = {"op": op, "M": M, "N": N, "K": K}
        if op == "lin":
            c["bias"] = rng.random() < 0.3
        return c
    while True:
        c = {"op": op, "tokens": _log(rng, 1, 4352), "k": rng.randint(1, 8),
             "experts": _log(rng, 2, 256), "N": 16 * _log(rng, 8, 160),
             "K": 16 * _log(rng, 8, 200)}
        c["k"] = min(c["k"], c["experts"])
        wide = c["N"] * (2 if op == "experts_swiglu" else 1)
        if (c["experts"] * wide * c["K"] <= 64 * 2048 * 2048
                and c["tokens"] * c["k"] * wide * c["K"] <= 34816 * 2048 * 2048):
            return c


# ---- inputs, from the seed alone -------------------------------------------------
def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(tag.encode())) % (1 << 62))
    return g


def _randn(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _rows(g, rows, D):
    """Activations: rows of unequal size, some columns far larger than others."""
    t = _randn(g, (rows, D)) * torch.exp(_randn(g, (D,), 0.5)) * torch.exp(_randn(g, (rows, 1), 0.3))
    return t.to(torch.bfloat16)


def _blocks(n):
    return (n + 127) // 128


def _scale_up(t):
    """The least bf16 value of at least t (64-bit, positive)."""
    s = t.float().to(torch.bfloat16)
    return torch.where(s.double() < t, (s.view(torch.int16) + 1).view(torch.bfloat16), s)


def _codes_of_rows(t):
    """[rows][D] -> codes [rows][D] and bf16 scales [blocks][rows], as the quantizer has them.
    In 64 bits: values often lie on the border of two codes (a ratio of 8-bit values)."""
    rows, D = t.shape
    p = torch.nn.functional.pad(t.double(), (0, _blocks(D) * 128 - D)).view(rows, -1, 128)
    s = _scale_up(p.abs().amax(-1).clamp(min=TINY) / MOST)
    q = (p / s.double()[..., None]).float().to(F8).view(rows, -1)
    return q[:, :D].contiguous(), s.t().contiguous()


def _weight(seed, tag, shape, halves):
    """Projections [..., halves * N, K] as a checkpoint holds them: codes, and a scale for
    each 128 x 128 block of every half, [..., halves * blocks of N, blocks of K]."""
    E, N, K = shape
    g = _gen(seed, tag)
    codes, scales = [], []
    nb, kb = _blocks(N), _blocks(K)
    for _ in range(halves):
        # blocks of unequal size
        w = _randn(g, (E, nb, 128, kb, 128), 1.0 / math.sqrt(K))
        w *= torch.exp(_randn(g, (E, nb, 1, kb, 1), 0.2))
        w.view(E, nb * 128, kb * 128)[:, N:] = 0.0
        w.view(E, nb * 128, kb * 128)[:, :, K:] = 0.0
        top = w.abs().amax((2, 4), keepdim=True).clamp(min=TINY)
        q = (w * MOST / top).to(F8).view(E, nb * 128, kb * 128)[:, :N, :K]
        codes.append(q.contiguous().view(torch.uint8))
        scales.append((top / MOST).view(E, nb, kb))
    return {"codes": torch.cat(codes, 1).contiguous().view(F8),
            "scales": torch.cat(scales, 1).contiguous(), "N": N, "K": K, "halves": halves}


def _plan(seed, tokens, k, experts):
    """Each token's k experts, none twice, some more popular, in expert order."""
    r = np.random.default_rng([int(seed) & 0x7FFFFFFF, zlib.crc32(b"choices")])
    key = r.normal(0.0, 0.7, experts)[None, :] + r.gumbel(size=(tokens, experts))
    flat = np.argsort(-key, axis=1, kind="stable")[:, :k].astype(np.int32).reshape(-1)
    counts = np.bincount(flat, minlength=experts)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return offsets, np.argsort(flat, kind="stable").astype(np.int32), counts


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _inputs(c, seed):
    op, g = c["op"], _gen(seed, "x")
    if op == "quantize":
        return {"x": _rows(g, c["rows"], c["D"])}
    if op == "norm":
        return {"x": _rows(g, c["rows"], c["D"]),
                "sub": _rows(g, c["rows"], c["D"]) if c["add"] else None,
                "w": (1.0 + _randn(g, (c["D"],), 0.2)).to(torch.bfloat16)}
    gated = op in ("swiglu", "experts_swiglu")
    if op in ("lin", "swiglu"):
        x, xs = _codes_of_rows(_rows(g, c["M"], c["K"]))
        d = {"x": x, "xs": xs, "w": _weight(seed, "w", (1, c["N"], c["K"]), 2 if gated else 1)}
        d["bias"] = _randn(g, (c["N"],), 0.5).to(torch.bfloat16) if c.get("bias") else None
        return d
    n = c["tokens"] * c["k"]
    offsets, order, counts = _plan(seed, c["tokens"], c["k"], c["experts"])
    # gate and up read the tokens' rows, the down product rows in expert order
    x, xs = _codes_of_rows(_rows(g, c["tokens"] if gated else n, c["K"]))
    return {"x": x, "xs": xs, "counts": counts, "offsets": _dev(offsets),
            "order": _dev(order) if gated else None,
            "w": _weight(seed, "w", (c["experts"], c["N"], c["K"]), 2 if gated else 1)}


# ---- what a program keeps ----------------------------------------------------------
class State:
    pass


_kept = {}


def _library():
    """The program's one context, on a stream of its own."""
    if not _kept:
        sys.path.insert(0, os.path.join(ROOT, "vpipe-ming-image_amd"))
        import ming_dit_amd as m
        _kept["m"] = m
        _kept["stream"] = torch.cuda.Stream()
        _kept["ctx"] = m.Ctx(0, _kept["stream"].cuda_stream)
    return _kept["m"], _kept["ctx"]


def _empty(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    st = State()
    st.c, st.d = case, _inputs(case, seed)
    if own:
        _handles(st)
    return st


def _handles(st):
    """Resident weights, output planes and workspaces of the library's calls."""
    c, d, op = st.c, st.d, st.c["op"]
    m, ctx = _library()
    torch.cuda.synchronize()      # the library reads the inputs on its own stream
    if op in ("quantize", "norm"):
        rows, wide = c["rows"], c["D"]
        if op == "norm":
            st.h = _empty(rows, wide) if c["add"] else None
            st.y = _empty(rows, wide) if c["y"] else None
    else:
        rows = c["M"] if "M" in c else c["tokens"] * c["k"]
        wide = c["N"]
        st.w = m.F8(ctx, d["w"]["codes"], d["w"]["scales"], wide, gated=d["w"]["halves"] == 2,
                    on_device=True)
        st.ws = _empty(max(1, st.w.workspace_bytes(rows)), dtype=torch.uint8)
        st.n = rows
    if op in ("lin", "experts_lin"):
        st.y = _empty(rows, wide)
    else:
        st.codes = _empty(rows, wide, dtype=F8)
        st.scales = _empty(_blocks(wide), rows)
    ctx.synchronize()


def run(st):
    if own:
        return _own(st)
    return {"quantize": _quantize, "norm": _norm, "lin": _lin, "swiglu": _swiglu,
            "experts_lin": _experts, "experts_swiglu": _experts}[st.c["op"]](st.c, st.d)


def _own(st):
    c, d, op = st.c, st.d, st.c["op"]
    ctx = _kept["ctx"]
    if op == "quantize":
        ctx.f8_quantize(d["x"], c["rows"], c["D"], st.codes, st.scales)
        return [st.codes, st.scales]
    if op == "norm":
        ctx.f8_rmsnorm(d["x"], d["w"], c["rows"], c["D"], st.codes, st.scales, sub=d["sub"],
                       h=st.h, y=st.y, eps=EPS)
        return [st.h, st.y, st.codes, st.scales]
    if op == "lin":
        ctx.f8_lin(st.w, d["x"], d["xs"], st.y, c["M"], bias=d["bias"], ws=st.ws)
        return st.y
    if op == "swiglu":
        ctx.f8_swiglu(st.w, d["x"], d["xs"], st.codes, st.scales, c["M"], ws=st.ws)
        return [st.codes, st.scales]
    if op == "experts_lin":
        ctx.f8_experts_lin(st.w, d["x"], d["xs"], st.n, None, d["offsets"], st.n, st.y, ws=st.ws)
        return st.y
    ctx.f8_experts_swiglu(st.w, d["x"], d["xs"], c["tokens"], d["order"], d["offsets"], st.n,
                          st.codes, st.scales, fan=c["k"], ws=st.ws)
    return [st.codes, st.scales]


# ---- the plain forms ------------------------------------------------------------------
def _f32(x, xs):
    """Rows in 32 bits: code * scale."""
    return x.float() * xs.float().t().repeat_interleave(128, 1)[:, :x.shape[1]]


def _w32(w):
    """Projections in 32 bits [E][halves * N][K]."""
    nb = _blocks(w["N"])
    s = w["scales"].view(-1, w["halves"], nb, w["scales"].shape[-1])
    s = s.repeat_interleave(128, 2)[:, :, :w["N"]].repeat_interleave(128, 3)[..., :w["K"]]
    return w["codes"].float() * s.flatten(1, 2)


def _quantize(c, d):
    return list(_codes_of_rows(d["x"]))


def _norm(c, d):
    h = d["x"]
    if c["add"]:
        h = (h.float() + d["sub"].float()).to(torch.bfloat16)
    v = h.float()
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * d["w"].float()
    return [h if c["add"] else None, v.to(torch.bfloat16) if c["y"] else None, *_codes_of_rows(v)]


def _lin(c, d):
    y = _f32(d["x"], d["xs"]) @ _w32(d["w"])[0].t()
    return (y if d["bias"] is None else y + d["bias"].float()).to(torch.bfloat16)


def _swiglu(c, d):
    y = _f32(d["x"], d["xs"]) @ _w32(d["w"])[0].t()
    g, u = y[:, :c["N"]], y[:, c["N"]:]
    return list(_codes_of_rows(g / (1.0 + torch.exp(-g)) * u))


def _experts(c, d):
    """Each expert's rows side by side, padded to the most any expert has."""
    n, cap = c["tokens"] * c["k"], int(d["counts"].max())
    off = d["offsets"].long()
    p = (off[:-1, None] + torch.arange(cap, device="cuda")).clamp(max=n - 1)
    src = p if d["order"] is None else d["order"].long()[p] // c["k"]
    y = torch.bmm(_f32(d["x"], d["xs"])[src], _w32(d["w"]).transpose(1, 2).contiguous())
    p = torch.arange(n, device="cuda")
    e = torch.searchsorted(off[1:], p, right=True)
    y = y[e, p - off[e]]
    if c["op"] == "experts_lin":
        return y.to(torch.bfloat16)
    g, u = y[:, :c["N"]], y[:, c["N"]:]
    return list(_codes_of_rows(g / (1.0 + torch.exp(-g)) * u))


# ---- the work a pass cannot do without ---------------------------------------------------
def work(case):
    c, op = case, case["op"]
    if op in ("quantize", "norm"):
        n = float(c["rows"]) * c["D"]
        each = 3.0 if op == "quantize" else 3.0 + (4.0 if c["add"] else 0.0) + (2.0 if c["y"] else 0.0)
        return {"bytes": each * n + 2.0 * c["rows"] * _blocks(c["D"]) + 2.0 * c["D"] * (op == "norm"),
                "flops": (4.0 if op == "quantize" else 8.0) * n}
    gated = op in ("swiglu", "experts_swiglu")
    N, K = c["N"], c["K"]
    wide = N * (2 if gated else 1)
    n = c["M"] if "M" in c else c["tokens"] * c["k"]
    rows = c["tokens"] if op == "experts_swiglu" else n
    E = c.get("experts", 1)
    live = E * (1.0 - (1.0 - 1.0 / E) ** n) if E > 1 else 1.0     # experts with a row, about
    out = n * (N + 2.0 * _blocks(N)) if gated else 2.0 * n * N
    return {"bytes": live * (wide * K + wide / 32.0 * _blocks(K)) + rows * (K + 2.0 * _blocks(K))
            + out + (2.0 * N if c.get("bias") else 0.0) + (4.0 * n if E > 1 else 0.0),
            "flops": 2.0 * n * wide * K}


# ---- the definitions in 64 bits ------------------------------------------------------------
def _e4m3_64(v):
    """The nearest e4m3 value of |v| <= 448 in 64 bits, ties to even: steps of 2^(e - 3) in
    [2^e, 2^(e + 1)), of 2^-9 below 2^-6."""
    a = v.abs().clamp(min=2.0 ** -6)
    step = a / torch.frexp(a)[0] / 16.0           # 2^(e + 1) / 16
    return torch.round(v / step) * step


def _quantize64(v):
    """Codes and scales of 64-bit rows, block by block. The codes go by the scale as it is
    stored, in bf16 and not below the largest value's 448th; that 448th is returned."""
    codes, scales = torch.empty_like(v), []
    for a in range(0, v.shape[1], 128):
        b = v[:, a:a + 128]
        s = torch.clamp(b.abs().max(1, keepdim=True).values, min=TINY) / 448.0
        m = torch.frexp(s)[0]
        kept = torch.ceil(m * 256.0) / 256.0 * (s / m)            # 8 bits
        codes[:, a:a + 128] = _e4m3_64(b / kept)
        scales.append(s[:, 0])
    return [codes, torch.stack(scales)]


def _product64(x, xs, w, e, half):
    """x . W_e^T of one half's rows, block by block of K."""
    N, nb = w["N"], _blocks(w["N"])
    codes = w["codes"][e, half * N:(half + 1) * N].double()
    sc = w["scales"][e, half * nb:(half + 1) * nb].double()
    col = torch.arange(N, device="cuda") // 128
    y = torch.zeros((x.shape[0], N), dtype=torch.float64, device="cuda")
    for b in range(xs.shape[0]):
        part = x[:, 128 * b:128 * b + 128].double() @ codes[:, 128 * b:128 * b + 128].t()
        y += part * xs[b].double()[:, None] * sc[col, b]
    return y


def exact(case, seed):
    c, op = case, case["op"]
    d = _inputs(c, seed)
    if op == "quantize":
        return _quantize64(d["x"].double())
    if op == "norm":
        h = d["x"].double()
        if c["add"]:
            h = (h + d["sub"].double())
        # the sum that goes on is the stored one
        kept = h.to(torch.bfloat16).double() if c["add"] else h
        v = kept / torch.sqrt(kept.square().mean(1, keepdim=True) + EPS) * d["w"].double()
        return [h if c["add"] else None, v if c["y"] else None, *_quantize64(v)]
    gated = op in ("swiglu", "experts_swiglu")
    if op in ("lin", "swiglu"):
        y = _product64(d["x"], d["xs"], d["w"], 0, 0)
        if not gated:
            return y if d["bias"] is None else y + d["bias"].double()
        return _quantize64(torch.nn.functional.silu(y) * _product64(d["x"], d["xs"], d["w"], 0, 1))
    n, ends = c["tokens"] * c["k"], np.cumsum(d["counts"])
    y = torch.zeros((n, c["N"]), dtype=torch.float64, device="cuda")
    for e in np.flatnonzero(d["counts"]):
        a, b = int(ends[e] - d["counts"][e]), int(ends[e])
        at = slice(a, b) if d["order"] is None else d["order"][a:b].long() // c["k"]
        x, xs = d["x"].view(torch.uint8)[at].view(F8), d["xs"][:, at].contiguous()
        t = _product64(x, xs, d["w"], e, 0)
        y[a:b] = torch.nn.functional.silu(t) * _product64(x, xs, d["w"], e, 1) if gated else t
    return _quantize64(y) if gated else y
