"""The operators whose rows choose their own weights, as cases that can be
timed and checked: the router that chooses each token's experts, the grouping
of its choices by expert, the experts' ragged products (plain and SwiGLU-gated),
the weighted sum that brings the rows back to their tokens, and a projection
whose rows carry the low-rank adapters of many requests.

A case is a dict of plain values. prepare() makes what a program has in hand
(inputs, weights, a plan), run() is one pass: the plain form in elementary
torch operations where `own` is false, the library's calls where it is true.
exact() is each operator's definition in 64 bits.
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
HID, FFN = 3840, 10240         # the image model's widths
FLT_MAX = 3.4028234663852886e38

# Adapter sets: the ranks in a bank, by turns, and how many adapters it holds.
BANKS = {
    "one": ((16,), 1),
    "four": ((16, 32, 64, 16), 4),
    "odd": ((4, 12, 20, 7, 33), 11),
    "many": ((16, 16, 8, 32), 32),
    "wide": ((64, 128), 6),
}


# ---- the cases -----------------------------------------------------------------
def listed():
    return [
        # a few prompts' next tokens through the router: 256 experts in eight
        # groups, of which four may serve a token, sigmoid scores with a
        # balancing bias, logits as a bf16 projection leaves them
        {"name": "route_sigmoid_bf16_8", "op": "route", "rows": 8, "experts": 256, "k": 8,
         "groups": 8, "top_groups": 4, "score": "sigmoid", "bias": True, "f32": False,
         "normalize": True, "masked": False},
        # a batch of prompts (odd length), 60 experts of which some are taken
        # out of service, softmax scores, f32 logits
        {"name": "route_softmax_f32_4099", "op": "route", "rows": 4099, "experts": 60, "k": 6,
         "groups": 1, "top_groups": 1, "score": "softmax", "bias": False, "f32": True,
         "normalize": False, "masked": True},
        # the next tokens' choices in expert order: one small launch
        {"name": "group_64_of_256", "op": "group", "n": 64, "groups": 256, "dropped": 0.0},
        # a long batch's choices, an eighth of them dropped (no expert)
        {"name": "group_34816_of_64", "op": "group", "n": 34816, "groups": 64, "dropped": 0.125},
        # the next tokens of eight prompts through the experts' gate and up
        # products: most experts idle or with one row
        {"name": "swiglu_dense_8x8_of_64", "op": "swiglu", "bits": 16, "tokens": 8, "k": 8,
         "experts": 64, "K": 2048, "N": 1024},
        # the experts' down product over a prompt of odd length, w8
        {"name": "lin_w8_203x6_of_60", "op": "lin", "bits": 8, "tokens": 203, "k": 6,
         "experts": 60, "K": 1024, "N": 2048},
        # gate and up over a batch of prompts, a w4 pack, many experts
        {"name": "swiglu_w4_2048x8_of_128", "op": "swiglu", "bits": 4, "tokens": 2048, "k": 8,
         "experts": 128, "K": 2048, "N": 512},
        # the same over a long batch, bf16 weights
        {"name": "swiglu_dense_4352x8_of_64", "op": "swiglu", "bits": 16, "tokens": 4352, "k": 8,
         "experts": 64, "K": 2048, "N": 1024},
        # the next tokens' expert rows back to their tokens
        {"name": "combine_8x8", "op": "combine", "tokens": 8, "k": 8, "N": 2048, "add": False},
        # a long batch's, onto the shared expert's output
        {"name": "combine_4352x8_add", "op": "combine", "tokens": 4352, "k": 8, "N": 2048,
         "add": True},
        # 37 short rows of 32 requests, each with its own adapter, over an
        # unquantized projection
        {"name": "adapters_dense_37_many", "op": "adapters", "bits": 16, "M": 37, "N": HID,
         "K": HID, "bank": "many", "requests": 32},
        # two images of 1024 x 1024 with their captions, five requests' rows
        # with four adapters, over the w4 feed-forward's first projection
        {"name": "adapters_w4_8704_four", "op": "adapters", "bits": 4, "M": 8704, "N": FFN,
         "K": HID, "bank": "four", "requests": 5},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "group", "swiglu", "swiglu", "lin", "combine", "adapters",
                     "adapters"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log(rng, 2, 512 // groups)
        top_groups = rng.randint(1, groups)
        return {"op": op, "rows": _log(rng, 1, 8192), "experts": experts,
                "k": rng.randint(1, min(16, experts // groups * top_groups)), "groups": groups,
                "top_groups": top_groups, "score": rng.choice(["sigmoid", "softmax"]),
                "bias": rng.random() < 0.5, "f32": rng.random() < 0.5,
                "normalize": rng.random() < 0.6, "masked": rng.random() < 0.3}
    if op == "group":
        return {"op": op, "n": _log(rng, 1, 262144), "groups": _log(rng, 1, 1024),
                "dropped": rng.choice([0.0, 0.0, 0.3])}
    if op in ("swiglu", "lin"):
        bits = rng.choice([4, 8, 16, 16])
        while True:
            c = {"op": op, "bits": bits, "tokens": _log(rng, 1, 4352), "k": rng.randint(1, 8),
                 "experts": _log(rng, 2, 256), "K": 64 * _log(rng, 2, 60),
                 "N": 8 * _log(rng, 8, 400)}
            c["k"] = min(c["k"], c["experts"])
            wide = c["N"] * (2 if op == "swiglu" else 1)
            if (c["experts"] * wide * c["K"] <= 64 * 2048 * 2048
                    and c["tokens"] * c["k"] * wide * c["K"] <= 34816 * 2048 * 2048):
                return c
    if op == "combine":
        return {"op": op, "tokens": _log(rng, 1, 4352), "k": rng.randint(1, 8),
                "N": 8 * _log(rng, 8, 512), "add": rng.random() < 0.5}
    N, K = rng.choice([(HID, HID), (HID, HID), (FFN, HID), (HID, FFN),
                       (8 * _log(rng, 8, 640), 64 * _log(rng, 2, 80))])
    M = _log(rng, 1, 8704)
    if M * N * K > 8704 * FFN * HID:
        M = 8704 * FFN * HID // (N * K)
    return {"op": op, "bits": rng.choice([4, 4, 8, 16]), "M": M, "N": N, "K": K,
            "bank": rng.choice(sorted(BANKS)), "requests": min(M, _log(rng, 1, 48))}


# ---- inputs, from the seed alone -------------------------------------------------
def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(tag.encode())) % (1 << 62))
    return g


def _rng(seed, tag):
    return np.random.default_rng([int(seed) & 0x7FFFFFFF, zlib.crc32(tag.encode())])


def _randn(g, shape, std=1.0, mean=0.0):
    t = torch.randn(shape, generator=g, device="cuda")
    return (t * std + mean if (std != 1.0 or mean) else t).to(torch.bfloat16)


def _weight(seed, tag, shape, bits):
    """Projections [..., N, K] as a checkpoint holds them: dense bf16, or
    group-64 codes (LSB-first words) with bf16 scales and biases."""
    g = _gen(seed, tag)
    K = shape[-1]
    if bits == 16:
        return {"w": _randn(g, shape, 1.0 / math.sqrt(K))}
    w = torch.randn(shape[:-1] + (K // 64, 64), generator=g, device="cuda") * 0.02
    if bits == 4:
        lo = w.amin(-1)
        s = ((w.amax(-1) - lo) / 15.0).to(torch.bfloat16)
        b = lo.to(torch.bfloat16)
        q = torch.round((w - b.float()[..., None]) / s.float()[..., None]).clamp_(0, 15)
    else:
        s = (w.abs().amax(-1) / 127.0).to(torch.bfloat16)
        b = (s.float() * -128.0).to(torch.bfloat16)
        q = torch.round(w / s.float()[..., None]).clamp_(-127, 127) + 128
    per = 32 // bits
    q = q.to(torch.int32).reshape(shape[:-1] + (K // per, per))
    shift = torch.arange(per, device="cuda", dtype=torch.int32) * bits
    # the fields of a word do not overlap: their sum is the word
    words = (q << shift).sum(-1, dtype=torch.int32)
    return {"codes": words, "scales": s, "biases": b, "bits": bits, "shift": shift}


def _choices(seed, tokens, k, experts):
    """Each token's k experts, none twice, some experts more popular."""
    r = _rng(seed, "choices")
    pop = r.normal(0.0, 0.7, experts)
    key = pop[None, :] + r.gumbel(size=(tokens, experts))
    return np.argsort(-key, axis=1, kind="stable")[:, :k].astype(np.int32)


def _plan(ids, experts):
    """The choices in expert order: (offsets, order, place) over flat indices."""
    flat = ids.reshape(-1)
    order = np.argsort(flat, kind="stable").astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts))])
    place = np.empty(flat.size, np.int32)
    place[order] = np.arange(flat.size, dtype=np.int32)
    return offsets.astype(np.int32), order, place


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _inputs(c, seed):
    op, g = c["op"], _gen(seed, "x")
    if op == "route":
        E = c["experts"]
        l = torch.randn((c["rows"], E), generator=g, device="cuda") * 1.5
        l += torch.randn((E,), generator=g, device="cuda")
        if c["masked"]:
            # experts out of service, for everyone or for some tokens
            off = torch.rand((c["rows"], E), generator=g, device="cuda") < 0.1
            off[:, E // 2] = True
            l = l.masked_fill(off, -math.inf)
        return {"logits": l if c["f32"] else l.to(torch.bfloat16),
                "bias": torch.randn((E,), generator=g, device="cuda") * 0.05 if c["bias"] else None}
    if op == "group":
        r = _rng(seed, "ids")
        pop = np.exp(r.normal(0.0, 0.7, c["groups"]))
        ids = r.choice(c["groups"], size=c["n"], p=pop / pop.sum()).astype(np.int32)
        ids[r.random(c["n"]) < c["dropped"]] = -1
        return {"ids": _dev(ids)}
    if op in ("swiglu", "lin"):
        E, K, n = c["experts"], c["K"], c["tokens"] * c["k"]
        offsets, order, _ = _plan(_choices(seed, c["tokens"], c["k"], E), E)
        N = c["N"] * 2 if op == "swiglu" else c["N"]     # gate rows, then up rows
        return {"x": _randn(g, (c["tokens"] if op == "swiglu" else n, K)),
                "w": _weight(seed, "w", (E, N, K), c["bits"]), "counts": np.diff(offsets),
                "offsets": _dev(offsets), "order": _dev(order) if op == "swiglu" else None}
    if op == "combine":
        _, _, place = _plan(_choices(seed, c["tokens"], c["k"], 64), 64)
        w = torch.rand((c["tokens"], c["k"]), generator=g, device="cuda") + 0.05
        return {"y": _randn(g, (c["tokens"] * c["k"], c["N"])), "place": _dev(place),
                "weights": w / w.sum(1, keepdim=True) * 2.5,
                "add": _randn(g, (c["tokens"], c["N"])) if c["add"] else None}
    # adapters: the requests' rows one after another, each request with an
    # adapter of the bank and a strength, some with none
    r = _rng(seed, "requests")
    M, N, K = c["M"], c["N"], c["K"]
    ranks, held = BANKS[c["bank"]]
    ranks = [ranks[i % len(ranks)] for i in range(held)]
    cuts = np.sort(r.choice(np.arange(1, M), size=c["requests"] - 1, replace=False)) \
        if c["requests"] > 1 else np.empty(0, np.int64)
    lengths = np.diff(np.concatenate([[0], cuts, [M]]))
    ids = r.permutation(np.arange(c["requests"]) % held)
    ids[r.random(c["requests"]) < 0.15] = -1
    strength = r.choice([1.0, 0.8, 0.5, 1.2, -0.3], size=c["requests"])
    R = sum(ranks)
    return {"x": _randn(g, (M, K)), "w": _weight(seed, "w", (N, K), c["bits"]),
            "A": _randn(g, (R, K), 1.0 / math.sqrt(K)), "B": _randn(g, (N, R), 0.05),
            "ranks": ranks, "col": _dev(np.repeat(np.arange(held), ranks).astype(np.int32)),
            "ids": _dev(np.repeat(ids, lengths).astype(np.int32)),
            "scale": _dev(np.repeat(strength, lengths).astype(np.float32))}


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
    if op == "route":
        st.ids = _empty(c["rows"], c["k"], dtype=torch.int32)
        st.w = _empty(c["rows"], c["k"], dtype=torch.float32)
    elif op == "group":
        st.offsets = _empty(c["groups"] + 1, dtype=torch.int32)
        st.order, st.place = (_empty(c["n"], dtype=torch.int32) for _ in range(2))
        st.ws = _empty(max(1, m.group_rows_workspace_bytes(c["n"], c["groups"])),
                       dtype=torch.uint8)
    elif op in ("swiglu", "lin"):
        w = d["w"]
        st.ex = m.Experts.dense(ctx, w["w"], on_device=True) if "w" in w else \
            m.Experts.quantized(ctx, w["codes"], w["scales"], w["biases"], w["bits"],
                                on_device=True)
        st.y = _empty(c["tokens"] * c["k"], c["N"])
        st.ws = _empty(max(1, st.ex.workspace_bytes(d["x"].shape[0])), dtype=torch.uint8)
    elif op == "combine":
        st.out = _empty(c["tokens"], c["N"])
    else:
        w = d["w"]
        st.qw = m.QWeight.dense(ctx, w["w"], on_device=True) if "w" in w else \
            m.QWeight.quantized(ctx, w["codes"], w["scales"], w["biases"], w["bits"],
                                on_device=True)
        st.bank = m.Adapters(ctx, c["N"], c["K"], len(d["ranks"]), max(d["ranks"]))
        at = 0
        for i, r in enumerate(d["ranks"]):
            st.bank.set(i, d["A"][at:at + r].contiguous(), d["B"][:, at:at + r].contiguous(),
                        on_device=True)
            at += r
        st.y = _empty(c["M"], c["N"])
        st.ws = _empty(max(1, ctx.lin_adapters_workspace_bytes(st.qw, st.bank, c["M"])),
                       dtype=torch.uint8)
    ctx.synchronize()


def run(st):
    if own:
        return _own(st)
    return {"route": _route, "group": _group, "swiglu": _experts, "lin": _experts,
            "combine": _combine, "adapters": _adapters}[st.c["op"]](st.c, st.d)


def _own(st):
    c, d, op = st.c, st.d, st.c["op"]
    ctx = _kept["ctx"]
    if op == "route":
        ctx.topk_route(d["logits"], c["rows"], c["experts"], c["k"], st.ids, st.w, bias=d["bias"],
                       n_groups=c["groups"], top_groups=c["top_groups"], score=c["score"],
                       normalize=c["normalize"], scale=2.5)
        return [st.ids, st.w]
    if op == "group":
        ctx.group_rows(d["ids"], c["n"], c["groups"], st.offsets, st.order, st.place, st.ws)
        return [st.offsets, st.order, st.place]
    if op == "swiglu":
        ctx.experts_swiglu(st.ex, d["x"], c["tokens"], d["order"], d["offsets"],
                           c["tokens"] * c["k"], st.y, fan=c["k"], ws=st.ws)
        return st.y
    if op == "lin":
        ctx.experts_lin(st.ex, d["x"], c["tokens"] * c["k"], None, d["offsets"],
                        c["tokens"] * c["k"], st.y, ws=st.ws)
        return st.y
    if op == "combine":
        ctx.experts_combine(st.d["y"], c["tokens"] * c["k"], d["place"], d["weights"], c["tokens"],
                            c["k"], st.out, c["N"], add=d["add"])
        return st.out
    ctx.lin_adapters(st.qw, st.bank, d["x"], st.y, c["M"], d["ids"], d["scale"], st.ws)
    return st.y


# ---- the plain forms ------------------------------------------------------------------
def _f32(w):
    """A projection in 32 bits: the dense values, or scale * code + bias."""
    if "w" in w:
        return w["w"].float()
    q = (w["codes"][..., None] >> w["shift"]) & ((1 << w["bits"]) - 1)
    s, b = w["scales"].float(), w["biases"].float()
    q = q.reshape(s.shape + (64,)).float()
    return (q * s[..., None] + b[..., None]).flatten(-2)


def _route(c, d):
    # in 64 bits: a choice goes by the difference of two scores
    l = d["logits"].double()
    ok = l > -math.inf
    l = l.clamp(max=FLT_MAX)
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        top = torch.where(ok, l, -math.inf).amax(1, keepdim=True)
        e = torch.where(ok, torch.exp(l - top), 0.0)
        s = e / e.sum(1, keepdim=True)
    key = s if d["bias"] is None else s + d["bias"].double()
    key = torch.where(ok, key, -math.inf)
    if c["groups"] > 1:
        per = key.view(key.shape[0], c["groups"], -1)
        two = per.sort(dim=-1, descending=True).values[..., :2]
        score = torch.where(two > -math.inf, two, 0.0).sum(-1)
        score = torch.where(two[..., 0] > -math.inf, score, -math.inf)
        best = score.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        may = torch.zeros_like(score, dtype=torch.bool).scatter_(1, best, True)
        key = torch.where(may[..., None], per, -math.inf).flatten(1)
    val, ids = key.sort(dim=1, descending=True, stable=True)
    val, ids = val[:, :c["k"]], ids[:, :c["k"]]
    chosen = val > -math.inf
    w = torch.where(chosen, s.gather(1, ids), 0.0)
    if c["normalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0.0, w / total, 0.0)
    return [torch.where(chosen, ids, -1).to(torch.int32), (w * 2.5).float()]


def _group(c, d):
    G, n = c["groups"], c["n"]
    ids = d["ids"].long()
    key, order = torch.where((ids >= 0) & (ids < G), ids, G).sort(stable=True)
    offsets = torch.searchsorted(key, torch.arange(G + 1, device="cuda"))
    p = torch.arange(n, device="cuda")
    place = torch.empty_like(order).scatter_(0, order, torch.where(key < G, p, -1))
    order = torch.where(key < G, order, -1)
    return [offsets.to(torch.int32), order.to(torch.int32), place.to(torch.int32)]


def _experts(c, d):
    """Each expert's rows side by side, padded to the most any expert has."""
    n, cap = c["tokens"] * c["k"], int(d["counts"].max())
    off = d["offsets"].long()
    p = (off[:-1, None] + torch.arange(cap, device="cuda")).clamp(max=n - 1)
    src = p if d["order"] is None else d["order"].long()[p] // c["k"]
    y = torch.bmm(d["x"].float()[src], _f32(d["w"]).transpose(1, 2).contiguous())
    if c["op"] == "swiglu":
        g, u = y[..., :c["N"]], y[..., c["N"]:]
        y = g / (1.0 + torch.exp(-g)) * u
    p = torch.arange(n, device="cuda")
    e = torch.searchsorted(off[1:], p, right=True)
    return y[e, p - off[e]].to(torch.bfloat16)


def _combine(c, d):
    at = d["place"].long().view(c["tokens"], c["k"])
    w = torch.where(at >= 0, d["weights"], 0.0)
    out = (d["y"].float()[at.clamp(min=0)] * w[..., None]).sum(1)
    return (out if d["add"] is None else out + d["add"].float()).to(torch.bfloat16)


def _adapters(c, d):
    x = d["x"].float()
    t = (x @ d["A"].float().t()) * (d["ids"][:, None] == d["col"]) * d["scale"][:, None]
    return (x @ _f32(d["w"]).t() + t @ d["B"].float().t()).to(torch.bfloat16)


# ---- the work a pass cannot do without ---------------------------------------------------
def _bytes(N, K, bits):
    return 2.0 * N * K if bits == 16 else N * K * bits / 8.0 + 4.0 * N * K / 64


def work(case):
    c, op = case, case["op"]
    if op == "route":
        n = float(c["rows"]) * c["experts"]
        return {"bytes": n * (4 if c["f32"] else 2) + 8.0 * c["rows"] * c["k"], "flops": 4.0 * n}
    if op == "group":
        return {"bytes": 12.0 * c["n"] + 4.0 * c["groups"], "flops": 4.0 * c["n"]}
    if op in ("swiglu", "lin"):
        n, E, K = c["tokens"] * c["k"], c["experts"], c["K"]
        N = c["N"] * 2 if op == "swiglu" else c["N"]
        live = E * (1.0 - (1.0 - 1.0 / E) ** n)          # experts with a row, about
        rows = c["tokens"] if op == "swiglu" else n
        return {"bytes": live * _bytes(N, K, c["bits"]) + 2.0 * rows * K + 2.0 * n * c["N"]
                + 4.0 * n, "flops": 2.0 * n * N * K}
    if op == "combine":
        n = float(c["tokens"]) * c["k"]
        return {"bytes": 2.0 * n * c["N"] + 8.0 * n
                + 2.0 * c["tokens"] * c["N"] * (2 if c["add"] else 1), "flops": 2.0 * n * c["N"]}
    ranks, held = BANKS[c["bank"]]
    used = min(held, c["requests"])
    r = sum(ranks[i % len(ranks)] for i in range(held)) / held
    return {"bytes": _bytes(c["N"], c["K"], c["bits"]) + 2.0 * c["M"] * (c["N"] + c["K"])
            + 2.0 * used * r * (c["N"] + c["K"]) + 8.0 * c["M"],
            "flops": 2.0 * c["M"] * c["N"] * c["K"] + 2.0 * c["M"] * r * (c["N"] + c["K"])}


# ---- the definitions in 64 bits ------------------------------------------------------------
def _w64(w, e=None):
    w = {k: (v[e] if e is not None and k in ("w", "codes", "scales", "biases") else v)
         for k, v in w.items()}
    if "w" in w:
        return w["w"].double()
    bits = w["bits"]
    fields = [((w["codes"] >> (bits * i)) & ((1 << bits) - 1)).double() for i in range(32 // bits)]
    q = torch.stack(fields, -1).reshape(w["scales"].shape[0], -1, 64)
    return (q * w["scales"].double()[..., None] + w["biases"].double()[..., None]).flatten(1)


def _route64(c, d):
    rows = d["logits"].float().cpu().numpy().astype(np.float64)
    bias = np.zeros(c["experts"]) if d["bias"] is None else \
        d["bias"].cpu().numpy().astype(np.float64)
    ids = np.full((c["rows"], c["k"]), -1, np.int32)
    out = np.zeros((c["rows"], c["k"]))
    size = c["experts"] // c["groups"]
    for t, l in enumerate(rows):
        live = np.flatnonzero(l > -np.inf)
        if not live.size:
            continue
        if c["score"] == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-l[live]))
        else:
            s = np.exp(l[live] - l[live].max())
            s /= s.sum()
        key = s + bias[live]
        if c["groups"] > 1:
            best = []
            for g in range(c["groups"]):
                k = np.sort(key[live // size == g])[::-1]
                if k.size:
                    best.append((-k[:2].sum(), g))
            keep = np.isin(live // size, [g for _, g in sorted(best)[:c["top_groups"]]])
            live, s, key = live[keep], s[keep], key[keep]
        pick = np.lexsort((live, -key))[:c["k"]]
        ids[t, :pick.size] = live[pick]
        w = s[pick]
        if c["normalize"]:
            w = w / w.sum() if w.sum() > 0 else w * 0.0
        out[t, :pick.size] = w * 2.5
    return [ids, out]


def exact(case, seed):
    c, op = case, case["op"]
    d = _inputs(c, seed)
    if op == "route":
        return _route64(c, d)
    if op == "group":
        return None                     # whole numbers, compared as they are
    if op in ("swiglu", "lin"):
        ends = np.cumsum(d["counts"])
        y = torch.zeros((c["tokens"] * c["k"], c["N"]), dtype=torch.float64, device="cuda")
        for e in np.flatnonzero(d["counts"]):
            a, b = int(ends[e] - d["counts"][e]), int(ends[e])
            rows = d["x"][a:b] if d["order"] is None else d["x"][d["order"][a:b].long() // c["k"]]
            t = rows.double() @ _w64(d["w"], e).t()
            if op == "swiglu":
                t = torch.nn.functional.silu(t[:, :c["N"]]) * t[:, c["N"]:]
            y[a:b] = t
        return y
    if op == "combine":
        y = torch.zeros((c["tokens"], c["N"]), dtype=torch.float64, device="cuda")
        if c["add"]:
            y += d["add"].double()
        at = d["place"].long().view(c["tokens"], c["k"])
        for j in range(c["k"]):
            y += d["weights"][:, j:j + 1].double() * d["y"].double()[at[:, j]]
        return y
    x = d["x"].double()
    y = x @ _w64(d["w"]).t()
    at = 0
    for i, r in enumerate(d["ranks"]):
        rows = torch.nonzero(d["ids"] == i)[:, 0]
        if rows.numel():
            t = (x[rows] @ d["A"][at:at + r].double().t()) * d["scale"][rows, None].double()
            y[rows] += t @ d["B"][:, at:at + r].double().t()
        at += r
    return y
