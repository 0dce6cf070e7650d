"""Plain 64-bit forms of the operators whose rows choose their own weights, and
the bounds their rounding gives (numpy, on the CPU)."""
import numpy as np

import oracle as orc

# Half a step of a rounding, relative to the value.
BF16, FP16, F32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24


def route(logits, k, bias=None, n_groups=1, top_groups=1, score="softmax", normalize=True,
          scale=1.0):
    rows, E = logits.shape
    ids = np.full((rows, k), -1, np.int32)
    out = np.zeros((rows, k))
    size = E // n_groups
    for t in range(rows):
        l = np.minimum(logits[t].astype(np.float64), float(np.finfo(np.float32).max))
        live = np.flatnonzero(l > -np.inf)
        if not live.size:
            continue
        with np.errstate(over="ignore"):
            if score == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-l[live]))
            else:
                s = np.exp(l[live] - l[live].max())
                s = s / s.sum()
        key = s + (0.0 if bias is None else bias[live].astype(np.float64))
        fine = key > -np.inf
        live, s, key = live[fine], s[fine], key[fine]
        if n_groups > 1:
            best = sorted((-np.sort(key[live // size == g])[::-1][:2].sum(), g)
                          for g in range(n_groups) if np.any(live // size == g))
            keep = np.isin(live // size, [g for _, g in best[:top_groups]])
            live, s, key = live[keep], s[keep], key[keep]
        pick = np.lexsort((live, -key))[:k]
        ids[t, :pick.size] = live[pick]
        w = s[pick]
        if normalize:
            w = w / w.sum() if w.sum() > 0 else 0.0 * w
        out[t, :pick.size] = w * float(np.float32(scale))
    return ids, out


def group(ids, G):
    n = ids.size
    key = np.where((ids >= 0) & (ids < G), ids, G)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(G + 1)).astype(np.int32)
    held = np.arange(n) < offsets[G]
    place = np.empty(n, np.int32)
    place[order] = np.where(held, np.arange(n), -1)
    return offsets, np.where(held, order, -1).astype(np.int32), place


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def products(x, w, offsets, src, gated, bits):
    """(y, bound): f64 products of places' rows src with their experts' weights
    w [E][N][K], and how far the library's may be: one rounding of the output to
    bf16, f32 sums (K + 8 roundings), and for quantized weights one of each
    weight to fp16."""
    n = int(offsets[-1])
    E, N, K = w.shape
    width = N // 2 if gated else N
    y, b = np.zeros((n, width)), np.zeros((n, width))
    per = (K + 8) * F32 + (FP16 if bits != 16 else 0.0)
    for e in range(E):
        r = slice(int(offsets[e]), int(offsets[e + 1]))
        if r.stop <= r.start:
            continue
        rows = x[src[r]].astype(np.float64)
        t = rows @ w[e].astype(np.float64).T
        s = np.abs(rows) @ np.abs(w[e].astype(np.float64)).T * per
        if gated:
            g, u = t[:, :width], t[:, width:]
            y[r] = silu(g) * u
            # |silu'| <= 1.1; the two base-2 functions of silu are good to 2 steps
            b[r] = 1.1 * s[:, :width] * (np.abs(u) + s[:, width:]) \
                + (np.abs(silu(g))) * (s[:, width:] + 8 * F32 * np.abs(u))
        else:
            y[r], b[r] = t, s
    return y, b * (1 + BF16) + BF16 * np.abs(y) + 1e-30


def combine(y, place, weights, add, n):
    tokens, k = weights.shape
    out = np.zeros((tokens, y.shape[1]))
    s = np.zeros_like(out)
    for t in range(tokens):
        for j in range(k):
            p = int(place[t, j])
            if 0 <= p < n:
                v = float(weights[t, j]) * y[p].astype(np.float64)
                out[t] += v
                s[t] += np.abs(v)
    if add is not None:
        out += add
        s += np.abs(add)
    return out, (k + 2) * F32 * s + BF16 * np.abs(out) + 1e-30


def adapters(x, w, bank, ids, scale, bits):
    """(y, bound) of x . W^T plus each row's own adapter, bank {id: (A, B,
    fold)}: T rounded once to bf16, f32 sums, the output rounded once."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    K = x.shape[1]
    y = x @ w.T
    b = np.abs(x) @ np.abs(w).T * ((K + 64) * F32 + (FP16 if bits != 16 else 0.0))
    for m, a in enumerate(ids):
        if int(a) not in bank or scale[m] == 0.0:
            continue
        A, B, fold = bank[int(a)]
        A, B = A.astype(np.float64), B.astype(np.float64)
        c = float(scale[m]) * fold
        t = c * (A @ x[m])
        dt = abs(c) * (np.abs(A) @ np.abs(x[m])) * (K + 8) * F32
        y[m] += B @ t
        b[m] += np.abs(B) @ (BF16 * np.abs(t) + dt * (1 + BF16)) \
            + (np.abs(B) @ np.abs(t)) * (A.shape[0] + 8) * F32
    return y, b * (1 + BF16) + BF16 * np.abs(y) + 1e-30


def rel(got, want):
    return float(np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300))


# One rounding to bf16: errors of at most half a step of the value's binade are
# at most BF16 of it; spread evenly their root mean square is a third of that
# squared. Quantized weights add FP16's the same way (over sums, so less).
REL = BF16 / np.sqrt(3.0) * 1.02


def stack(seed, E, N, K, bits):
    """(create arguments, f32 weights [E][N][K]) of a stack of projections."""
    from helpers import make_weight
    packs = [make_weight(seed + e, N, K, bits, std=0.02 if bits != 16 else 1.0 / np.sqrt(K))
             for e in range(E)]
    keys = ("w",) if bits == 16 else ("codes", "scales", "biases")
    return {k: np.stack([p[0][k] for p in packs]) for k in keys}, np.stack([p[1] for p in packs])


def make_experts(ctx, seed, E, N, K, bits):
    import ming_dit_amd as m
    pack, w = stack(seed, E, N, K, bits)
    if bits == 16:
        return m.Experts.dense(ctx, pack["w"]), w
    return m.Experts.quantized(ctx, pack["codes"], pack["scales"], pack["biases"], bits), w


def plan_of(counts, n=None, fan=1, seed=0, x_rows=None):
    """A plan with given rows an expert: (offsets, order, sources), the order a
    shuffle, `n` places of which those past the last group are dropped."""
    rng = np.random.default_rng(seed)
    held = int(sum(counts))
    n = held if n is None else n
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    order = np.full(n, -1, np.int32)
    order[:held] = rng.permutation(n)[:held] if x_rows is None else \
        rng.integers(0, x_rows * fan, held)
    return offsets, order, order[:held] // fan


def experts_cut(E, N, K, bits, n):
    """Which kernel the plan gives n places: 0 the few-row one, else the tiles' cut."""
    import ming_dit_amd as m
    return m.lib()._ZN4ming11experts_cutEiiiii(E, N, K, bits, n)


def set_experts_cut(ctx, cut):
    """Experts' products on ctx take this cut whatever their size; -1 the plan's."""
    import ctypes as C

    import ming_dit_amd as m
    f = m.lib()._ZN4ming18rt_set_experts_cutEP8ming_ctxi
    f.argtypes, f.restype = [C.c_void_p, C.c_int], None
    f(ctx.h, cut)


CUTS = {16: (0, 2, 4), 8: (0, 2, 8), 4: (0, 2, 4)}


__all__ = ["route", "group", "products", "combine", "adapters", "rel", "REL", "orc"]
