"""The operators in 8-bit floating point against their 64-bit definitions: the
quantizers and the norm (codes to the bit), the products over one row to many, odd
widths and K, strides, groups that are empty or end inside a tile, NaN that stays in
its row, captured calls, and a feed-forward from the residual to the next norm."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import ming_dit_amd as m
import rows_ref
from helpers import bf16, f32, from_dev, randn, sync, to_dev

pytestmark = pytest.mark.gpu
S8, S16 = 0x3b, 0x4242     # what outputs hold before a call


def dev8(a, pad=0, fill=ref.NAN):
    """Codes on the device with `pad` columns of NaN beside them."""
    out = np.full((max(a.shape[0], 1), a.shape[1] + pad), fill, np.uint8)
    out[:a.shape[0], :a.shape[1]] = a
    return to_dev(out)


def dev_scales(s, pad=0, fill=0x7fc0):
    out = np.full((s.shape[0], s.shape[1] + pad), fill, np.uint16)
    out[:, :s.shape[1]] = s
    return to_dev(out)


# ---- the quantizers ------------------------------------------------------------------
def quantize(ctx, x, padx=0, padc=0, pads=0):
    rows, D = x.shape
    xs = np.full((rows, D + padx), 0x7fc0, np.uint16)
    xs[:, :D] = x
    xd, cd = to_dev(xs), to_dev(np.full((rows, D + padc), S8, np.uint8))
    sd = to_dev(np.full((ref.blocks(D), rows + pads), S16, np.uint16))
    sync()
    ctx.f8_quantize(xd, rows, D, cd, sd, ldx=D + padx, ldc=D + padc, lds=rows + pads)
    ctx.synchronize()
    codes, scales = from_dev(cd), from_dev(sd)
    assert np.all(codes[:, D:] == S8) and np.all(scales[:, rows:] == S16)
    return codes[:, :D], scales[:, :rows]


@pytest.mark.parametrize("rows,D", [(1, 16), (3, 128), (2, 112), (5, 144), (7, 1040), (1, 3840),
                                    (300, 272), (33, 10240)])
@pytest.mark.parametrize("pad", [0, 16])
def test_quantize(ctx, rows, D, pad):
    """Codes and scales to the bit."""
    x = bf16(randn(100 + rows, (rows, D)) * np.exp(randn(7, (1, D))))
    codes, scales = quantize(ctx, x, pad, pad, pad)
    want, s = ref.quantize(f32(x).astype(np.float64))
    assert np.array_equal(codes, want)
    assert np.array_equal(scales, s)


def test_quantize_every_ratio(ctx):
    """Every bf16 significand over every largest one: the borders of two codes among
    them, at sizes from the smallest to the largest."""
    m8 = (128 + np.arange(128)) / 128.0
    for size in (2.0 ** -90, 2.0 ** -3, 1.0, 2.0 ** 60, 2.0 ** 126):
        x = np.zeros((128 * 4, 128))
        for i, down in enumerate((0, 1, 3, 9)):
            x[128 * i:128 * i + 128, :127] = m8[None, :127] * 2.0 ** -down * size
            x[128 * i:128 * i + 128, 127] = m8 * size
        x[:, ::3] *= -1
        b = bf16(x.astype(np.float32))
        codes, scales = quantize(ctx, b)
        want, s = ref.quantize(f32(b).astype(np.float64))
        assert np.array_equal(codes, want), size
        assert np.array_equal(scales, s)


def test_quantize_odd_values(ctx):
    """Zeros, the smallest and the largest values, -0, and blocks with inf or NaN that
    leave the others of their row alone."""
    x = randn(5, (6, 300))
    x[0] = 0.0
    x[1, :128] = -0.0
    x[1, 5] = 1e-39
    x[2, :] = 3.3e38
    x[2, ::2] = -1e-38
    x[3, 130] = np.inf
    x[4, 299] = np.nan
    x[5, 7] = -np.inf
    x = x[:, :288].copy()
    x[4, 287] = np.nan
    b = bf16(x)
    codes, scales = quantize(ctx, b)
    bad = np.zeros((6, 3), bool)
    bad[3, 1] = bad[4, 2] = bad[5, 0] = True
    v = f32(b).astype(np.float64)
    wide = np.repeat(bad, 128, 1)[:, :288]
    want, s = ref.quantize(np.where(wide, 0.0, v))
    assert np.all(np.isnan(ref.decode(codes)[wide])) and np.all(scales.T[bad] == 0x7fc0)
    assert np.array_equal(codes[~wide], want[~wide])
    assert np.array_equal(scales.T[~bad], s.T[~bad])


@pytest.mark.parametrize("N,K", [(8, 16), (128, 128), (130, 144), (1, 1040), (300, 272)])
def test_quantize_weight(ctx, N, K):
    w = bf16(randn(900 + N, (N, K), 0.02))
    cd = to_dev(np.full(N * K + 16, S8, np.uint8))
    sd = to_dev(np.full(ref.blocks(N) * ref.blocks(K) + 1, 123.5, np.float32))
    wd = to_dev(w)
    sync()
    ctx.f8_quantize_weight(wd, N, K, cd, sd)
    ctx.synchronize()
    codes, scales = ref.quantize_weight(f32(w))
    got, gots = from_dev(cd), from_dev(sd)
    assert np.array_equal(got[:-16].reshape(N, K), codes) and np.all(got[-16:] == S8)
    assert np.array_equal(gots[:-1], scales.reshape(-1)) and gots[-1] == np.float32(123.5)


# ---- the norm --------------------------------------------------------------------------
def norm(ctx, x, w, sub=None, y=False, eps=1e-6, pad=0, inplace=None):
    rows, D = x.shape

    def wide(a):
        out = np.full((rows, D + pad), S16, np.uint16)
        if a is not None:
            out[:, :D] = a
        return to_dev(out)

    xd, wd = wide(x), to_dev(w)
    sd = wide(sub) if sub is not None else None
    hd = None if sub is None else {None: wide(None), "x": xd, "sub": sd}[inplace]
    yd = wide(None) if y else None
    cd = to_dev(np.full((rows, D + pad), S8, np.uint8))
    sc = to_dev(np.full((ref.blocks(D), rows + pad), S16, np.uint16))
    ld = D + pad
    sync()
    ctx.f8_rmsnorm(xd, wd, rows, D, cd, sc, sub=sd, h=hd, y=yd, eps=eps, ldx=ld, ldsub=ld, ldh=ld,
                   ldy=ld, ldc=ld, lds=rows + pad)
    ctx.synchronize()
    codes, scales = from_dev(cd), from_dev(sc)
    assert np.all(codes[:, D:] == S8) and np.all(scales[:, rows:] == S16)
    out = []
    for t in (hd, yd):
        t = None if t is None else from_dev(t)
        assert t is None or np.all(t[:, D:] == S16)
        out.append(None if t is None else t[:, :D])
    return out[0], out[1], codes[:, :D], scales[:, :rows]


def check_norm(x, w, sub, eps, h, y, codes, scales):
    v = f32(x)
    if sub is not None:
        want = bf16(v + f32(sub))               # the f32 sum, rounded to bf16
        assert np.array_equal(h, want)
        v = f32(want)
    v = v.astype(np.float64)
    inv = 1.0 / np.sqrt((v * v).mean(1, keepdims=True) + float(np.float32(eps)))
    t = v * f32(w).astype(np.float64) * inv
    # roundings of the value: those of a sum (16 in a thread, 6 + 8 across) count half
    # under the root; the division, the root, the reciprocal and two products
    off = ((16 + 6 + 8 + 2) / 2 + 6) * ref.F32
    ref.check_quantized(codes, scales, t, off * np.abs(t))
    if y is not None:
        got = f32(y).astype(np.float64)
        assert np.all(np.abs(got - t) <= (ref.BF16 + 2 * off) * np.abs(t) + 1e-40)


@pytest.mark.parametrize("rows,D", [(1, 16), (2, 128), (3, 112), (5, 1040), (1, 2560), (9, 3840),
                                    (4, 8192), (65, 272), (2, 8176)])
@pytest.mark.parametrize("add,y,pad", [(False, False, 0), (True, False, 16), (False, True, 16),
                                       (True, True, 0)])
def test_norm(ctx, rows, D, add, y, pad):
    x = bf16(randn(200 + rows, (rows, D)) * np.exp(0.5 * randn(7, (1, D))))
    w = bf16(1.0 + randn(8, (D,), 0.3))
    sub = bf16(randn(300 + rows, (rows, D))) if add else None
    h, yy, codes, scales = norm(ctx, x, w, sub, y, pad=pad)
    check_norm(x, w, sub, 1e-6, h, yy, codes, scales)


@pytest.mark.parametrize("inplace", ["x", "sub"])
def test_norm_in_place(ctx, inplace):
    x, sub = bf16(randn(1, (37, 1040))), bf16(randn(2, (37, 1040)))
    w = bf16(1.0 + randn(8, (1040,), 0.3))
    a = norm(ctx, x, w, sub, True)
    b = norm(ctx, x, w, sub, True, inplace=inplace)
    for p, q in zip(a, b):
        assert np.array_equal(p, q)


def test_norm_odd_rows(ctx):
    """Rows of zeros, of tiny and of large values, weights that are zero, and rows with
    NaN or inf, whose neighbours stay as they are."""
    x = randn(3, (8, 400))
    x[0] = 0.0
    x[1] *= 1e-18
    x[2] *= 1e17
    x[3, 1:] = 0.0
    x = bf16(x)
    w = 1.0 + randn(8, (400,), 0.3)
    w[128:256] = 0.0
    w = bf16(w)
    _, y, codes, scales = norm(ctx, x, w, y=True, eps=1e-5)
    check_norm(x, w, None, 1e-5, None, y, codes, scales)
    bad = x.copy()
    bad[4, 399] = 0x7fc0
    bad[6, 0] = 0x7f80
    _, y2, codes2, scales2 = norm(ctx, bad, w, y=True, eps=1e-5)
    keep = [0, 1, 2, 3, 5, 7]
    for p, q in ((y, y2), (codes, codes2), (scales.T, scales2.T)):
        assert np.array_equal(p[keep], q[keep])
    assert np.all((codes2[[4, 6]] & 0x7f) == ref.NAN) and np.all(scales2.T[[4, 6]] == 0x7fc0)


# ---- the products ------------------------------------------------------------------------
class Weights:
    def __init__(self, ctx, seed, E, N, K, gated, on_device=False):
        self.codes, self.scales = ref.make_weight(seed, E, N, K, gated)
        c, s = (to_dev(self.codes), to_dev(self.scales)) if on_device else (self.codes, self.scales)
        sync()
        self.w = m.F8(ctx, c, s, N, gated=gated, on_device=on_device)
        self.E, self.N, self.K, self.gated = E, N, K, gated


def call(ctx, W, x, xs, offsets=None, order=None, n=None, fan=1, bias=None, pad=0):
    """A call's outputs (y as f64, or codes and scales) over the rows the plan holds."""
    rows = x.shape[0]
    n = rows if n is None else n
    held = n if offsets is None else int(offsets[-1])
    xd, sd = dev8(x, pad), dev_scales(xs, pad)
    ws = torch.full((W.w.workspace_bytes(n) + 16,), 255, dtype=torch.uint8, device="cuda")
    od = None if order is None else to_dev(order)
    fd = None if offsets is None else to_dev(offsets)
    bd = None if bias is None else to_dev(bias)
    kw = dict(ws=ws, ldx=W.K + pad, ldxs=rows + pad)
    if W.gated:
        h = to_dev(np.full((n + 2, W.N + pad), S8, np.uint8))
        hs = to_dev(np.full((ref.blocks(W.N), n + 2), S16, np.uint16))
        kw.update(ldh=W.N + pad, ldhs=n + 2)
        sync()
        if offsets is None:
            ctx.f8_swiglu(W.w, xd, sd, h, hs, n, **kw)
        else:
            ctx.f8_experts_swiglu(W.w, xd, sd, rows, od, fd, n, h, hs, fan=fan, **kw)
        ctx.synchronize()
        h, hs = from_dev(h), from_dev(hs)
        assert np.all(h[held:] == S8) and np.all(h[:, W.N:] == S8) and np.all(hs[:, held:] == S16)
        return h[:held, :W.N], hs[:, :held]
    y = to_dev(np.full((n + 2, W.N + pad), S16, np.uint16))
    kw["ldy"] = W.N + pad
    sync()
    if offsets is None:
        ctx.f8_lin(W.w, xd, sd, y, n, bias=bd, **kw)
    else:
        ctx.f8_experts_lin(W.w, xd, sd, rows, od, fd, n, y, fan=fan, **kw)
    ctx.synchronize()
    y = from_dev(y)
    assert np.all(y[held:] == S16) and np.all(y[:, W.N:] == S16)
    return f32(y[:held, :W.N]).astype(np.float64)


def check(got, W, x, xs, offsets=None, src=None, bias=None):
    v, d = ref.products(x, xs, W.codes, W.scales, offsets, src, W.gated,
                        None if bias is None else f32(bias).astype(np.float64))
    if W.gated:
        ref.check_quantized(*got, v, d)
        return
    bound = ref.bf16_bound(v, d)
    assert got.shape == v.shape
    assert got.size == 0 or np.max(np.abs(got - v) / bound) <= 1.0
    if got.size > 1000:
        assert rows_ref.rel(got, v) <= rows_ref.REL


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K", [(16, 16), (144, 128), (272, 240), (528, 1152), (1040, 592),
                                 (2064, 144)])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 130, 257, 520])
def test_products(ctx, gated, N, K, M):
    print(f"case f8 gated={gated} N={N} K={K} M={M}", flush=True)
    W = Weights(ctx, 1000 + N, 1, N, K, gated)
    x, xs = ref.make_rows(2000 + M, M, K)
    check(call(ctx, W, x, xs, pad=16), W, x, xs)
    W.w.close()


@pytest.mark.parametrize("N,K,M", [(8, 128, 3), (24, 272, 70), (136, 128, 200), (520, 640, 300)])
def test_bias_and_narrow_widths(ctx, N, K, M):
    W = Weights(ctx, 1100 + N, 1, N, K, False, on_device=True)
    x, xs = ref.make_rows(2100 + M, M, K)
    bias = bf16(randn(11, (N,), 2.0))
    a = call(ctx, W, x, xs, bias=bias)
    check(a, W, x, xs, bias=bias)
    assert np.array_equal(a, call(ctx, W, x, xs, bias=bias, pad=32))
    W.w.close()


COUNTS = {
    "one row": [0, 1, 0],
    "a row each": [1] * 7,
    "edges": [15, 0, 16, 17, 1, 0, 63],
    "tiles": [64, 65, 0, 127, 128, 129],
    "uneven": [0, 300, 2, 0, 0, 31],
    "large": [255, 256, 257, 513],
    "none": [0, 0, 0],
}


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("what", COUNTS)
def test_experts(ctx, gated, what):
    counts = COUNTS[what]
    E, K, N = len(counts), 208, 144
    print(f"case f8 experts gated={gated} {what}", flush=True)
    W = Weights(ctx, 3000, E, N, K, gated)
    offsets, order, src = rows_ref.plan_of(counts, n=sum(counts) + 11, fan=2, seed=E, x_rows=50)
    x, xs = ref.make_rows(3100, 50, K)
    got = call(ctx, W, x, xs, offsets, order, order.size, fan=2, pad=16)
    check(got, W, x, xs, offsets, src)
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K,counts", [(16, 16, [3, 0, 70, 40]), (272, 128, [3, 0, 70, 40]),
                                        (528, 1088, [200, 0, 1, 130]), (1040, 592, [9, 300])])
def test_experts_in_place_order(ctx, gated, N, K, counts):
    W = Weights(ctx, 3200, len(counts), N, K, gated, on_device=True)
    offsets, _, _ = rows_ref.plan_of(counts)
    n = sum(counts)
    x, xs = ref.make_rows(3300, n, K)
    got = call(ctx, W, x, xs, offsets, None, n)
    check(got, W, x, xs, offsets, np.arange(n))
    W.w.close()


@pytest.fixture()
def plan(ctx):
    yield lambda p: ref.set_plan(ctx, p)
    ref.set_plan(ctx, -1)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K", [(16, 16), (144, 128), (400, 272), (528, 1168), (272, 2576)])
@pytest.mark.parametrize("M", [1, 63, 64, 65, 128, 200, 257, 513])
def test_every_kernel(ctx, plan, gated, N, K, M):
    """Each kernel at and beside every tile height, one block of K to odd and even counts
    of them, columns and K that end inside a tile; the tiles give the same bits."""
    W = Weights(ctx, 6000 + N, 1, N, K, gated)
    x, xs = ref.make_rows(6100 + M, M, K)
    first = None
    for p in ref.PLANS if gated else ref.PLANS + ref.DUO:
        print(f"case f8 plan {p} gated={gated} N={N} K={K} M={M}", flush=True)
        plan(p)
        got = call(ctx, W, x, xs, pad=16 * (p % 2))
        check(got, W, x, xs)
        if p == 1:
            first = got
        if 1 < p < 10:
            for a, b in zip(first, got):
                assert np.array_equal(a, b)
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K,counts", [
    (528, 1088, [1, 64, 65, 0, 127, 128, 129, 63, 2, 200, 130, 100]),
    (560, 576, [255, 256, 257, 1, 513, 0, 192, 193, 321, 449]),
    (2064, 64, [300, 700, 15, 0, 1, 900]),
    (272, 1216, [40, 1000]), (16, 128, [70, 0, 9])])
def test_every_grouped_kernel(ctx, plan, gated, N, K, counts):
    E, n = len(counts), sum(counts)
    W = Weights(ctx, 6200, E, N, K, gated)
    offsets, order, src = rows_ref.plan_of(counts, n=n + 70, fan=3, seed=N, x_rows=300)
    x, xs = ref.make_rows(6300, 300, K)
    # rows in place order: the gathered rows' copies
    gx, gs = x[src], np.ascontiguousarray(xs[:, src])
    for p in ref.GROUPED_PLANS:
        print(f"case f8 grouped plan {p} gated={gated} N={N} K={K}", flush=True)
        plan(p)
        got = call(ctx, W, x, xs, offsets, order, order.size, fan=3, pad=16)
        check(got, W, x, xs, offsets, src)
        for a, b in zip(got, call(ctx, W, gx, gs, offsets, None, n)):
            assert np.array_equal(a, b)
    W.w.close()


@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_nan_stays_in_its_row(ctx, gated, M):
    """A row with a block of NaN is NaN and no other changes, with K short of a block and
    x's columns past K holding NaN."""
    N, K = 272, 400
    W = Weights(ctx, 4000, 1, N, K, gated)
    x, xs = ref.make_rows(4100, M, K)
    a = call(ctx, W, x, xs, pad=16)
    x2, xs2 = x.copy(), xs.copy()
    at = [1, M - 1]
    x2[1, 130] = 0xff
    xs2[0, M - 1] = 0x7fc0
    b = call(ctx, W, x2, xs2, pad=16)
    keep = [r for r in range(M) if r not in at]
    if gated:
        assert np.array_equal(a[0][keep], b[0][keep])
        assert np.array_equal(a[1].T[keep], b[1].T[keep])
        assert np.all((b[0][at] & 0x7f) == ref.NAN) and np.all(b[1].T[at] == 0x7fc0)
    else:
        assert np.array_equal(a[keep], b[keep]) and np.all(np.isnan(b[at]))
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [5, 90, 300])
def test_extreme_scales(ctx, gated, M):
    """Scales over eighty powers of two, and a row of zeros."""
    N, K = 144, 640
    W = Weights(ctx, 4200, 1, N, K, gated)
    x, xs = ref.make_rows(4300, M, K)
    rng = np.random.default_rng(4)
    xs = bf16((f32(xs) * 2.0 ** rng.integers(-20, 20, xs.shape)).astype(np.float32))
    x[2] = 0
    W.w.close()
    scales = (W.scales * 2.0 ** rng.integers(-20, 20, W.scales.shape)).astype(np.float32)
    W.scales = scales
    W.w = m.F8(ctx, W.codes, scales, N, gated=gated)
    check(call(ctx, W, x, xs), W, x, xs)
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [1, 40, 600])
def test_same_bits_every_time(ctx, gated, M):
    """Twice the same bits, and a row's bits do not depend on the rows beside it."""
    N, K = 528, 1040
    W = Weights(ctx, 4400, 1, N, K, gated)
    x, xs = ref.make_rows(4500, M, K)
    a, b = call(ctx, W, x, xs), call(ctx, W, x, xs, pad=16)
    for p, q in zip(a, b):
        assert np.array_equal(p, q)
    W.w.close()


def test_calls_of_no_rows_take_empty_arrays(ctx):
    W = Weights(ctx, 4600, 1, 16, 16, False)
    G = Weights(ctx, 4601, 2, 16, 16, True)
    ctx.f8_quantize(None, 0, 16, None, None)
    ctx.f8_rmsnorm(None, None, 0, 16, None, None)
    ctx.f8_lin(W.w, None, None, None, 0)
    ctx.f8_experts_swiglu(G.w, None, None, 0, None, None, 0, None, None)
    ctx.synchronize()
    W.w.close()
    G.w.close()


def test_refusals(ctx):
    W = Weights(ctx, 4700, 1, 32, 144, False)
    G = Weights(ctx, 4701, 1, 32, 144, True)
    X = Weights(ctx, 4702, 2, 32, 144, True)
    M = 4
    x, xs = dev8(ref.make_rows(1, M, 144)[0]), dev_scales(ref.make_rows(1, M, 144)[1])
    y = to_dev(np.zeros((M, 32), np.uint16))
    h, hs = to_dev(np.zeros((M, 32), np.uint8)), to_dev(np.zeros((1, M), np.uint16))
    ws = torch.zeros(max(16, G.w.workspace_bytes(M)), dtype=torch.uint8, device="cuda")
    off = to_dev(np.array([0, 2, 4], np.int32))
    xb = to_dev(np.zeros((M, 144), np.uint16))
    c, s = to_dev(np.zeros((M, 144), np.uint8)), to_dev(np.zeros((2, M), np.uint16))
    sf = to_dev(np.zeros((1, 2), np.float32))
    wn = to_dev(np.zeros(144, np.uint16))
    sync()
    bad = [
        lambda: ctx.f8_lin(G.w, x, xs, y, M, ws=ws),                    # gated weights
        lambda: ctx.f8_swiglu(W.w, x, xs, h, hs, M, ws=ws),             # plain weights
        lambda: ctx.f8_swiglu(X.w, x, xs, h, hs, M, ws=ws),             # a stack
        lambda: ctx.f8_lin(W.w, x, xs, y, -1),
        lambda: ctx.f8_lin(W.w, x, xs, y, M, ldx=128),
        lambda: ctx.f8_lin(W.w, x, xs, y, M, ldx=152),                  # not of 16
        lambda: ctx.f8_lin(W.w, x, xs, y, M, ldxs=M - 1),
        lambda: ctx.f8_lin(W.w, x, xs, y, M, ldy=36),
        lambda: ctx.f8_lin(W.w, x.data_ptr() + 8, xs, y, M),
        lambda: ctx.f8_lin(W.w, x, xs, x, M),                           # y over x
        lambda: ctx.f8_lin(W.w, x, xs, None, M),
        lambda: ctx.f8_lin(W.w, x, xs, y, M, ldx=1 << 22),
        lambda: ctx.f8_lin(W.w, x, xs, y, (1 << 28) + 1, ldxs=1 << 29),
        lambda: ctx.f8_swiglu(G.w, x, xs, h, hs, M, ldh=24),
        lambda: ctx.f8_swiglu(G.w, x, xs, h, hs, M, ldhs=M - 1, ws=ws),
        lambda: ctx.f8_swiglu(G.w, x, xs, h, h, M, ws=ws),              # scales over codes
        lambda: ctx.f8_experts_swiglu(X.w, x, xs, M, None, off, M + 1, h, hs, ws=ws, ldhs=M + 1),
        lambda: ctx.f8_experts_swiglu(X.w, x, xs, 0, off, off, M, h, hs, ws=ws),
        lambda: ctx.f8_experts_swiglu(X.w, x, xs, M, None, None, M, h, hs, ws=ws),
        lambda: ctx.f8_experts_swiglu(X.w, x, xs, M, None, off, M, h, hs, ws=ws, fan=0),
        lambda: ctx.f8_quantize(xb, M, 140, c, s),
        lambda: ctx.f8_quantize(xb, M, 144, c, s, ldc=152),
        lambda: ctx.f8_quantize(xb, M, 144, c, s, lds=M - 1),
        lambda: ctx.f8_quantize(xb, M, 144, xb, s),
        lambda: ctx.f8_quantize(xb, -1, 144, c, s),
        lambda: ctx.f8_rmsnorm(xb, wn, M, 144, c, s, sub=xb),           # no h
        lambda: ctx.f8_rmsnorm(xb, wn, M, 144, c, s, h=xb),             # no sub
        lambda: ctx.f8_rmsnorm(xb, wn, M, 8208, c, s),
        lambda: ctx.f8_rmsnorm(xb, wn, M, 144, c, s, eps=0.0),
        lambda: ctx.f8_rmsnorm(xb, wn, M, 144, c, s, eps=float("nan")),
        lambda: ctx.f8_rmsnorm(xb, wn, M, 144, c, s, y=xb),
        lambda: ctx.f8_quantize_weight(xb, M, 140, c, sf),
        lambda: ctx.f8_quantize_weight(xb, 0, 144, c, sf),
        lambda: m.F8(ctx, np.zeros((4, 144), np.uint8), np.zeros((1, 2), np.float32), 4),
        lambda: m.F8(ctx, np.zeros((16, 140), np.uint8), np.zeros((1, 2), np.float32), 16),
        lambda: m.F8(ctx, np.zeros((16, 144), np.uint8), np.zeros((2, 2), np.float32), 8, True),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(m.MingError) as e:
            f()
        assert e.value.code in (1, 2), i
    if G.w.workspace_bytes(M):
        with pytest.raises(m.MingError):
            ctx.f8_swiglu(G.w, x, xs, h, hs, M)
        with pytest.raises(m.MingError):
            ctx.f8_swiglu(G.w, x, xs, h, hs, M, ws=ws[:16])
    ctx.synchronize()
    for w in (W, G, X):
        w.w.close()


# ---- together ------------------------------------------------------------------------------
def test_feed_forward_captured(ctx):
    """From the residual to the next norm, as a program runs it, captured and replayed
    with eager calls between: every replay has the eager calls' bits, and those are what
    the operators give one after another."""
    s = torch.cuda.Stream()
    c = m.Ctx(0, s.cuda_stream)
    T, H, F = 70, 400, 272
    GU, DN = Weights(c, 5000, 1, F, H, True), Weights(c, 5001, 1, H, F, False)
    nw = bf16(1.0 + randn(1, (H,), 0.2))

    def new(shape, dtype):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    x, sub, nwd = new((T, H), torch.bfloat16), new((T, H), torch.bfloat16), to_dev(nw)
    h1, out, h2 = (new((T, H), torch.bfloat16) for _ in range(3))
    c1, s1 = new((T, H), torch.uint8), new((ref.blocks(H), T), torch.int16)
    ch, sh = new((T, F), torch.uint8), new((ref.blocks(F), T), torch.int16)
    c2, s2 = new((T, H), torch.uint8), new((ref.blocks(H), T), torch.int16)
    ws = new((16 + max(w.w.workspace_bytes(T) for w in (GU, DN)),), torch.uint8)
    outs = (h1, c1, s1, ch, sh, out, h2, c2, s2)

    def step():
        c.f8_rmsnorm(x, nwd, T, H, c1, s1, sub=sub, h=h1)
        c.f8_swiglu(GU.w, c1, s1, ch, sh, T, ws=ws)
        c.f8_lin(DN.w, ch, sh, out, T, ws=ws)
        c.f8_rmsnorm(h1, nwd, T, H, c2, s2, sub=out, h=h2)

    sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        step()
    for it in range(3):
        hx, hs = bf16(randn(5100 + it, (T, H))), bf16(randn(5200 + it, (T, H)))
        x.copy_(to_dev(hx).view(torch.bfloat16))
        sub.copy_(to_dev(hs).view(torch.bfloat16))
        sync()
        g.replay()
        sync()
        got = [from_dev(t).copy() for t in outs]
        for t in outs:
            t.zero_()
        sync()
        step()
        c.synchronize()
        for a, t in zip(got, outs):
            assert np.array_equal(a, from_dev(t))
        gh1, gc1, gs1, gch, gsh, gout, gh2, gc2, gs2 = got
        check_norm(hx, nw, hs, 1e-6, gh1, None, gc1, gs1)
        check((gch, gsh), GU, gc1, gs1)
        check(f32(gout).astype(np.float64), DN, gch, gsh)
        check_norm(gh1, nw, gout, 1e-6, gh2, None, gc2, gs2)
    del g
    GU.w.close()
    DN.w.close()
    c.close()


def test_mixture_of_experts(ctx):
    """Router, grouping, gate and up, down, weighted sum: a mixture's feed-forward over
    8-bit weights."""
    T, H, F, E, k = 37, 272, 144, 6, 2
    n = T * k
    GU, DN = Weights(ctx, 5300, E, F, H, True), Weights(ctx, 5310, E, H, F, False)
    x = bf16(randn(5320, (T, H)))
    logits = randn(5321, (T, E))
    xd, ld = to_dev(x), to_dev(logits)
    ids, wt = (torch.zeros((T, k), dtype=t, device="cuda") for t in (torch.int32, torch.float32))
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    order, place = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    c1 = torch.zeros((T, H), dtype=torch.uint8, device="cuda")
    s1 = torch.zeros((ref.blocks(H), T), dtype=torch.int16, device="cuda")
    ch = torch.zeros((n, F), dtype=torch.uint8, device="cuda")
    sh = torch.zeros((ref.blocks(F), n), dtype=torch.int16, device="cuda")
    y = torch.zeros((n, H), dtype=torch.int16, device="cuda")
    out = torch.zeros((T, H), dtype=torch.int16, device="cuda")
    ws = torch.zeros(16 + max(w.w.workspace_bytes(n) for w in (GU, DN)), dtype=torch.uint8,
                     device="cuda")
    sync()
    ctx.f8_quantize(xd, T, H, c1, s1)
    ctx.topk_route(ld, T, E, k, ids, wt)
    ctx.group_rows(ids, n, E, off, order, place)
    ctx.f8_experts_swiglu(GU.w, c1, s1, T, order, off, n, ch, sh, fan=k, ws=ws)
    ctx.f8_experts_lin(DN.w, ch, sh, n, None, off, n, y, ws=ws)
    ctx.experts_combine(y, n, place, wt, T, k, out, H, add=xd)
    ctx.synchronize()
    ho, hi = from_dev(off), from_dev(order)
    want, s = ref.quantize(f32(x).astype(np.float64))
    assert np.array_equal(from_dev(c1), want)
    check((from_dev(ch), from_dev(sh)), GU, want, s, ho, hi // k)
    gy = from_dev(y)
    check(f32(gy).astype(np.float64), DN, from_dev(ch), from_dev(sh), ho, np.arange(n))
    o, b = rows_ref.combine(f32(gy), from_dev(place).reshape(T, k), from_dev(wt),
                            f32(x).astype(np.float64), n)
    assert np.all(np.abs(f32(from_dev(out)) - o) <= b)
    GU.w.close()
    DN.w.close()
