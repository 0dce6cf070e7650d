"""The experts' ragged products (plain and SwiGLU-gated; w4, w8 and dense
stacks) against 64-bit products: uneven groups, rows at every tile edge, places
that were dropped, strides, routes, captured calls, and the whole feed-forward
from logits to tokens."""
import numpy as np
import pytest
import torch

import ming_dit_amd as m
import rows_ref as ref
from helpers import bf16, f32, from_dev, randn, sync, to_dev

pytestmark = pytest.mark.gpu
SENTINEL = 0x4242


def run(ctx, ex, gated, x, offsets, order, n, fan=1, padx=0, pady=0):
    """y of one call, with sentinels behind the last group and in the padding."""
    width = ex.N // 2 if gated else ex.N
    rows = x.shape[0]
    xs = np.full((max(rows, 1), ex.K + padx), 0x7fc0, np.uint16)   # NaN beside the columns
    xs[:rows, :ex.K] = x
    xd, y = to_dev(xs), to_dev(np.full((n + 3, width + pady), SENTINEL, np.uint16))
    ws = torch.empty(max(1, ex.workspace_bytes(rows)), dtype=torch.uint8, device="cuda")
    call = ctx.experts_swiglu if gated else ctx.experts_lin
    od = None if order is None else to_dev(order)
    offd = to_dev(offsets)
    sync()
    call(ex, xd, rows, od, offd, n, y, fan=fan, ws=ws, ldx=ex.K + padx, ldy=width + pady)
    ctx.synchronize()
    y = from_dev(y)
    held = int(offsets[-1])
    assert np.all(y[held:] == SENTINEL) and np.all(y[:, width:] == SENTINEL)
    return y[:held, :width]


def check(got, w, x, offsets, src, gated, bits):
    want, bound = ref.products(f32(x), w, offsets, src, gated, bits)
    got = f32(got).astype(np.float64)
    assert got.shape == want.shape
    worst = np.max(np.abs(got - want) / bound) if got.size else 0.0
    assert worst <= 1.0, worst
    if got.size > 1000:
        assert ref.rel(got, want) <= ref.REL


COUNTS = {
    "one row": [0, 1, 0],
    "a row each": [1] * 7,
    "edges": [15, 0, 16, 17, 1, 0, 63],
    "tiles": [64, 65, 0, 127, 128, 129],
    "uneven": [0, 300, 2, 0, 0, 31],
    "large": [255, 256, 257, 513],
}


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("what", COUNTS)
def test_products(ctx, bits, gated, what):
    counts = COUNTS[what]
    E, K, N = len(counts), 192, 144
    ex, w = ref.make_experts(ctx, 11000, E, N, K, bits)
    offsets, order, src = ref.plan_of(counts, n=sum(counts) + 11, fan=2, seed=E, x_rows=50)
    x = bf16(randn(11100, (50, K)))
    got = run(ctx, ex, gated, x, offsets, order, order.size, fan=2, padx=8, pady=8)
    check(got, w, x, offsets, src, gated, bits)
    ex.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K", [(16, 64), (272, 128), (528, 1088), (1040, 576)])
def test_product_shapes(ctx, bits, gated, N, K):
    """Narrow and odd widths, one K group to many; places in the rows' order."""
    counts = [3, 0, 70, 40]
    ex, w = ref.make_experts(ctx, 11200, 4, N, K, bits)
    offsets, _, _ = ref.plan_of(counts)
    n = sum(counts)
    x = bf16(randn(11300, (n, K)))
    got = run(ctx, ex, gated, x, offsets, None, n)
    check(got, w, x, offsets, np.arange(n), gated, bits)
    ex.close()


@pytest.fixture()
def cut(ctx):
    yield lambda c: ref.set_experts_cut(ctx, c)
    ref.set_experts_cut(ctx, -1)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K,counts", [
    (528, 1088, [1, 64, 65, 0, 127, 128, 129, 63, 2, 200, 130, 100]),
    (560, 576, [255, 256, 257, 1, 513, 0, 192, 193, 321, 449]),
    (2064, 64, [300, 700, 15, 0, 1, 900]),
    (272, 1216, [40, 1000]), (16, 128, [70, 0, 9])])
def test_every_kernel(ctx, cut, bits, gated, N, K, counts):
    """Each kernel on groups that end at and beside every tile height, one K stage
    to odd counts of them, columns that end inside a tile; rows gathered and rows
    in place order to the same bits, twice."""
    E, n = len(counts), sum(counts)
    ex, w = ref.make_experts(ctx, 12900, E, N, K, bits)
    offsets, order, src = ref.plan_of(counts, n=n + 70, fan=3, seed=N, x_rows=300)
    x = bf16(randn(12950, (300, K)))
    for c in ref.CUTS[bits]:
        cut(c)
        got = run(ctx, ex, gated, x, offsets, order, order.size, fan=3, padx=8, pady=16)
        check(got, w, x, offsets, src, gated, bits)
        assert np.array_equal(run(ctx, ex, gated, x[src], offsets, None, n), got)
    ex.close()


def test_the_plan_takes_each_kernel():
    """Few rows: no tiles; a batch's: the low cut; long batches: the tall one."""
    for bits, cuts in ref.CUTS.items():
        assert [ref.experts_cut(64, 2048, 2048, bits, n) for n in (8, 2048, 34816)] == list(cuts)


@pytest.mark.parametrize("bits", [4, 8])
def test_tiles_report_what_fp16_cannot_hold(ctx, cut, bits):
    E, N, K, counts = 3, 560, 576, [300, 10, 400]
    ex, w = ref.make_experts(ctx, 13000, E, N, K, bits)
    offsets, order, src = ref.plan_of(counts, x_rows=64)
    x = bf16(randn(13100, (64, K)))
    x[5, 7] = bf16(np.float32([7.0e4]))[0]
    cut(2)
    with pytest.raises(m.MingError) as e:
        run(ctx, ex, True, x, offsets, order, order.size)
    assert e.value.code == m.ERR_RANGE
    ctx.set_route("wide")
    try:
        check(run(ctx, ex, True, x, offsets, order, order.size), w, x, offsets, src, True, bits)
    finally:
        ctx.set_route("auto")
    xd, y = to_dev(x), to_dev(np.zeros((order.size, N), np.uint16))
    ws = torch.empty(ex.workspace_bytes(64) - 16, dtype=torch.uint8, device="cuda")
    for bad in (None, ws):
        with pytest.raises(m.MingError, match="ws|workspace"):
            ctx.experts_lin(ex, xd, 64, to_dev(order), to_dev(offsets), order.size, y, ws=bad)
    ex.close()


@pytest.mark.parametrize("E", [63, 64, 65, 200, 1000])
def test_many_experts(ctx, E):
    rng = np.random.default_rng(E)
    counts = rng.integers(0, 4, E) * (rng.random(E) < 0.5)
    counts[E - 1] = 2
    ex, w = ref.make_experts(ctx, 11400, E, 16, 64, 16)
    offsets, order, src = ref.plan_of(counts, fan=1, seed=E, x_rows=30)
    x = bf16(randn(11500, (30, 64)))
    got = run(ctx, ex, False, x, offsets, order, order.size)
    check(got, w, x, offsets, src, False, 16)
    ex.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_wide_and_general_routes_take_any_finite_row(ctx, bits):
    """fp16 holds magnitudes below 2^16; the other routes multiply bf16."""
    counts = [200, 0, 130]
    ex, w = ref.make_experts(ctx, 11600, 3, 64, 128, bits)
    offsets, order, src = ref.plan_of(counts, x_rows=64)
    x = bf16(randn(11700, (64, 128)))
    x[5, 7] = bf16(np.float32([3.0e6]))[0]
    try:
        for route in ("wide", "general"):
            ctx.set_route(route)
            got = run(ctx, ex, True, x, offsets, order, order.size)
            check(got, w, x, offsets, src, True, bits)
    finally:
        ctx.set_route("auto")
    ex.close()


@pytest.mark.parametrize("kernel", [0, 2, 4])
def test_a_bad_row_stays_its_own(ctx, cut, kernel):
    """NaN and infinity in one token reach that token's places alone."""
    cut(kernel)
    counts = [5, 100, 0, 64]
    ex, w = ref.make_experts(ctx, 11800, 4, 64, 128, 16)
    offsets, order, src = ref.plan_of(counts, x_rows=40)
    x = bf16(randn(11900, (40, 128)))
    clean = run(ctx, ex, True, x, offsets, order, order.size)
    x[3, 0], x[3, 1] = 0x7fc0, 0x7f80
    got = run(ctx, ex, True, x, offsets, order, order.size)
    assert np.isnan(f32(got[src == 3])).all()
    assert np.array_equal(got[src != 3], clean[src != 3])
    ex.close()


@pytest.mark.parametrize("bits,kernel", [(4, 0), (16, 0), (4, 2), (8, 8), (16, 4)])
def test_captured_products_follow_the_plan(bits, kernel):
    """A captured call replays with the plan that is in memory then, on a stream
    and context of its own, with eager calls between."""
    s = torch.cuda.Stream()
    c = m.Ctx(0, s.cuda_stream)
    ref.set_experts_cut(c, kernel)
    E, N, K, T, k = 9, 96, 192, 70, 3
    n = T * k
    ex, w = ref.make_experts(c, 12000, E, N, K, bits)
    rng = np.random.default_rng(1)
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    x, y = to_dev(np.zeros((T, K), np.uint16)), to_dev(np.zeros((n, N // 2), np.uint16))
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    order, place = torch.zeros_like(ids), torch.zeros_like(ids)
    ws = torch.empty(max(1, ex.workspace_bytes(T)), dtype=torch.uint8, device="cuda")

    def call():
        c.group_rows(ids, n, E, off, order, place)
        c.experts_swiglu(ex, x, T, order, off, n, y, fan=k, ws=ws)

    sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        call()
    for it in range(3):
        hi = rng.integers(-1, E if it else 2, n).astype(np.int32)
        hx = bf16(randn(12100 + it, (T, K)))
        ids.copy_(to_dev(hi))
        x.copy_(to_dev(hx))
        y.fill_(0)
        sync()
        g.replay()
        sync()
        got = from_dev(y)
        offsets, horder, _ = ref.group(hi, E)
        held = int(offsets[-1])
        check(got[:held], w, hx, offsets, horder[:held] // k, True, bits)
        assert not got[held:].any()
        y.fill_(0)
        sync()
        call()
        c.synchronize()
        assert np.array_equal(from_dev(y), got)
    del g
    ex.close()
    c.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("T", [1, 6, 150])
def test_feed_forward(ctx, orc, bits, T):
    """Logits to tokens: route, group, gate and up, down, the weighted sum onto
    the shared output, each step from what the one before left."""
    E, k, H, F = 12, 4, 192, 160
    n = T * k
    gu, wgu = ref.make_experts(ctx, 12200, E, 2 * F, H, bits)
    # down takes K = F rounded up to whole groups: 192 columns, the last 32 zero
    FP = 192
    dn, wdn = ref.make_experts(ctx, 12300, E, H, FP, bits)
    x = bf16(randn(12400 + T, (T, H)))
    logits = randn(12500 + T, (T, E), 2.0)
    shared = bf16(randn(12600 + T, (T, H)))
    i32 = lambda size: torch.empty(size, dtype=torch.int32, device="cuda")
    ids, off, order, place = i32((T, k)), i32(E + 1), i32(n), i32(n)
    wt = torch.empty((T, k), dtype=torch.float32, device="cuda")
    h, y = to_dev(np.zeros((n, FP), np.uint16)), to_dev(np.zeros((n, H), np.uint16))
    out = to_dev(shared)
    xd, ld = to_dev(x), to_dev(logits)
    ws = torch.empty(max(gu.workspace_bytes(T), dn.workspace_bytes(n), 1), dtype=torch.uint8,
                     device="cuda")
    sync()
    ctx.topk_route(ld, T, E, k, ids, wt, score="sigmoid", scale=1.5)
    ctx.group_rows(ids, n, E, off, order, place)
    ctx.experts_swiglu(gu, xd, T, order, off, n, h, fan=k, ws=ws, ldy=FP)
    ctx.experts_lin(dn, h, n, None, off, n, y, ws=ws)
    ctx.experts_combine(y, n, place, wt, T, k, out, H, add=out)
    ctx.synchronize()
    wid, ww = ref.route(logits, k, score="sigmoid", scale=1.5)
    assert np.array_equal(from_dev(ids), wid)
    offsets, worder, wplace = ref.group(wid.reshape(-1), E)
    assert np.array_equal(from_dev(order), worder) and np.array_equal(from_dev(off), offsets)
    hh = from_dev(h)
    check(hh[:, :F], wgu, x, offsets, worder // k, True, bits)
    assert not hh[:, F:].any()
    check(from_dev(y), wdn, hh, offsets, np.arange(n), False, bits)
    want, bound = ref.combine(f32(from_dev(y)), wplace.reshape(T, k), from_dev(wt), f32(shared), n)
    assert np.all(np.abs(f32(from_dev(out)) - want) <= bound)
    # and the chain in 64 bits: four roundings to bf16 (h, y, out, and the
    # weights' to f32 or fp16 beside them), each at most BF16 / sqrt(3)
    h64, _ = ref.products(f32(x), wgu, offsets, worder // k, True, bits)
    h64 = np.concatenate([h64, np.zeros((n, FP - F))], 1)
    y64, _ = ref.products(h64, wdn, offsets, np.arange(n), False, bits)
    o64, _ = ref.combine(y64, wplace.reshape(T, k), ww, f32(shared), n)
    assert ref.rel(f32(from_dev(out)), o64) <= 2 * ref.REL
    gu.close()
    dn.close()


def test_products_refusals(ctx):
    ex, _ = ref.make_experts(ctx, 12700, 3, 40, 64, 16)
    x, y = to_dev(np.zeros((8, 64), np.uint16)), to_dev(np.zeros((8, 40), np.uint16))
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    order = torch.zeros(8, dtype=torch.int32, device="cuda")
    ok = dict(ex=ex, x=x, x_rows=8, order=order, offsets=off, n=8, y=y, fan=1)
    for kw in ({"n": -1}, {"fan": 0}, {"x_rows": -1}, {"x_rows": 0}, {"ldx": 56}, {"ldx": 68},
               {"ldy": 32}, {"ldy": 42}, {"x": None}, {"y": None}, {"offsets": None},
               {"y": x}, {"x": x.data_ptr() + 2}, {"order": None, "x_rows": 7},
               {"x_rows": 1 << 26}):
        with pytest.raises(m.MingError):
            ctx.experts_lin(**dict(ok, **kw))
    with pytest.raises(m.MingError, match="16"):     # 40 rows are not two halves of eights
        ctx.experts_swiglu(**ok)
    ctx.experts_lin(**dict(ok, n=0))
    other = m.Ctx(0)
    with pytest.raises(m.MingError, match="another"):
        other.experts_lin(**ok)
    other.close()
    with pytest.raises(m.MingError):                  # the context outlives its stacks
        m._check(m.lib().ming_ctx_destroy(ctx.h))
    ex.close()


@pytest.mark.parametrize("bits,kernel", [(16, 0), (16, 2), (4, 2)])
def test_shared_memory_and_sizes(ctx, cut, bits, kernel):
    """What every block reads may not be what others write; columns beside each
    other may. Calls of nothing, and of more than a launch holds."""
    E, N, K, n = 2, 64, 64, 20
    ex, w = ref.make_experts(ctx, 13200, E, N, K, bits)
    cut(kernel)
    offsets, order, src = ref.plan_of([12, 8], x_rows=n)
    x = bf16(randn(13300, (n, K)))
    both = np.zeros((n, K + N), np.uint16)
    both[:, :K] = x
    xy, od, fd = to_dev(both), to_dev(order), to_dev(offsets)
    ws = torch.zeros(ex.workspace_bytes(n) + 4096, dtype=torch.uint8, device="cuda")
    # 2^31 places of 2^16 columns: 2^32 tiles and more
    wide, _ = ref.make_experts(ctx, 13400, 1, 1 << 16, 64, bits)
    ok = dict(ex=ex, x=xy, x_rows=n, order=od, offsets=fd, n=n, y=xy.data_ptr() + 2 * K, ws=ws,
              ldx=K + N, ldy=K + N)
    sync()
    ctx.experts_lin(**ok)
    ctx.synchronize()
    check(from_dev(xy)[:, K:], w, x, offsets, src, False, bits)
    bad = [{"y": xy.data_ptr() + 2 * K - 16}, {"order": xy.data_ptr() + 2 * K},
           {"offsets": xy.data_ptr() + 2 * K + 4}]
    if ex.workspace_bytes(n):
        bad += [{"order": ws}, {"offsets": ws}, {"y": ws}, {"x": ws}]
    for kw in bad:
        with pytest.raises(m.MingError, match="share"):
            ctx.experts_lin(**dict(ok, **kw))
    if kernel:
        with pytest.raises(m.MingError, match="launch"):
            ctx.experts_lin(**dict(ok, n=2 ** 31 - 1, y=1 << 60, ldy=1 << 20, ex=wide))
    with pytest.raises(m.MingError, match="2\\^30"):
        ctx.experts_lin(**dict(ok, ldx=1 << 62))
    ctx.experts_lin(ex, None, 0, None, None, 0, None)
    wide.close()
    ex.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_outputs_past_32_bits(ctx, cut, bits):
    """Rows of y more than 2^32 bytes apart, and their sum from there."""
    E, N, K, n, ld = 3, 272, 128, 200, 1 << 24
    ex, w = ref.make_experts(ctx, 13700, E, N, K, bits)
    offsets, order, src = ref.plan_of([90, 0, 110], x_rows=40)
    x = bf16(randn(13800, (40, K)))
    xd, offd, od = to_dev(x), to_dev(offsets), to_dev(order)
    ws = torch.empty(max(1, ex.workspace_bytes(40)), dtype=torch.uint8, device="cuda")
    y = torch.empty((n, ld), dtype=torch.int16, device="cuda")
    for c in ref.CUTS[bits]:
        cut(c)
        y[:, :N + 8] = SENTINEL
        sync()
        ctx.experts_lin(ex, xd, 40, od, offd, n, y, ws=ws, ldy=ld)
        ctx.synchronize()
        got = from_dev(y[:, :N + 8].contiguous())
        assert np.all(got[:, N:] == SENTINEL)
        check(got[:, :N], w, x, offsets, src, False, bits)
    place = np.random.default_rng(2).permutation(n).astype(np.int32).reshape(n // 2, 2)
    wt = np.linspace(-1, 1, n, dtype=np.float32).reshape(n // 2, 2)
    pd, wd, out = to_dev(place), to_dev(wt), to_dev(np.zeros((n // 2, N), np.uint16))
    sync()
    ctx.experts_combine(y, n, pd, wd, n // 2, 2, out, N, ldy=ld)
    ctx.synchronize()
    want, bound = ref.combine(f32(got[:, :N]), place, wt, None, n)
    assert np.all(np.abs(f32(from_dev(out)) - want) <= bound)
    del y
    torch.cuda.empty_cache()
    ex.close()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("offsets", [[0, 300, 0, 300, 0, 300, 0], [300, 200, 100, 0, -5, 7, 9],
                                     [-9, 400, 2 ** 31 - 1, -2 ** 31, 50, 60, 2 ** 31 - 1],
                                     [7, 7, 7, 7, 7, 7, 7]])
def test_what_is_no_plan_stays_inside(ctx, cut, bits, offsets):
    """Offsets that descend or leave the places, an order out of range: some rows of y,
    none outside, and the context goes on."""
    E, N, K, n = 6, 272, 128, 300
    ex, w = ref.make_experts(ctx, 13500, E, N, K, bits)
    x = bf16(randn(13600, (20, K)))
    order = np.random.default_rng(1).integers(-2 ** 31, 2 ** 31, n).astype(np.int32)
    xd, offd, od = to_dev(x), to_dev(np.array(offsets, np.int32)), to_dev(order)
    ws = torch.empty(max(1, ex.workspace_bytes(20)), dtype=torch.uint8, device="cuda")
    for c in ref.CUTS[bits]:
        cut(c)
        y = torch.full(((n + 4) * N,), SENTINEL, dtype=torch.int16, device="cuda")
        sync()
        ctx.experts_lin(ex, xd, 20, od, offd, n, y[2 * N:], fan=1, ws=ws)
        ctx.synchronize()
        assert bool((y[:2 * N] == SENTINEL).all()) and bool((y[(n + 2) * N:] == SENTINEL).all())
    good, order, src = ref.plan_of([40, 0, 60, 0, 0, 200], x_rows=20)
    cut(-1)
    check(run(ctx, ex, False, x, good, order, order.size), w, x, good, src, False, bits)
    ex.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_create_refusals(ctx, bits):
    pack, _ = ref.stack(12800, 2, 16, 64, bits)
    for kw in ({"bits": 5}, {"group": 32}):
        with pytest.raises(m.MingError):
            m.Experts.quantized(ctx, pack["codes"], pack["scales"], pack["biases"],
                                kw.get("bits", bits), kw.get("group", 64))
    bad = pack["scales"].copy()
    bad[1, 3, 0] = 0x7f00                             # about 2^127
    with pytest.raises(m.MingError, match="fp16") as e:
        m.Experts.quantized(ctx, pack["codes"], bad, pack["biases"], bits)
    assert e.value.code == m.ERR_RANGE
    with pytest.raises(m.MingError):
        m.Experts.dense(ctx, np.zeros((2, 12, 64), np.uint16))
    with pytest.raises(m.MingError):
        m.Experts.dense(ctx, np.zeros((2, 16, 72), np.uint16))


@pytest.mark.parametrize("bits,kernel", [(4, 2), (4, 4), (8, 2), (8, 8)])
def test_rows_that_no_place_names_may_hold_anything(ctx, cut, bits, kernel):
    """Choices that were dropped leave rows of h unwritten and tokens unread: what lies
    there is no range fault, in the gathered product or in the one after it."""
    E, k, T, H, F = 6, 3, 260, 192, 320
    n = T * k
    gu, wgu = ref.make_experts(ctx, 18700, E, 2 * F, H, bits)
    dn, wdn = ref.make_experts(ctx, 18750, E, H, F, bits)
    rng = np.random.default_rng(kernel)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < 0.3] = -1
    away = rng.permutation(T)[:25]
    ids[away] = E + 3
    x = bf16(randn(18800, (T, H)))
    x[away, rng.integers(0, H, 25)] = np.resize(np.uint16([0x7f80, 0x7fc0, 0xff80, 0x4780, 0xc7ff]), 25)
    offsets, order, _ = ref.group(ids.reshape(-1), E)
    held = int(offsets[-1])
    assert 0 < held < n - 75
    h = np.resize(np.uint16([0x7f80, 0x7fc0, 0x4780]), (n, F))
    xd, hd, yd = to_dev(x), to_dev(h), to_dev(np.full((n, H), SENTINEL, np.uint16))
    ws = torch.empty(max(gu.workspace_bytes(T), dn.workspace_bytes(n)), dtype=torch.uint8, device="cuda")
    od, fd = to_dev(order), to_dev(offsets)
    cut(kernel)
    sync()
    ctx.experts_swiglu(gu, xd, T, od, fd, n, hd, fan=k, ws=ws)
    ctx.synchronize()
    ctx.experts_lin(dn, hd, n, None, fd, n, yd, ws=ws)
    ctx.synchronize()
    hh, y = from_dev(hd), from_dev(yd)
    check(hh[:held], wgu, x, offsets, order[:held] // k, True, bits)
    check(y[:held], wdn, hh, offsets, np.arange(held), False, bits)
    assert np.array_equal(hh[held:], h[held:]) and np.all(y[held:] == SENTINEL)
    gu.close()
    dn.close()


@pytest.mark.parametrize("bits,kernel", [(4, 2), (4, 4), (8, 2), (8, 8)])
def test_a_row_that_a_place_names_is_reported(ctx, cut, bits, kernel):
    """Wherever it stands among the places: first and last of a group and of its tiles."""
    E, N, K, counts = 3, 560, 128, [300, 0, 517]
    ex, _ = ref.make_experts(ctx, 18900, E, N, K, bits)
    offsets, _, _ = ref.plan_of(counts)
    n = sum(counts)
    x, fd = to_dev(bf16(randn(18950, (n, K)))), to_dev(offsets)
    y = to_dev(np.zeros((n, N), np.uint16))
    ws = torch.empty(ex.workspace_bytes(n), dtype=torch.uint8, device="cuda")
    cut(kernel)
    for at in (0, 31, 64, 150, 299, 300, 558, n - 1):
        was = x[at, K - 1].clone()
        x[at, K - 1] = 0x4780
        sync()
        ctx.experts_lin(ex, x, n, None, fd, n, y, ws=ws)
        with pytest.raises(m.MingError) as e:
            ctx.synchronize()
        assert e.value.code == m.ERR_RANGE
        x[at, K - 1] = was
        sync()
        ctx.experts_lin(ex, x, n, None, fd, n, y, ws=ws)
        ctx.synchronize()
    ex.close()


@pytest.mark.parametrize("bits,kernel", [(4, 0), (16, 0), (4, 2), (16, 4)])
def test_counts_past_an_int(ctx, cut, bits, kernel):
    """Places and choices whose counts pass 2^31 before they end are refused by their
    number alone: the arrays are small."""
    ex, _ = ref.make_experts(ctx, 19900, 1, 16, 64, bits)
    x, y = to_dev(np.zeros((8, 64), np.uint16)), to_dev(np.zeros((8, 16), np.uint16))
    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    w = torch.zeros(8, device="cuda")
    ws = torch.empty(4096, dtype=torch.uint8, device="cuda")
    cut(kernel)
    for n in ((1 << 30) + 1, 2 ** 31 - 16, 2 ** 31 - 1):
        with pytest.raises(m.MingError, match="2\\^30") as e:
            ctx.experts_lin(ex, x, 8, i, i, n, 1 << 56, ws=ws)
        assert e.value.code == 2
        with pytest.raises(m.MingError, match="2\\^30"):
            ctx.experts_swiglu(ex, x, 8, i, i, n, 1 << 56, ws=ws)
        with pytest.raises(m.MingError, match="2\\^30"):
            ctx.experts_combine(y, 8, i, w, 1, n, 1 << 56, 16)
    ex.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("K", [64, 512, 1024, 2112])
def test_w4_sums_of_few_rows_are_exact_where_f32_is(ctx, cut, gated, K):
    """Whole numbers whose sums with codes of up to 31 stay below 2^24: every f32 sum is
    exact, in any order, and what is left of them after the bias is a small number. Sums
    of 128 more than the codes would pass 2^25 and lose it."""
    E, N, T = 2, 32, 5
    rng = np.random.default_rng(K)
    # a group: one x of 1 under a code of its own, the others large under 8
    x = (rng.integers(129, 256, (T, K)) * 32).astype(np.float32)
    at = 64 * np.arange(K // 64) + rng.integers(0, 64, K // 64)
    x[:, at] = 1.0
    assert 31 * x.reshape(T, -1, 64).sum(-1).max() < 2 ** 24
    assert 136 * x.reshape(T, -1, 64).sum(-1).min() > 2 ** 25
    q = np.full((E, 2 * N if gated else N, K), 8, np.uint32)
    q[:, :, at] = rng.integers(1, 16, q[:, :, at].shape)
    if gated:                                   # the gates' sums 32 a group, so silu is them
        q[:, :N, at] = 8 + 7
        extra = 64 * np.arange(K // 64) + (at + 1) % 64
        x[:, extra] = 8.0
        q[:, :N, extra] = 8 + 4
    codes = (q.reshape(*q.shape[:2], K // 8, 8) << (4 * np.arange(8, dtype=np.uint32))).sum(-1)
    ones = np.full(q.shape[:2] + (K // 64,), 0x3f80, np.uint16)
    ex = m.Experts.quantized(ctx, codes.astype(np.uint32), ones, np.full_like(ones, 0xc100), 4)
    offsets, order, src = ref.plan_of([3, 40], x_rows=T)
    cut(0)
    got = f32(run(ctx, ex, gated, bf16(x), offsets, order, order.size)).astype(np.float64)
    e = np.repeat([0, 1], [3, 40])
    t = np.einsum("pk,pnk->pn", x[src].astype(np.float64), q[e].astype(np.float64) - 8.0)
    if gated:
        assert (t[:, :N] == 39 * (K // 64)).all()
        want = t[:, :N] * t[:, N:]
        # silu(g) is g but for 2 of its own steps and e^-39: one rounding to bf16
        assert np.all(np.abs(got - want) <= (ref.BF16 + 4 * ref.F32) * np.abs(want))
    else:
        assert np.abs(t).max() <= 256            # exact in bf16
        assert np.array_equal(got, t)
    ex.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_sources_on_the_host_and_on_the_device(ctx, bits):
    """The same stack from host arrays, in more than one piece, from device arrays, and
    from device arrays that start beside a word."""
    E, N, K = 6, 2048, 8192 if bits == 8 else 16384      # 16 MiB of codes an expert
    rng = np.random.default_rng(bits)
    codes = rng.integers(0, 2 ** 32, (E, N, K * bits // 32), dtype=np.uint32)
    sc = bf16(rng.choice([0.5, 0.25, 2.0], (E, N, K // 64)).astype(np.float32) / 1024)
    bi = bf16(rng.choice([-0.5, -0.25, 1.0], (E, N, K // 64)).astype(np.float32) / 16)
    dev = [to_dev(a.view(np.int32) if a is codes else a) for a in (codes, sc, bi)]
    odd = []
    for t in dev:
        b = torch.empty(t.numel() * t.element_size() + 1, dtype=torch.uint8, device="cuda")
        b[1:] = t.reshape(-1).view(torch.uint8)
        odd.append(b[1:])
    n = 8
    x, y = to_dev(bf16(randn(20000, (n, K)))), to_dev(np.zeros((n, N), np.uint16))
    off = to_dev(np.minimum(np.arange(E + 1) * 2, n).astype(np.int32))
    got = []
    sync()
    for src in (None, dev, odd):
        if src is None:
            ex = m.Experts.quantized(ctx, codes, sc, bi, bits)
        else:
            h = m.C.c_void_p()
            m._check(m.lib().ming_experts_create(ctx.h, E, N, K, bits, 64, *map(m._ptr, src), 1,
                                                 m.C.byref(h)))
            ex = m.Experts(ctx, h)
        for shift in (0, 4):                             # two rows to each of four experts
            o = torch.zeros_like(off)
            o[shift // 2:] = off[:E + 1 - shift // 2]
            sync()
            ctx.experts_lin(ex, x, n, None, o, n, y)
            ctx.synchronize()
            got.append(from_dev(y))
        ex.close()
    assert np.array_equal(got[0], got[2]) and np.array_equal(got[0], got[4])
    assert np.array_equal(got[1], got[3]) and np.array_equal(got[1], got[5])
    assert not np.array_equal(got[0], got[1])


@pytest.mark.parametrize("on_device", [True, False])
def test_a_stack_needs_its_own_memory_and_little_more(ctx, on_device):
    """Created where three quarters of its size again are free, beside its sources."""
    E, N, K = 16, 8192, 16384                            # 2 GiB of w8 codes
    codes = torch.zeros((E, N, K // 4), dtype=torch.int32, device="cuda" if on_device else "cpu")
    sc = torch.full((E, N, K // 64), 0x3f80, dtype=torch.int16, device=codes.device)
    size = codes.numel() * 4 + sc.numel() * 4
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    fill = torch.empty(free - size * 7 // 4, dtype=torch.uint8, device="cuda")
    try:
        ex = m.Experts.quantized(ctx, codes, sc, sc, 8, on_device=on_device)
        assert (ex.n_experts, ex.N, ex.K) == (E, N, K)
        ex.close()
    finally:
        del fill, codes, sc
        torch.cuda.empty_cache()


@pytest.mark.parametrize("K", [1088, 2048, 4160])
@pytest.mark.parametrize("counts", [[0, 1, 0, 2], [17, 1, 40, 3]])
def test_wide_and_narrow_few_row_blocks(ctx, cut, counts, K):
    """Dense plain products past K = 1024, few places and many: blocks of 16 columns and
    of 32, a row's bits its own whichever ran."""
    E, N = 4, 4104
    ex, w = ref.make_experts(ctx, 20100, E, N, K, 16)
    offsets, order, src = ref.plan_of(counts, x_rows=9)
    x = bf16(randn(20200, (9, K)))
    cut(0)
    got = run(ctx, ex, False, x, offsets, order, order.size)
    check(got, w, x, offsets, src, False, 16)
    one = np.zeros(E + 1, np.int32)
    one[2:] = 1                                          # the first place of expert 1 alone
    at = int(offsets[1])
    alone = run(ctx, ex, False, x, one, order[at:at + 1], 1)
    assert np.array_equal(alone[0], got[at])
    ex.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("where", ["pinned", "other device"])
def test_sources_that_are_not_the_devices_own(ctx, bits, where):
    """Arrays said to be on the device that lie in host memory the device can reach, or
    on another device, come over by copies."""
    if where == "other device" and torch.cuda.device_count() < 2:
        pytest.skip("one device")
    E, N, K = 3, 48, 192
    pack, w = ref.stack(20300, E, N, K, bits)
    there = []
    for a in pack.values():
        t = torch.from_numpy(np.ascontiguousarray(a).view(np.int32 if a.dtype == np.uint32 else np.int16))
        there.append(t.pin_memory() if where == "pinned" else t.to("cuda:1"))
    if bits == 16:
        ex = m.Experts.dense(ctx, there[0], on_device=True)
    else:
        ex = m.Experts.quantized(ctx, *there, bits, on_device=True)
    offsets, order, src = ref.plan_of([5, 0, 9], x_rows=20)
    x = bf16(randn(20400, (20, K)))
    check(run(ctx, ex, False, x, offsets, order, order.size), w, x, offsets, src, False, bits)
    ex.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_inputs_as_far_apart_as_they_may_be(ctx, cut, bits):
    """Rows of x whose last lies 2 GiB from the first: the bits of rows side by side."""
    E, N, K, T = 3, 272, 128, 64
    ld = ((1 << 30) - 1) // T // 8 * 8
    ex, w = ref.make_experts(ctx, 20500, E, N, K, bits)
    offsets, order, src = ref.plan_of([90, 0, 110], x_rows=T)
    order[5], src[5] = T - 1, T - 1
    n = order.size
    x = bf16(randn(20600, (T, K)))
    far = torch.empty((T, ld), dtype=torch.int16, device="cuda")
    far[:, :K] = to_dev(x)
    od, fd, y = to_dev(order), to_dev(offsets), to_dev(np.zeros((n, N), np.uint16))
    ws = torch.empty(max(1, ex.workspace_bytes(T)), dtype=torch.uint8, device="cuda")
    for c in ref.CUTS[bits]:
        cut(c)
        near = run(ctx, ex, False, x, offsets, order, n)
        check(near, w, x, offsets, src, False, bits)
        y.zero_()
        sync()
        ctx.experts_lin(ex, far, T, od, fd, n, y, ws=ws, ldx=ld)
        ctx.synchronize()
        assert np.array_equal(from_dev(y), near)
    del far
    torch.cuda.empty_cache()
    ex.close()
