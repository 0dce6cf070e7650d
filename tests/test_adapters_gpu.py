"""ming_lin_adapters: a projection whose rows carry the adapters of many
requests, against 64-bit arithmetic: every weight type and route, from one row
to many tiles, requests that end inside tiles, rows without an adapter, ranks
that are no multiple of 8, strengths, strides, captured calls."""
import re

import numpy as np
import pytest
import torch

import ming_dit_amd as m
import rows_ref as ref
from helpers import (bf16, dense_plan, f32, from_dev, make_weight, plan_rows, randn, split_plan,
                     sync, to_dev)

pytestmark = pytest.mark.gpu
SENTINEL = 0x4242


def weight(ctx, seed, N, K, bits):
    pack, w = make_weight(seed, N, K, bits, std=0.02 if bits != 16 else 1.0 / np.sqrt(K))
    if bits == 16:
        return m.QWeight.dense(ctx, pack["w"]), w
    return m.QWeight.quantized(ctx, pack["codes"], pack["scales"], pack["biases"], bits), w


def make_bank(ctx, seed, N, K, ranks, cap=None, max_rank=None, std=0.05):
    """(bank, {id: (A, B, fold)}): adapter i of ranks[i], 0 for none."""
    bank = m.Adapters(ctx, N, K, cap or len(ranks), max_rank or max(ranks))
    held = {}
    for i, r in enumerate(ranks):
        if r == 0:
            continue
        A = bf16(randn(seed + 2 * i, (r, K), 1.0 / np.sqrt(K)))
        B = bf16(randn(seed + 2 * i + 1, (N, r), std))
        fold = (1.0, 0.5, 2.0)[i % 3]
        bank.set(i, A, B, fold)
        held[i] = (f32(A), f32(B), fold)
    return bank, held


def call(ctx, qw, bank, x, ids, scale, padx=0, pady=0):
    M = x.shape[0]
    xs = np.full((M, qw.K + padx), 0x7fc0, np.uint16)
    xs[:, :qw.K] = x
    xd, y = to_dev(xs), to_dev(np.full((M + 2, qw.N + pady), SENTINEL, np.uint16))
    need = ctx.lin_adapters_workspace_bytes(qw, bank, M)
    ws = torch.full((need + 256,), 0xAB, dtype=torch.uint8, device="cuda")
    idd, sd = to_dev(ids.astype(np.int32)), None if scale is None else to_dev(scale)
    sync()
    ctx.lin_adapters(qw, bank, xd, y, M, idd, sd, ws[:need], ldx=qw.K + padx, ldy=qw.N + pady)
    ctx.synchronize()
    assert bool((ws[need:] == 0xAB).all())
    y = from_dev(y)
    assert np.all(y[M:] == SENTINEL) and np.all(y[:, qw.N:] == SENTINEL)
    return y[:M, :qw.N]


def check(got, x, w, held, ids, scale, bits):
    s = np.ones(len(ids), np.float32) if scale is None else scale
    want, bound = ref.adapters(f32(x), w, held, ids, s, bits)
    worst = np.max(np.abs(f32(got) - want) / bound)
    assert worst <= 1.0, worst
    if got.size > 4000:
        # the output's rounding and, on the rows' sums, T's
        assert ref.rel(f32(got), want) <= ref.REL * np.sqrt(2.0)


def requests(M, seed, held, cuts=None):
    """Ids and strengths of requests that lie one after another."""
    rng = np.random.default_rng(seed)
    n = min(M, 7) if cuts is None else cuts
    edges = np.sort(rng.choice(np.arange(1, M), n - 1, replace=False)) if n > 1 else []
    lengths = np.diff(np.concatenate([[0], edges, [M]])).astype(int)
    ids = rng.integers(-1, held, n)
    s = rng.choice([1.0, 0.8, -0.3, 0.0], n).astype(np.float32)
    return np.repeat(ids, lengths), np.repeat(s, lengths)


RANKS = (16, 4, 33, 8, 64, 7)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("M", [1, 2, 8, 9, 31, 37, 64, 130, 257, 700])
def test_rows(ctx, bits, M):
    N, K = 264, 320
    qw, w = weight(ctx, 13000, N, K, bits)
    bank, held = make_bank(ctx, 13100, N, K, RANKS)
    x = bf16(randn(13200 + M, (M, K)))
    ids, s = requests(M, M, len(RANKS))
    got = call(ctx, qw, bank, x, ids, s, padx=8, pady=8)
    check(got, x, w, held, ids, s, bits)
    # every row its own, in no order
    ids = np.random.default_rng(M).integers(-1, len(RANKS), M)
    got = call(ctx, qw, bank, x, ids, None)
    check(got, x, w, held, ids, None, bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("M,N,K", [(5, 1024, 2048), (40, 1024, 2048), (300, 2048, 640),
                                   (1100, 1280, 256), (2300, 2304, 192), (600, 64, 128)])
def test_shapes(ctx, bits, M, N, K):
    """Split and unsplit launches, narrow weights, one or several tile rows."""
    qw, w = weight(ctx, 13300, N, K, bits)
    bank, held = make_bank(ctx, 13400, N, K, RANKS)
    x = bf16(randn(13500 + M, (M, K)))
    ids, s = requests(M, N, len(RANKS))
    got = call(ctx, qw, bank, x, ids, s)
    check(got, x, w, held, ids, s, bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("M", [3, 40, 600])
def test_every_row_its_own_adapter(ctx, bits, M):
    """As many adapters as rows (up to 90), so tiles hold many."""
    N, K, n = 136, 256, min(M, 90)
    qw, w = weight(ctx, 13600, N, K, bits)
    bank, held = make_bank(ctx, 13700, N, K, [8 + i % 9 for i in range(n)])
    x = bf16(randn(13800 + M, (M, K)))
    ids = np.random.default_rng(M).permutation(np.arange(M) % n)
    got = call(ctx, qw, bank, x, ids, None)
    check(got, x, w, held, ids, None, bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("route", ["general", "wide"])
@pytest.mark.parametrize("M", [4, 300])
def test_routes(ctx, bits, route, M):
    N, K = 264, 320
    qw, w = weight(ctx, 13900, N, K, bits)
    bank, held = make_bank(ctx, 14000, N, K, RANKS)
    x = bf16(randn(14100, (M, K)))
    ids, s = requests(M, 3, len(RANKS))
    ctx.set_route(route)
    try:
        got = call(ctx, qw, bank, x, ids, s)
    finally:
        ctx.set_route("auto")
    check(got, x, w, held, ids, s, bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("M,N,K", [(3, 264, 320), (37, 1024, 2048), (300, 264, 320),
                                   (1300, 1280, 256)])
def test_rows_without_an_adapter_are_plain_rows(ctx, bits, M, N, K):
    """Strength 0, an id of none, of nothing bound and out of range: ming_lin's
    bits, all of them; and a row's own bits do not depend on its neighbours'
    adapters (the sign of a zero aside)."""
    qw, _ = weight(ctx, 14200, N, K, bits)
    bank, _ = make_bank(ctx, 14300, N, K, (16, 0, 40))
    x = bf16(randn(14400 + M, (M, K)))
    xd, y = to_dev(x), to_dev(np.zeros((M, N), np.uint16))
    sync()
    ctx.lin(qw, xd, y, M)
    ctx.synchronize()
    plain = from_dev(y)
    none = np.resize(np.array([-1, 1, 3, 2 ** 31 - 1, -2 ** 31]), M)
    assert np.array_equal(call(ctx, qw, bank, x, none, None), plain)
    off = np.zeros(M, np.float32)
    off[::2] = -0.0
    assert np.array_equal(call(ctx, qw, bank, x, np.full(M, 2), off), plain)
    mixed = np.where(np.arange(M) % 3 == 0, 0, none)
    a = call(ctx, qw, bank, x, mixed, None)
    b = call(ctx, qw, bank, x, np.where(mixed == 0, 0, 2), None)
    mine = mixed == 0
    same = (a == b) | ((a | b) & 0x7fff == 0)
    assert same[mine].all()
    same = (a == plain) | ((a | plain) & 0x7fff == 0)
    assert same[~mine].all()
    assert not np.array_equal(a[mine], plain[mine])
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [16])
def test_a_bad_row_stays_its_own(ctx, bits):
    N, K = 264, 320
    for M in (6, 40, 300):
        qw, _ = weight(ctx, 14500, N, K, bits)
        bank, _ = make_bank(ctx, 14600, N, K, (16, 24))
        x = bf16(randn(14700, (M, K)))
        ids, s = np.arange(M) % 2, np.full(M, 0.5, np.float32)
        clean = call(ctx, qw, bank, x, ids, s)
        x[3, 1] = 0x7f80
        s[4] = np.inf
        got = call(ctx, qw, bank, x, ids, s)
        others = ~np.isin(np.arange(M), (3, 4))
        assert np.array_equal(got[others], clean[others])
        assert not np.isfinite(f32(got[3:5])).any()
        bank.close()
        qw.close()


def test_concat_weight(ctx):
    """q|k|v as one weight, its bank as wide as the three."""
    N, K, M = 256, 192, 90
    parts = [weight(ctx, 14800 + i, N, K, 4) for i in range(3)]
    cat = m.QWeight.concat(ctx, [p[0] for p in parts])
    w = np.concatenate([p[1] for p in parts])
    for Mi in (4, 90, 1000):
        bank, held = make_bank(ctx, 14900, 3 * N, K, RANKS)
        x = bf16(randn(15000, (Mi, K)))
        ids, s = requests(Mi, 5, len(RANKS))
        check(call(ctx, cat, bank, x, ids, s), x, w, held, ids, s, 4)
        bank.close()
    cat.close()
    for p in parts:
        p[0].close()


def test_bound_slots_take_no_part(ctx):
    N, K, M = 136, 128, 40
    qw, w = weight(ctx, 15100, N, K, 16)
    bank, held = make_bank(ctx, 15200, N, K, (8,))
    x = bf16(randn(15300, (M, K)))
    before = call(ctx, qw, bank, x, np.zeros(M), None)
    qw.bind_lora(0, bf16(randn(15301, (4, K))), bf16(randn(15302, (N, 4))))
    assert np.array_equal(call(ctx, qw, bank, x, np.zeros(M), None), before)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits,M", [(4, 5), (4, 300), (16, 40), (16, 300), (8, 40)])
def test_captured_call_follows_the_requests(bits, M):
    """A captured call replays with the ids, strengths and factors of the
    moment; eager calls of another size run between the replays."""
    s = torch.cuda.Stream()
    c = m.Ctx(0, s.cuda_stream)
    N, K = 264, 1024
    qw, w = weight(c, 15400, N, K, bits)
    bank, held = make_bank(c, 15500, N, K, (8, 0, 16, 40), max_rank=48)
    x, y = to_dev(np.zeros((M, K), np.uint16)), to_dev(np.zeros((M, N), np.uint16))
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    sc = torch.zeros(M, dtype=torch.float32, device="cuda")
    ws = torch.empty(c.lin_adapters_workspace_bytes(qw, bank, M), dtype=torch.uint8, device="cuda")
    sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        c.lin_adapters(qw, bank, x, y, M, ids, sc, ws)
    xo = bf16(randn(15600, (M + 200, K)))
    for it in range(3):
        if it == 2:                                    # a larger rank, bound after the capture
            A, B = bf16(randn(15601, (48, K), 0.03)), bf16(randn(15602, (N, 48), 0.05))
            bank.set(1, A, B, 1.0)
            held[1] = (f32(A), f32(B), 1.0)
        hid, hs = requests(M, 10 + it, 4)
        hx = bf16(randn(15610 + it, (M, K)))
        for d, h in ((ids, hid.astype(np.int32)), (sc, hs), (x, hx)):
            d.copy_(to_dev(h))
        y.zero_()
        sync()
        g.replay()
        sync()
        got = from_dev(y)
        check(got, hx, w, held, hid, hs, bits)
        y.zero_()
        oid, osc = requests(M + 200, it, 4)
        call(c, qw, bank, xo, oid, osc)
        c.lin_adapters(qw, bank, x, y, M, ids, sc, ws)
        c.synchronize()
        assert np.array_equal(from_dev(y), got)
    del g
    bank.close()
    qw.close()
    c.close()


def test_set_replaces_and_clear_empties(ctx):
    N, K, M = 64, 128, 20
    qw, w = weight(ctx, 15700, N, K, 4)
    bank, held = make_bank(ctx, 15800, N, K, (8, 16), max_rank=32)
    x = bf16(randn(15900, (M, K)))
    ids = np.arange(M) % 2
    assert (bank.rank(0), bank.rank(1), bank.rank(2)) == (8, 16, 0)
    check(call(ctx, qw, bank, x, ids, None), x, w, held, ids, None, 4)
    A, B = bf16(randn(15901, (20, K), 0.1)), bf16(randn(15902, (N, 20), 0.05))
    bank.set(0, A, B, -1.5)
    held[0] = (f32(A), f32(B), -1.5)
    bank.clear(1)
    del held[1]
    assert (bank.rank(0), bank.rank(1)) == (20, 0)
    check(call(ctx, qw, bank, x, ids, None), x, w, held, ids, None, 4)
    # device sources
    bank.set(1, to_dev(A), to_dev(B), 1.0, on_device=True)
    held[1] = (f32(A), f32(B), 1.0)
    check(call(ctx, qw, bank, x, ids, None), x, w, held, ids, None, 4)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("M,N,K,ranks", [
    (900, 264, 320, (16, 4, 32, 8, 7)),              # x.A of two chunks a pass
    (800, 136, 576, tuple(8 + i % 57 for i in range(70))),   # many adapters, many passes
    (768, 72, 4160, RANKS), (767, 72, 4160, RANKS),  # many K steps, the last one short
    (5, 72, 4160, RANKS), (40, 72, 4160, RANKS),
    (900, 512, 4096, RANKS), (760, 512, 4096, RANKS), (60, 2048, 1088, (512, 130, 1))])
def test_large_and_long(ctx, bits, M, N, K, ranks):
    """Both forms of the down-projection with K past one reading of it, and with
    more chunks than a pass holds; splits too wide for blocks beside them."""
    qw, w = weight(ctx, 16300, N, K, bits)
    bank, held = make_bank(ctx, 16400, N, K, ranks)
    x = bf16(randn(16500 + M, (M, K)))
    ids, s = requests(M, N, len(ranks), cuts=min(M, 2 * len(ranks)))
    check(call(ctx, qw, bank, x, ids, s, padx=8), x, w, held, ids, s, bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,tiles,stages", [(3460, 41, 6), (6560, 22, 6)])
def test_rows_in_two_heights(ctx, bits, M, tiles, stages):
    """A plan of full tiles and a rest of lower ones: requests across the seam."""
    N, K = 256 * tiles - 32, 64 * stages
    p = plan_rows(M, tiles, stages, False)
    assert 0 < p.rows_main < M and split_plan(M, N, K)[0] < 2
    qw, w = weight(ctx, 16600, N, K, bits)
    bank, held = make_bank(ctx, 16700, N, K, RANKS)
    x = bf16(randn(16800, (M, K)))
    ids, s = requests(M, 3, len(RANKS), cuts=9)
    seam = p.rows_main
    ids[seam - 20:seam + 30], s[seam - 20:seam + 30] = 4, 0.7
    got = call(ctx, qw, bank, x, ids, s)
    some = np.unique(np.concatenate([np.arange(0, M, 61), np.arange(seam - 40, seam + 50), [M - 1]]))
    check(got[some], x[some], w, held, ids[some], s[some], bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("M,N,K", [(40, 64, 64), (600, 128, 192), (1500, 192, 576),
                                   (3000, 1024, 1024), (3000, 192, 4096), (1500, 320, 4096)])
def test_dense_splits(ctx, M, N, K):
    """Narrow dense weights: one slice takes what the adapters add as a plane,
    several add it in their sum."""
    qw, w = weight(ctx, 16900, N, K, 16)
    assert dense_plan(M, N, K)[2] >= 1
    bank, held = make_bank(ctx, 17000, N, K, RANKS)
    x = bf16(randn(17100 + M, (M, K)))
    ids, s = requests(M, 5, len(RANKS), cuts=12)
    some = np.unique(np.concatenate([np.arange(0, M, 7), [M - 1]]))
    got = call(ctx, qw, bank, x, ids, s)[some]
    check(got, x[some], w, held, ids[some], s[some], 16)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits,M,N,K", [(4, 1500, 2040, 1088), (8, 1500, 2040, 1088),
                                        (16, 3000, 1024, 4096)])
def test_sums_of_many_rows(ctx, bits, M, N, K):
    """A split whose sum has work for the chip in its widest blocks."""
    assert (split_plan(M, N, K)[0] if bits != 16 else dense_plan(M, N, K)[2]) >= 2
    assert (M + 15) // 16 * ((N + 255) // 256) >= 512
    qw, w = weight(ctx, 17800, N, K, bits)
    bank, held = make_bank(ctx, 17900, N, K, RANKS)
    x = bf16(randn(18000, (M, K)))
    ids, s = requests(M, 6, len(RANKS), cuts=30)
    ids[100:140] = np.arange(40) % len(RANKS)             # a row its own, in turn
    some = np.unique(np.concatenate([np.arange(0, M, 13), np.arange(96, 144), [M - 1]]))
    got = call(ctx, qw, bank, x, ids, s)[some]
    check(got, x[some], w, held, ids[some], s[some], bits)
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits,M,N,K", [(4, 37, 1024, 2048), (8, 64, 2048, 1088),
                                        (16, 37, 1024, 2048), (16, 130, 512, 4096)])
def test_bits_do_not_depend_on_the_bank(ctx, bits, M, N, K):
    """A bank of two adapters and one of forty run other launches to the same bits."""
    qw, w = weight(ctx, 18100, N, K, bits)
    few, held = make_bank(ctx, 18200, N, K, (24, 64), cap=40, max_rank=64)
    many, _ = make_bank(ctx, 18200, N, K, (24, 64) + (64,) * 38)
    x = bf16(randn(18300 + M, (M, K)))
    ids, s = np.arange(M) % 3 - 1, np.linspace(-1, 1, M).astype(np.float32)
    a = call(ctx, qw, few, x, ids, s)
    check(a, x, w, held, ids, s, bits)
    assert np.array_equal(call(ctx, qw, many, x, ids, s), a)
    for h in (few, many, qw):
        h.close()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("M,N,K", [(6, 64, 128), (200, 264, 128), (300, 1024, 2048)])
def test_outputs_past_32_bits(ctx, bits, M, N, K):
    """Rows of y more than 2^32 bytes apart: the bits of rows beside each other."""
    ld = 1 << 30 if M == 6 else 1 << 24
    qw, _ = weight(ctx, 18400, N, K, bits)
    bank, _ = make_bank(ctx, 18500, N, K, RANKS)
    x = bf16(randn(18600, (M, K)))
    ids, s = requests(M, 8, len(RANKS))
    want = call(ctx, qw, bank, x, ids, s)
    y = torch.empty((M, ld), dtype=torch.int16, device="cuda")
    xd, idd, sd = to_dev(x), to_dev(ids.astype(np.int32)), to_dev(s)
    ws = torch.empty(ctx.lin_adapters_workspace_bytes(qw, bank, M), dtype=torch.uint8,
                     device="cuda")
    sync()
    ctx.lin_adapters(qw, bank, xd, y, M, idd, sd, ws, ldy=ld)
    ctx.synchronize()
    assert np.array_equal(from_dev(y[:, :N].contiguous()), want)
    del y
    torch.cuda.empty_cache()
    bank.close()
    qw.close()


def test_two_contexts_at_once(ctx):
    """Calls on two streams, a workspace each, over one x: the bits of one alone."""
    N, K, M = 1024, 2048, 200
    x = to_dev(bf16(randn(17200, (M, K))))
    ids = torch.arange(M, dtype=torch.int32, device="cuda") % 3
    got = []
    held = []
    for i in range(2):
        s = torch.cuda.Stream()
        c = m.Ctx(0, s.cuda_stream)
        qw, _ = weight(c, 17300, N, K, 4)
        bank, _ = make_bank(c, 17400, N, K, (16, 40, 8))
        y = to_dev(np.zeros((M, N), np.uint16))
        ws = torch.empty(c.lin_adapters_workspace_bytes(qw, bank, M), dtype=torch.uint8,
                         device="cuda")
        held.append((s, c, qw, bank, y, ws))
    sync()
    for _ in range(20):
        for _, c, qw, bank, y, ws in held:
            c.lin_adapters(qw, bank, x, y, M, ids, None, ws)
    sync()
    for _, c, qw, bank, y, ws in held:
        got.append(from_dev(y))
        y.zero_()
    sync()
    for i, (_, c, qw, bank, y, ws) in enumerate(held):
        c.lin_adapters(qw, bank, x, y, M, ids, None, ws)
        c.synchronize()
        assert np.array_equal(from_dev(y), got[i])
        bank.close()
        qw.close()
        c.close()
    assert np.array_equal(got[0], got[1])


def test_shared_memory_is_refused(ctx):
    """Blocks resolve their rows by themselves while others store: what they read
    may not be what they write. Columns beside each other are not shared."""
    N, K, M = 64, 64, 20
    qw, w = weight(ctx, 17500, N, K, 16)
    bank, held = make_bank(ctx, 17600, N, K, (8, 24))
    x = bf16(randn(17700, (M, K)))
    both = np.zeros((M, K + N), np.uint16)
    both[:, :K] = x
    xy = to_dev(both)
    ids, s = torch.arange(M, dtype=torch.int32, device="cuda") % 2, torch.ones(M, device="cuda")
    need = ctx.lin_adapters_workspace_bytes(qw, bank, M)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
    ok = dict(qw=qw, bank=bank, x=xy, y=xy.data_ptr() + 2 * K, M=M, row_adapter=ids,
              row_scale=s, ws=ws, ldx=K + N, ldy=K + N)
    sync()
    ctx.lin_adapters(**ok)
    ctx.synchronize()
    check(from_dev(xy)[:, K:], x, w, held, from_dev(ids), from_dev(s), 16)
    inside = ws[256:256 + 4 * M].view(torch.int32)
    for kw in ({"y": xy.data_ptr() + 2 * K - 16}, {"row_adapter": inside}, {"row_scale": inside},
               {"y": ws}, {"x": ws}, {"y": ids, "ldy": N}, {"y": s, "ldy": N},
               {"ldy": K + N + 4}, {"y": xy.data_ptr() + 2 * K + 8}):
        with pytest.raises(m.MingError, match="share|16-byte"):
            ctx.lin_adapters(**dict(ok, **kw))
    bank.close()
    qw.close()


def test_refusals(ctx):
    N, K, M = 64, 128, 10
    qw, _ = weight(ctx, 16000, N, K, 16)
    bank, _ = make_bank(ctx, 16100, N, K, (8,), max_rank=16)
    A, B = bf16(randn(16101, (8, K))), bf16(randn(16102, (N, 8)))
    for bad in ((-1, A, B, 1.0), (1, A, B, 1.0)):
        with pytest.raises(m.MingError):
            bank.set(*bad)
    with pytest.raises(m.MingError):
        bank.set(0, bf16(randn(1, (17, K))), bf16(randn(1, (N, 17))))
    for where in (0, 1):
        f = [A.copy(), B.copy()]
        for v in (0x7f80, 0xff80, 0x7fc0):
            f[where][-1, -1] = v
            with pytest.raises(m.MingError, match="finite") as e:
                bank.set(0, *f)
            assert e.value.code == m.ERR_RANGE
    with pytest.raises(m.MingError, match="finite"):
        bank.set(0, A, B, float("nan"))
    assert bank.rank(0) == 8                              # what was bound stays
    with pytest.raises(m.MingError):
        bank.clear(1)
    for shape in ((0, K, 1, 8), (N, 100, 1, 8), (60, K, 1, 8), (N, K, 0, 8), (N, K, 4097, 8),
                  (N, K, 1, 0), (N, K, 1, 513)):
        with pytest.raises(m.MingError):
            m.Adapters(ctx, *shape)
    x, y = to_dev(np.zeros((M, K), np.uint16)), to_dev(np.zeros((M, N), np.uint16))
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    need = ctx.lin_adapters_workspace_bytes(qw, bank, M)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    ok = dict(qw=qw, bank=bank, x=x, y=y, M=M, row_adapter=ids, row_scale=None, ws=ws)
    for kw in ({"ws": ws[:need - 256]}, {"ws": None}, {"row_adapter": None}, {"x": None},
               {"y": None}, {"M": -1}, {"ldx": 120}, {"ldy": 60}, {"y": x, "ldy": 64},
               {"ws": ws[4:]}):
        with pytest.raises(m.MingError):
            ctx.lin_adapters(**dict(ok, **kw))
    with pytest.raises(m.MingError, match="2\\^28"):
        ctx.lin_adapters(**dict(ok, M=1 << 28, row_adapter=1 << 50, y=1 << 56))
    assert ctx.lin_adapters_workspace_bytes(qw, bank, 2 ** 31 - 1) == 0
    ctx.lin_adapters(**dict(ok, M=0))
    wide, _ = make_bank(ctx, 16200, 72, K, (8,))
    with pytest.raises(m.MingError, match="shape"):
        ctx.lin_adapters(**dict(ok, bank=wide))
    other = m.Ctx(0)
    with pytest.raises(m.MingError, match="another"):
        other.lin_adapters(**ok)
    other.close()
    for h in (bank, wide, qw):
        h.close()


@pytest.mark.parametrize("bits,M,N,K", [(16, 200, 3840, 3840), (16, 700, 3840, 3840),
                                        (16, 300, 1024, 2048), (4, 200, 3840, 3840),
                                        (8, 700, 3840, 3840)])
def test_beside_and_apart_give_the_same_bits(ctx, bits, M, N, K):
    """A bank of two adapters runs its x.A beside the split's blocks, one of forty in a
    launch of its own (the profile says so): the same rows, the same bits."""
    qw, w = weight(ctx, 19000, N, K, bits)
    few, held = make_bank(ctx, 19100, N, K, (8, 24), cap=40, max_rank=64)
    many, _ = make_bank(ctx, 19100, N, K, (8, 24) + (64,) * 38)
    x = bf16(randn(19300 + M, (M, K)))
    ids, s = np.arange(M) % 3 - 1, np.linspace(-1, 1, M).astype(np.float32)
    got = []
    for bank, apart in ((few, 0), (many, 1)):
        ctx.profile_collect()
        ctx.set_profiling(True)
        try:
            got.append(call(ctx, qw, bank, x, ids, s))
            assert ctx.profile_collect().get("row_adapters", {"launches": 0})["launches"] == apart
        finally:
            ctx.set_profiling(False)
    some = np.unique(np.concatenate([np.arange(0, M, 9), [M - 1]]))
    check(got[0][some], x[some], w, held, ids[some], s[some], bits)
    assert np.array_equal(got[1], got[0])
    for h in (few, many, qw):
        h.close()


@pytest.mark.parametrize("bits", [4, 16])
def test_an_empty_batch(ctx, bits):
    """No rows: nothing runs, and empty tensors, which have no address, will do. What is
    no call of this bank and weight is refused all the same."""
    N, K = 64, 128
    qw, _ = weight(ctx, 19400, N, K, bits)
    bank, _ = make_bank(ctx, 19500, N, K, (8,))
    none = torch.empty(0, dtype=torch.int16, device="cuda")
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    assert none.data_ptr() == 0 and ctx.lin_adapters_workspace_bytes(qw, bank, 0) == 0
    ctx.lin_adapters(qw, bank, none, none, 0, ids, None, none)
    ctx.lin_adapters(qw, bank, None, None, 0, None, None, None)
    ctx.synchronize()
    wide, _ = make_bank(ctx, 19600, 72, K, (8,))
    with pytest.raises(m.MingError, match="shape"):
        ctx.lin_adapters(qw, wide, None, None, 0, None, None, None)
    with pytest.raises(m.MingError):
        ctx.lin_adapters(qw, bank, None, None, -1, None, None, None)
    for h in (bank, wide, qw):
        h.close()


@pytest.mark.parametrize("M", [2 ** 28 - 31, 2 ** 28 - 1, 2 ** 31 - 1])
def test_more_rows_than_a_launch_holds(ctx, M):
    N, K = 64, 128
    qw, _ = weight(ctx, 19700, N, K, 16)
    bank, _ = make_bank(ctx, 19800, N, K, (8,))
    far = 1 << 56
    with pytest.raises(m.MingError, match="2\\^28") as e:
        ctx.lin_adapters(qw, bank, far, far << 1, M, far << 2, None,
                         torch.empty(4096, dtype=torch.uint8, device="cuda"))
    assert e.value.code == 2 and ctx.lin_adapters_workspace_bytes(qw, bank, M) == 0
    bank.close()
    qw.close()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("M", [6, 40, 300])
def test_inputs_past_32_bits(ctx, bits, M):
    """Rows of x that span more than 4 GiB. A dense projection takes another launch for
    them and says what it needs."""
    N, K, ld = 1032, 1024, 1 << 29 if M == 6 else 1 << 26 if M == 40 else 1 << 23
    qw, w = weight(ctx, 20700, N, K, bits)
    bank, held = make_bank(ctx, 20800, N, K, RANKS)
    x = bf16(randn(20900, (M, K)))
    ids, s = requests(M, 8, len(RANKS))
    far = torch.empty((M, ld), dtype=torch.int16, device="cuda")
    far[:, :K] = to_dev(x)
    y = to_dev(np.zeros((M, N), np.uint16))
    idd, sd = to_dev(ids.astype(np.int32)), to_dev(s)
    need = ctx.lin_adapters_workspace_bytes(qw, bank, M)
    sync()
    for _ in range(2):
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        try:
            ctx.lin_adapters(qw, bank, far, y, M, idd, sd, ws, ldx=ld)
            break
        except m.MingError as e:
            assert bits == 16 and e.code == 2
            need = int(re.search(r"needs (\d+) bytes", str(e)).group(1))
    ctx.synchronize()
    check(from_dev(y), x, w, held, ids, s, bits)
    del far
    torch.cuda.empty_cache()
    bank.close()
    qw.close()
