"""Calls of the operators in 8-bit floating point as programs make them: a workspace for
the largest batch, addresses past 32 bits, outputs that pass the caches, a K beyond the
tiles', two contexts at once, captured plans that change, and index arrays that are no
plan."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import ming_dit_amd as m
import rows_ref
from helpers import f32, from_dev, sync, to_dev
from test_f8_gpu import S8, S16, Weights, call, check, plan  # noqa: F401

pytestmark = pytest.mark.gpu


def codes_like(rows, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(0, 256, (rows, K), generator=g, device="cuda", dtype=torch.uint8)
    x[(x & 0x7f) == ref.NAN] = 0x30
    s = torch.rand((ref.blocks(K), rows), generator=g, device="cuda") * 0.01 + 0.001
    return x, s.bfloat16().view(torch.int16)


# ---- a workspace of the most rows ---------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("E,N,K", [(1, 400, 272), (1, 528, 2576), (6, 144, 208), (20, 48, 1040)])
def test_a_workspace_serves_fewer_rows(ctx, gated, E, N, K):
    W = Weights(ctx, 7000 + N, E, N, K, gated)
    sizes = [W.w.workspace_bytes(n) for n in range(0, 1500)]
    assert sizes[0] == 0 and all(a <= b for a, b in zip(sizes, sizes[1:]))
    most = 5000
    ws = torch.full((max(16, W.w.workspace_bytes(most)),), 255, dtype=torch.uint8, device="cuda")
    assert W.w.workspace_bytes(most) >= sizes[-1]
    for n in (1, 2, 16, 17, 63, 65, 150, 203, 300, 600, 1100, 2400, 4097, most):
        x, xs = codes_like(n, K, n)
        counts = np.full(E, n // E)
        counts[0] += n - counts.sum()
        off = to_dev(rows_ref.plan_of(counts)[0])
        out = torch.zeros((n, N), dtype=torch.uint8 if gated else torch.int16, device="cuda")
        hs = torch.zeros((ref.blocks(N), n), dtype=torch.int16, device="cuda")
        sync()
        if gated and E == 1:
            ctx.f8_swiglu(W.w, x, xs, out, hs, n, ws=ws)
        elif gated:
            ctx.f8_experts_swiglu(W.w, x, xs, n, None, off, n, out, hs, ws=ws)
        elif E == 1:
            ctx.f8_lin(W.w, x, xs, out, n, ws=ws)
        else:
            ctx.f8_experts_lin(W.w, x, xs, n, None, off, n, out, ws=ws)
        ctx.synchronize()
        assert out.any()
    W.w.close()


# ---- a stack of one, and K beyond the tiles' ------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_a_stack_of_one(ctx, gated, n):
    """The groups' calls take a single projection, and give what its own calls give."""
    W = Weights(ctx, 7100, 1, 272, 400, gated)
    x, xs = ref.make_rows(7101 + n, n, 400)
    offsets, order, src = rows_ref.plan_of([n], n=n + 5, fan=1, seed=1, x_rows=n)
    got = call(ctx, W, x, xs, offsets, order, order.size)
    check(got, W, x, xs, offsets, src)
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("K", [131072, 131088])
def test_more_blocks_than_a_tile_holds(ctx, gated, K):
    W = Weights(ctx, 7200, 2, 16, K, gated, on_device=True)
    one = Weights(ctx, 7200, 1, 16, K, gated)
    for n in (1, 19):
        x, xs = ref.make_rows(7201 + n, n, K)
        check(call(ctx, one, x, xs), one, x, xs)
        offsets, order, src = rows_ref.plan_of([n // 3, n - n // 3], n=n, fan=1, seed=2, x_rows=n)
        check(call(ctx, W, x, xs, offsets, order, n), W, x, xs, offsets, src)
    W.w.close()
    one.w.close()


# ---- far addresses ----------------------------------------------------------------------
def spaced(t, ld):
    """t's rows ld elements apart in memory of their own."""
    flat = torch.empty((t.shape[0] - 1) * ld + t.shape[1], dtype=t.dtype, device="cuda")
    v = flat.as_strided(t.shape, (ld, 1))
    v.copy_(t)
    return flat, v


@pytest.mark.parametrize("gated", [False, True])
def test_products_far_apart(ctx, plan, gated):  # noqa: F811
    """Rows of x, scales and outputs whose offsets pass 32 bits give the bits of those
    side by side, whichever kernel takes them."""
    N, K, n = 272, 272, 1100
    W = Weights(ctx, 7300, 1, N, K, gated)
    x, xs = codes_like(n, K, 7301)
    ldx, lds, ldy = (1 << 22) - 16, (1 << 30) - 1, 1 << 22
    xf, _ = spaced(x, ldx)
    sf, _ = spaced(xs, lds)
    out = torch.zeros((n, N), dtype=torch.uint8 if gated else torch.int16, device="cuda")
    hs = torch.zeros((ref.blocks(N), n), dtype=torch.int16, device="cuda")
    of, ov = spaced(out, ldy)
    hf, hv = spaced(hs, lds)
    for p in (-1,) + (ref.PLANS if gated else ref.PLANS + (100, 200)):
        print(f"case f8 far plan {p} gated={gated}", flush=True)
        plan(p)
        ws = torch.zeros(16 + W.w.workspace_bytes(n), dtype=torch.uint8, device="cuda")
        for t in (out, hs, ov, hv):
            t.zero_()
        sync()
        if gated:
            ctx.f8_swiglu(W.w, x, xs, out, hs, n, ws=ws)
            ctx.f8_swiglu(W.w, xf, sf, of, hf, n, ws=ws, ldx=ldx, ldxs=lds, ldh=ldy, ldhs=lds)
        else:
            ctx.f8_lin(W.w, x, xs, out, n, ws=ws)
            ctx.f8_lin(W.w, xf, sf, of, n, ws=ws, ldx=ldx, ldxs=lds, ldy=ldy)
        ctx.synchronize()
        assert torch.equal(out, ov) and torch.equal(hs, hv)
        assert out.any()
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
def test_experts_far_apart(ctx, plan, gated):  # noqa: F811
    N, K, n, x_rows = 144, 272, 1300, 512
    counts = [300, 0, 700, 1, 299]
    W = Weights(ctx, 7350, 5, N, K, gated)
    x, xs = codes_like(x_rows, K, 7351)
    offsets, order, _ = rows_ref.plan_of(counts, n=n, fan=3, seed=3, x_rows=x_rows)
    od, fd = to_dev(order), to_dev(offsets)
    ldx, lds, ldy = ((1 << 31) - 1) // x_rows // 16 * 16, (1 << 30) - 1, 1 << 22
    xf, _ = spaced(x, ldx)
    sf, _ = spaced(xs, lds)
    out = torch.zeros((n, N), dtype=torch.uint8 if gated else torch.int16, device="cuda")
    hs = torch.zeros((ref.blocks(N), n), dtype=torch.int16, device="cuda")
    of, ov = spaced(out, ldy)
    hf, hv = spaced(hs, lds)
    for p in (-1,) + ref.GROUPED_PLANS:
        print(f"case f8 far groups plan {p} gated={gated}", flush=True)
        plan(p)
        ws = torch.zeros(16 + W.w.workspace_bytes(n), dtype=torch.uint8, device="cuda")
        for t in (out, hs, ov, hv):
            t.zero_()
        sync()
        if gated:
            ctx.f8_experts_swiglu(W.w, x, xs, x_rows, od, fd, n, out, hs, fan=3, ws=ws)
            ctx.f8_experts_swiglu(W.w, xf, sf, x_rows, od, fd, n, of, hf, fan=3, ws=ws, ldx=ldx,
                                  ldxs=lds, ldh=ldy, ldhs=lds)
        else:
            ctx.f8_experts_lin(W.w, x, xs, x_rows, od, fd, n, out, fan=3, ws=ws)
            ctx.f8_experts_lin(W.w, xf, sf, x_rows, od, fd, n, of, fan=3, ws=ws, ldx=ldx, ldxs=lds,
                               ldy=ldy)
        ctx.synchronize()
        assert torch.equal(out, ov) and torch.equal(hs, hv)
        assert out.any()
    W.w.close()


def test_quantizer_and_norm_far_apart(ctx):
    rows, D, ld, lds = 5, 400, (1 << 30) - 16, (1 << 30) - 1
    g = torch.Generator(device="cuda").manual_seed(7)
    x, sub = (torch.randn((rows, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.randn(D, generator=g, device="cuda").bfloat16()
    xf, _ = spaced(x, ld)
    y, h = (torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = torch.zeros((rows, D), dtype=torch.uint8, device="cuda")
    s = torch.zeros((ref.blocks(D), rows), dtype=torch.int16, device="cuda")
    (cf, cv), (sf, sv), (hf, hv), (yf, yv), (uf, _) = (
        spaced(c, ld), spaced(s, lds), spaced(h, ld), spaced(y, ld), spaced(sub, ld))
    sync()
    ctx.f8_quantize(x, rows, D, c, s)
    ctx.f8_quantize(xf, rows, D, cf, sf, ldx=ld, ldc=ld, lds=lds)
    ctx.synchronize()
    assert torch.equal(c, cv) and torch.equal(s, sv) and c.any()
    sync()
    ctx.f8_rmsnorm(x, w, rows, D, c, s, sub=sub, h=h, y=y)
    ctx.f8_rmsnorm(xf, w, rows, D, cf, sf, sub=uf, h=hf, y=yf, ldx=ld, ldsub=ld, ldh=ld, ldy=ld,
                   ldc=ld, lds=lds)
    ctx.synchronize()
    for a, b in ((c, cv), (s, sv), (h, hv), (y, yv)):
        assert torch.equal(a, b)


# ---- outputs that pass the caches ---------------------------------------------------------
def test_large_outputs(ctx, plan):  # noqa: F811
    """What is stored past the caches (more than 24 MB) has the bits of two halves that are
    not, and its first rows are the definition's."""
    n, N, K = 4300, 3200, 144
    W, half = Weights(ctx, 7400, 1, N, K, False), 2304      # a boundary of every tile
    hx, hxs = ref.make_rows(7401, n, K)
    x, xs = to_dev(hx), to_dev(hxs)
    y, z = (torch.zeros((n, N), dtype=torch.int16, device="cuda") for _ in range(2))
    for p in (1, 2, 3, 4, 5):
        plan(p)
        y.zero_()
        sync()
        ctx.f8_lin(W.w, x, xs, y, n)
        ctx.f8_lin(W.w, x, xs, z, half, ldxs=n)
        ctx.f8_lin(W.w, x[half:], xs.data_ptr() + 2 * half, z[half:], n - half, ldxs=n)
        ctx.synchronize()
        assert torch.equal(y, z)
    rows = 64
    check(f32(from_dev(y[:rows])).astype(np.float64), W, hx[:rows], np.ascontiguousarray(hxs[:, :rows]))
    W.w.close()
    G = Weights(ctx, 7410, 2, 6400, K, True)
    h, h2 = (torch.zeros((n, 6400), dtype=torch.uint8, device="cuda") for _ in range(2))
    hs, hs2 = (torch.zeros((50, n), dtype=torch.int16, device="cuda") for _ in range(2))
    off = to_dev(np.array([0, 1800, n], np.int32))
    lo, hi = to_dev(np.array([0, 1800, 1800], np.int32)), to_dev(np.array([0, 0, n - 1800], np.int32))
    plan(4)
    sync()
    ctx.f8_experts_swiglu(G.w, x, xs, n, None, off, n, h, hs)
    ctx.f8_experts_swiglu(G.w, x, xs, 1800, None, lo, 1800, h2, hs2, ldxs=n, ldhs=n)
    ctx.f8_experts_swiglu(G.w, x[1800:], xs.data_ptr() + 3600, n - 1800, None, hi, n - 1800, h2[1800:],
                          hs2.data_ptr() + 3600, ldxs=n, ldhs=n)
    ctx.synchronize()
    assert torch.equal(h, h2) and torch.equal(hs, hs2)
    G.w.close()
    D, rows = 4096, 6400
    v = torch.randn((rows, D), device="cuda").bfloat16()
    c, c2 = (torch.zeros((rows, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    s, s2 = (torch.zeros((D // 128, rows), dtype=torch.int16, device="cuda") for _ in range(2))
    sync()
    ctx.f8_quantize(v, rows, D, c, s)
    for a in (0, 3200):
        ctx.f8_quantize(v[a:], 3200, D, c2[a:], s2.data_ptr() + 2 * a, lds=rows)
    ctx.synchronize()
    assert torch.equal(c, c2) and torch.equal(s, s2)


# ---- two at once, and captured plans that change --------------------------------------------
def test_two_contexts_at_once():
    """Contexts on streams of their own, each with its weights and workspace, calls in
    flight together: the bits of calls by themselves. The sources of weights are
    overwritten as soon as their creation returns."""
    lanes = []
    for i in range(2):
        st = torch.cuda.Stream()
        c = m.Ctx(0, st.cuda_stream)
        GU = Weights(c, 7500 + i, 1, 528, 400, True)
        codes, scales = ref.make_weight(7510 + i, 1, 400, 528, False)
        cd, sd = to_dev(codes), to_dev(scales)
        sync()
        DN = m.F8(c, cd, sd, 400, on_device=True)
        cd.fill_(ref.NAN)
        sd.fill_(float("nan"))
        sync()
        n = 203 - 60 * i
        x, xs = codes_like(n, 400, 7520 + i)
        h = torch.zeros((n, 528), dtype=torch.uint8, device="cuda")
        hs = torch.zeros((ref.blocks(528), n), dtype=torch.int16, device="cuda")
        y = torch.zeros((n, 400), dtype=torch.int16, device="cuda")
        need = []
        for p, w in ((24, GU.w), (300, DN)):     # both go by the workspace
            ref.set_plan(c, p)
            need.append(w.workspace_bytes(n))
            assert need[-1] > 0
        ws = torch.zeros(max(need), dtype=torch.uint8, device="cuda")
        lanes.append((c, GU.w, DN, n, x, xs, h, hs, y, ws))
    sync()

    def step(c, gu, dn, n, x, xs, h, hs, y, ws):
        ref.set_plan(c, 24)
        c.f8_swiglu(gu, x, xs, h, hs, n, ws=ws)
        ref.set_plan(c, 300)
        c.f8_lin(dn, h, hs, y, n, ws=ws)

    alone = []
    for v in lanes:
        step(*v)
        v[0].synchronize()
        alone.append([t.clone() for t in v[6:9]])
        assert v[8].any()
    for it in range(20):
        for v in lanes:
            step(*v)
    for v, want in zip(lanes, alone):
        v[0].synchronize()
        for t, w in zip(v[6:9], want):
            assert torch.equal(t, w)
    for v in lanes:
        v[1].close()
        v[2].close()
        v[0].close()


@pytest.mark.parametrize("p", [-1, 11, 4])
def test_captured_groups_that_change(p):
    """A captured mixture reads its plan anew at each replay: groups that grow, vanish and
    end early, with eager calls between the replays."""
    s = torch.cuda.Stream()
    c = m.Ctx(0, s.cuda_stream)
    ref.set_plan(c, p)
    E, H, F, T, n = 4, 272, 144, 90, 400
    GU, DN = Weights(c, 7600, E, F, H, True), Weights(c, 7601, E, H, F, False)
    x, xs = ref.make_rows(7602, T, H)
    xd, sd = to_dev(x), to_dev(xs)
    off, order = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (E + 1, n))
    h, hs = to_dev(np.zeros((n, F), np.uint8)), to_dev(np.zeros((ref.blocks(F), n), np.uint16))
    y = to_dev(np.zeros((n, H), np.uint16))
    ws = torch.full((16 + max(w.w.workspace_bytes(n) for w in (GU, DN)),), 255, dtype=torch.uint8,
                    device="cuda")

    def step():
        c.f8_experts_swiglu(GU.w, xd, sd, T, order, off, n, h, hs, fan=5, ws=ws)
        c.f8_experts_lin(DN.w, h, hs, n, None, off, n, y, ws=ws)

    sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        step()
    for i, counts in enumerate(([100, 100, 100, 100], [0, 399, 0, 1], [0, 0, 0, 0], [7, 0, 300, 2])):
        held = sum(counts)
        o, od, src = rows_ref.plan_of(counts, n=n, fan=5, seed=i, x_rows=T)
        off.copy_(to_dev(o))
        order.copy_(to_dev(od))
        got = []
        for run in (g.replay, step):
            h.fill_(S8)
            hs.fill_(S16)
            y.fill_(S16)
            sync()
            run()
            sync()
            c.synchronize()
            got.append([from_dev(t).copy() for t in (h, hs, y)])
        for a, b in zip(*got):
            assert np.array_equal(a, b)
        gh, ghs, gy = got[0]
        assert np.all(gh[held:] == S8) and np.all(ghs[:, held:] == S16) and np.all(gy[held:] == S16)
        check((gh[:held], ghs[:, :held]), GU, x, xs, o, src)
        check(f32(gy[:held]).astype(np.float64), DN, gh[:held], np.ascontiguousarray(ghs[:, :held]), o,
              np.arange(held))
    del g
    GU.w.close()
    DN.w.close()
    c.close()


# ---- index arrays that are no plan ---------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
def test_no_plan_stays_in_bounds(ctx, plan, gated):  # noqa: F811
    """Offsets that fall, repeat, are negative or pass n, and an order of any numbers, name
    wrong rows but none outside: what lies beside the outputs stays."""
    N, K, n, E = 144, 272, 200, 4
    W = Weights(ctx, 7700, E, N, K, gated)
    x, xs = codes_like(30, K, 7701)
    order = to_dev(np.array([(-1) ** i * (i * 7919 % 2 ** 31) for i in range(n)], np.int32))
    for p in (-1,) + ref.GROUPED_PLANS:
        for offsets in ([0, 150, 20, 190, 60], [0, -5, 300, 2 ** 31 - 1, -2 ** 31], [200, 150, 100, 50, 0],
                        [50, 50, 200, 200, 2 ** 30]):
            print(f"case f8 no plan {p} {offsets}", flush=True)
            plan(p)
            fd = to_dev(np.array(offsets, np.int64).astype(np.int32))
            ws = torch.zeros(16 + W.w.workspace_bytes(n), dtype=torch.uint8, device="cuda")
            out = torch.full((n + 4, N + 16), 77, dtype=torch.uint8 if gated else torch.int16,
                             device="cuda")
            hs = torch.full((ref.blocks(N) + 2, n + 3), 77, dtype=torch.int16, device="cuda")
            at, sat = out[2:], hs[1:]
            sync()
            if gated:
                ctx.f8_experts_swiglu(W.w, x, xs, 30, order, fd, n, at, sat, fan=2, ws=ws, ldh=N + 16,
                                      ldhs=n + 3)
            else:
                ctx.f8_experts_lin(W.w, x, xs, 30, order, fd, n, at, fan=2, ws=ws, ldy=N + 16)
            ctx.synchronize()
            assert torch.all(out[:2] == 77) and torch.all(out[n + 2:] == 77)
            assert torch.all(out[:, N:] == 77)
            assert torch.all(hs[0] == 77) and torch.all(hs[-1] == 77) and torch.all(hs[:, n:] == 77)
    W.w.close()


def test_profiler_and_counters(ctx):
    n, N, K = 40, 144, 272
    L, G = Weights(ctx, 7800, 1, N, K, False), Weights(ctx, 7801, 1, N, K, True)
    x = torch.randn((n, K), device="cuda").bfloat16()
    w = torch.ones(K, device="cuda").bfloat16()
    c = torch.zeros((n, K), dtype=torch.uint8, device="cuda")
    s = torch.zeros((ref.blocks(K), n), dtype=torch.int16, device="cuda")
    y = torch.zeros((n, N), dtype=torch.int16, device="cuda")
    h = torch.zeros((n, N), dtype=torch.uint8, device="cuda")
    hs = torch.zeros((ref.blocks(N), n), dtype=torch.int16, device="cuda")
    ws = torch.zeros(16 + G.w.workspace_bytes(n), dtype=torch.uint8, device="cuda")
    ctx.profile_collect()
    ctx.set_profiling(True)
    before = ctx.engagement()
    sync()
    ctx.f8_quantize(x, n, K, c, s)
    ctx.f8_rmsnorm(x, w, n, K, c, s)
    ctx.f8_lin(L.w, c, s, y, n, ws=ws)
    ctx.f8_swiglu(G.w, c, s, h, hs, n, ws=ws)
    prof = ctx.profile_collect()
    ctx.set_profiling(False)
    after = ctx.engagement()
    for b, flops, size in (("f8_quantize", 0, 3 * n * K), ("f8_rmsnorm", 0, 3 * n * K),
                           ("f8_lin", 2 * n * N * K, N * K + n * K + 2 * n * N),
                           ("f8_swiglu", 4 * n * N * K, 2 * N * K + n * K + n * N)):
        assert prof[b]["launches"] == 1 and prof[b]["ms"] > 0, b
        assert prof[b]["flops"] == flops and prof[b]["bytes"] == size, b
    for k, v in (("gemm_q8", 2), ("rmsnorm", 1), ("elementwise", 1)):
        assert after[k] - before[k] == v, k
    L.w.close()
    G.w.close()
