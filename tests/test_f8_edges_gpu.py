"""Edges of the operators in 8-bit floating point that their documentation allows."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import ming_dit_amd as m
import rows_ref
from helpers import bf16, f32, from_dev, randn, sync, to_dev
from test_f8_gpu import S8, S16, Weights, call, check, check_norm, norm, plan  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- a part of a plan ------------------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts,e0", [([5, 9, 20, 3], 1), ([70, 0, 1, 130], 2), ([3, 0, 300, 40], 1)])
def test_a_part_of_a_plan(ctx, plan, gated, counts, e0):  # noqa: F811
    """The experts from e0 on with their part of the plan's offsets: their groups' rows have
    the whole plan's results, the rows of the groups before stay as they were."""
    E, N, K = len(counts), 272, 208
    W = Weights(ctx, 8000, E - e0, N, K, gated)
    offsets, order, src = rows_ref.plan_of(counts, n=sum(counts) + 11, fan=2, seed=E, x_rows=50)
    n, first, held = order.size, int(offsets[e0]), int(offsets[-1])
    x, xs = ref.make_rows(8001, 50, K)
    xd, sd, od = to_dev(x), to_dev(xs), to_dev(order)
    fd = to_dev(offsets)
    for p in (-1,) + ref.GROUPED_PLANS:
        print(f"case f8 part of a plan {p} gated={gated} {counts}", flush=True)
        plan(p)
        ws = torch.full((16 + W.w.workspace_bytes(n),), 0x41, dtype=torch.uint8, device="cuda")
        out = to_dev(np.full((n, N), S8 if gated else S16, np.uint8 if gated else np.uint16))
        hs = to_dev(np.full((ref.blocks(N), n), S16, np.uint16))
        sync()
        if gated:
            ctx.f8_experts_swiglu(W.w, xd, sd, 50, od, fd[e0:], n, out, hs, fan=2, ws=ws)
        else:
            ctx.f8_experts_lin(W.w, xd, sd, 50, od, fd[e0:], n, out, fan=2, ws=ws)
        ctx.synchronize()
        o, s = from_dev(out), from_dev(hs)
        away = [r for r in range(n) if r < first or r >= held]
        assert np.all(o[away] == (S8 if gated else S16))
        if gated:
            assert np.all(s[:, away] == S16)
            got = (o[first:held], np.ascontiguousarray(s[:, first:held]))
        else:
            got = f32(o[first:held]).astype(np.float64)
        check(got, W, x, xs, offsets[e0:] - first, src[first:])
    W.w.close()


# ---- norms -----------------------------------------------------------------------------
@pytest.mark.parametrize("add", [False, True])
def test_norm_of_a_mean_square_past_f32(ctx, add):
    """A row whose mean square is inf or NaN in f32 is NaN in y as in its codes, and the
    rows beside it stay as they are."""
    D = 400
    x = randn(8100, (7, D))
    w = bf16(1.0 + randn(8, (D,), 0.3))
    w[128:256] = 0                              # (its zeros too)
    sub = bf16(randn(8101, (7, D))) if add else None
    keep, odd = [0, 2, 4, 6], [1, 3, 5]
    a = norm(ctx, bf16(x), w, sub, y=True)
    x[1] = 1e20
    x[3, 7] = np.inf
    x[5, 399] = np.nan
    h, y, codes, scales = norm(ctx, bf16(x), w, sub, y=True)
    for p, q in zip((a[0], a[1], a[2], a[3].T), (h, y, codes, scales.T)):
        if p is not None:
            assert np.array_equal(p[keep], q[keep])
    assert np.all((codes[odd] & 0x7f) == ref.NAN) and np.all(scales.T[odd] == 0x7fc0)
    assert np.all(np.isnan(f32(y[odd])))


def test_norm_of_far_gains(ctx):
    """Gains so large or small that gain * rsqrt(mean square) leaves f32's range where the
    result does not."""
    D = 272
    x = randn(8110, (5, D))
    x[0] = 0.0
    x[1] *= 1e-10
    x[2] *= 1e18
    w = 1.0 + randn(8, (D,), 0.3)
    for size in (1e33, 1e-25):
        b, g = bf16(x), bf16((w * size).astype(np.float32))
        _, y, codes, scales = norm(ctx, b, g, y=True, eps=1e-12)
        check_norm(b, g, None, 1e-12, None, y, codes, scales)


# ---- gated results on the border of two codes --------------------------------------------
def border_case():
    """(codes, scales, x, v): a gated weight of 64 columns whose results v are exact in f32
    for the row x: 256 times whole numbers of 14 bits, each of four nibbles that x's columns
    0, 8, 16 and 24 take up. Each block of 128 columns has a scale of another 8-bit
    significand, and in it the borders of two codes with their neighbours."""
    N, K = 128 * 128, 64
    u = np.zeros(N, np.int64)
    for b in range(128):
        s = 128 + b
        near = [sign * (q * s + d) for q in range(17, 32, 2) for sign in (1, -1) for d in (-1, 0, 1)]
        u[128 * b:128 * b + 128] = np.resize(near, 128)
        u[128 * b + 127] = 56 * s               # 448 times the scale s / 8
    x = np.zeros((1, K))
    codes = np.zeros((1, 2 * N, K))
    codes[0, :N, 32], x[0, 32] = 16.0, 16.0     # gates of 256, whose sigmoid is 1
    for k, at, w in ((0, 64.0, 2.0 ** 6), (8, 16.0, 16.0), (16, 1.0, 16.0), (24, 1.0, 1.0)):
        x[0, k] = at
        nibble = (np.abs(u) >> int(np.log2(at * w))) & 15
        codes[0, N:, k] = np.sign(u) * nibble * w
    scales = np.ones((1, 256, 1), np.float32)
    v = 256.0 * u[None].astype(np.float64)
    return ref.encode(codes), scales, ref.encode(x), v


@pytest.mark.parametrize("M", [1, 70, 300])
def test_gated_results_between_two_codes(ctx, plan, M):  # noqa: F811
    """Codes are the nearest of v over the scale, ties to even, as the row quantizer's are."""
    codes, scales, x, v = border_case()
    N, K = codes.shape[1] // 2, codes.shape[2]
    want, s = ref.quantize(v)
    W = Weights.__new__(Weights)
    W.codes, W.scales, W.E, W.N, W.K, W.gated = codes, scales, 1, N, K, True
    W.w = m.F8(ctx, codes, scales, N, gated=True)
    x, xs = np.repeat(x, M, 0), np.full((1, M), 0x3f80, np.uint16)
    offsets = np.array([0, M], np.int32)
    for p in ref.PLANS + tuple(-q for q in ref.GROUPED_PLANS):
        print(f"case f8 borders plan {p} M={M}", flush=True)
        plan(abs(p))
        got, gs = call(ctx, W, x, xs) if p > 0 else call(ctx, W, x, xs, offsets, None, M)
        assert np.array_equal(gs, np.repeat(s, M, 1)), p
        assert np.array_equal(got, np.repeat(want, M, 0)), p
    W.w.close()


# ---- scales of inf -----------------------------------------------------------------------
@pytest.mark.parametrize("K", [128, 272, 640, 1168])
def test_a_scale_of_inf(ctx, plan, K):  # noqa: F811
    """A row whose last block has a scale of inf has infinities, of the block's sum's sign,
    from every kernel; the other rows have their own results."""
    N, M = 144, 70
    W = Weights(ctx, 8200, 1, N, K, False)
    W.w.close()
    W.codes[..., 128 * ((K - 1) // 128):] = 0x38          # ones
    W.w = m.F8(ctx, W.codes, W.scales, N)
    x, xs = ref.make_rows(8201, M, K)
    x[[3, 69], 128 * ((K - 1) // 128):] = 0x30
    x[69, 128 * ((K - 1) // 128):] = 0xb0
    for p in ref.PLANS + ref.DUO:
        print(f"case f8 inf plan {p} K={K}", flush=True)
        plan(p)
        big = xs.copy()
        big[-1, [3, 69]] = 0x7f80
        got = call(ctx, W, x, big)
        assert np.all(got[3] == np.inf) and np.all(got[69] == -np.inf), p
        keep = [r for r in range(M) if r not in (3, 69)]
        assert np.array_equal(got[keep], call(ctx, W, x, xs)[keep])
    W.w.close()


# ---- workspaces --------------------------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("E,N,K", [(1, 272, 400), (64, 48, 144), (1, 16, 131088)])
def test_workspaces_of_any_count(ctx, gated, E, N, K):
    """Counts beyond the 2^28 rows that a call takes name what those need."""
    W = Weights(ctx, 8300, E, N, K, gated)
    most = W.w.workspace_bytes(1 << 28)
    assert W.w.workspace_bytes((1 << 28) - 1) <= most
    for n in ((1 << 28) + 1, 2 ** 31 - 8, 2 ** 31 - 1):
        assert W.w.workspace_bytes(n) == most
    W.w.close()
