"""The 8-bit products against the matrix instruction's own sums: gated codes and scales and
bf16 results as close as f32 leaves them, from every kernel; outliers, stacks of up to a
thousand experts, a real width, and rows that do not feel each other."""
import numpy as np
import pytest

import f8_model as model
import f8_ref as ref
import ming_dit_amd as m
import rows_ref
from test_f8_gpu import Weights, call, check, plan  # noqa: F401

pytestmark = pytest.mark.gpu


def weights(ctx, codes, scales, gated):
    W = Weights.__new__(Weights)
    W.codes, W.scales, W.gated = codes, scales, gated
    W.E, W.N, W.K = codes.shape[0], codes.shape[1] // (2 if gated else 1), codes.shape[2]
    W.w = m.F8(ctx, codes, scales, W.N, gated=gated)
    return W


def any_codes(rng, shape):
    c = rng.integers(0, 256, shape, dtype=np.uint8)
    c[(c & 0x7f) == ref.NAN] = 0x30
    return c


def check_close(got, v, gated):
    if gated:
        model.check_gated(*got, v)
    else:
        model.check_plain(got, v)


# ---- close to the instruction's sums -----------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K", [(272, 272), (400, 1152)])
@pytest.mark.parametrize("M", [9, 70, 260])
def test_products_are_close(ctx, plan, gated, N, K, M):  # noqa: F811
    W = Weights(ctx, 9000 + N, 1, N, K, gated)
    x, xs = ref.make_rows(9001 + M, M, K)
    v = model.results(x, xs, W.codes[0], W.scales[0], gated)
    for p in ref.PLANS if gated else ref.PLANS + ref.DUO:
        print(f"case f8 close plan {p} gated={gated} N={N} K={K} M={M}", flush=True)
        plan(p)
        check_close(call(ctx, W, x, xs), v, gated)
    W.w.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts", [[1] * 9, [5, 0, 17, 40, 2], [130, 0, 70, 300, 257]])
def test_experts_are_close(ctx, plan, gated, counts):  # noqa: F811
    E, N, K = len(counts), 272, 400
    W = Weights(ctx, 9100, E, N, K, gated)
    offsets, order, src = rows_ref.plan_of(counts, n=sum(counts) + 11, fan=2, seed=E, x_rows=90)
    x, xs = ref.make_rows(9101, 90, K)
    v = np.concatenate([model.results(x[src[a:b]], np.ascontiguousarray(xs[:, src[a:b]]), W.codes[e],
                                      W.scales[e], gated)
                        for e, (a, b) in enumerate(zip(offsets, offsets[1:])) if b > a])
    for p in ref.GROUPED_PLANS:
        print(f"case f8 close groups plan {p} gated={gated} {counts}", flush=True)
        plan(p)
        check_close(call(ctx, W, x, xs, offsets, order, order.size, fan=2), v, gated)
    W.w.close()


# ---- codes that are not Gaussian ---------------------------------------------------------
@pytest.mark.parametrize("M", [3, 70, 300])
@pytest.mark.parametrize("what", ["outlier", "cancelling", "subnormal"])
def test_codes_of_unequal_size(ctx, plan, what, M):  # noqa: F811
    """A product of 448 * 448 among small ones, two that cancel, and codes below the
    smallest normal: the sums are the instruction's, within what the documentation says of
    exact ones."""
    N, K = 144, 272
    rng = np.random.default_rng(len(what))
    x = rng.integers(-8, 9, (M, K)) / 8.0
    w = rng.integers(-8, 9, (N, K)) / 8.0
    if what == "subnormal":
        x, w = x * 2.0 ** -6, w * 2.0 ** -6
    else:
        x[:, 5::32] = 448.0
        w[:, 5::32] = 448.0
        if what == "cancelling":
            x[:, 6::32] = -448.0
            w[:, 6::32] = 448.0
    x, codes = ref.encode(x), ref.encode(w)[None]
    scales = np.ones((1, ref.blocks(N), ref.blocks(K)), np.float32)
    xs = np.full((ref.blocks(K), M), 0x3f80, np.uint16)
    W = weights(ctx, codes, scales, False)
    v = model.results(x, xs, codes[0], scales[0])
    exact = ref.decode(x) @ ref.decode(codes[0]).T
    # f32: a sum of 8 is cut at 2^-24 of the block's largest, 16 a block
    step = np.abs(ref.decode(x)).max() * np.abs(ref.decode(codes[0])).max() * 8 * 2.0 ** -23
    f32_off = ref.blocks(K) * 18 * step
    # documented: of 8 products seven lose up to 2^-13 of the largest, a subnormal code
    # counting as 2^-6
    least = np.maximum(np.abs(ref.decode(x)), 2.0 ** -6), np.maximum(np.abs(ref.decode(codes[0])), 2.0 ** -6)
    cut = 7 * 2.0 ** -13 * ref.most8(least[0]) @ ref.most8(least[1]).T
    assert np.all(np.abs(v - exact) <= cut)
    for p in (-1,) + ref.PLANS + ref.DUO:
        plan(p)
        got = call(ctx, W, x, xs)
        assert np.all(np.abs(got - v) <= f32_off + ref.BF16 * (np.abs(v) + f32_off)), p
        assert np.all(np.abs(got - exact) <= cut + f32_off + ref.BF16 * (np.abs(exact) + cut + f32_off)), p
    W.w.close()


# ---- many experts ------------------------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("E", [63, 64, 65, 200, 1000, 1024])
def test_many_experts(ctx, plan, gated, E):  # noqa: F811
    """A lane of the groups' search holds up to 16 of them: groups that are empty, of one
    row, and of several tiles of rows and columns."""
    N, K, x_rows = 144, 144, 64
    rng = np.random.default_rng(E)
    codes = any_codes(rng, (E, 2 * N if gated else N, K))
    nb = (2 if gated else 1) * ref.blocks(N)
    scales = rng.uniform(1e-4, 1e-3, (E, nb, ref.blocks(K))).astype(np.float32)
    W = weights(ctx, codes, scales, gated)
    counts = rng.choice([0, 0, 1, 2, 5], E)
    counts[rng.choice(E, 4, replace=False)] = [17, 70, 130, 300]
    counts[-1] = 33
    offsets, order, src = rows_ref.plan_of(counts, n=int(counts.sum()) + 9, fan=3, seed=E, x_rows=x_rows)
    x = any_codes(rng, (x_rows, K))
    xs = np.ascontiguousarray(ref.scale_up(rng.uniform(1e-3, 1e-2, (ref.blocks(K), x_rows))))
    for p in (-1,) + ref.GROUPED_PLANS:
        print(f"case f8 experts E={E} plan {p} gated={gated}", flush=True)
        plan(p)
        check(call(ctx, W, x, xs, offsets, order, order.size, fan=3), W, x, xs, offsets, src)
    plan(-1)
    sizes = [W.w.workspace_bytes(n) for n in range(0, 40 * E, max(1, E // 16) + 1)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))
    W.w.close()


# ---- a real width ------------------------------------------------------------------------
@pytest.mark.parametrize("gated,N,K", [(False, 2560, 10240), (True, 10240, 2560)])
def test_every_kernel_at_a_real_width(ctx, plan, gated, N, K):  # noqa: F811
    """203 rows of the model's widths: some rows against the 64-bit form, from each kernel."""
    M, rows = 203, [0, 15, 16, 63, 64, 127, 128, 202]
    rng = np.random.default_rng(N)
    codes = any_codes(rng, (1, 2 * N if gated else N, K))
    nb = (2 if gated else 1) * ref.blocks(N)
    scales = rng.uniform(1e-5, 1e-4, (1, nb, ref.blocks(K))).astype(np.float32)
    W = weights(ctx, codes, scales, gated)
    x = any_codes(rng, (M, K))
    xs = np.ascontiguousarray(ref.scale_up(rng.uniform(1e-4, 1e-3, (ref.blocks(K), M))))
    some = x[rows], np.ascontiguousarray(xs[:, rows])
    v, d = ref.products(*some, codes, scales, gated=gated)
    for p in (-1,) + (ref.PLANS if gated else ref.PLANS + ref.DUO):
        print(f"case f8 width plan {p} gated={gated}", flush=True)
        plan(p)
        got = call(ctx, W, x, xs)
        if gated:
            ref.check_quantized(got[0][rows], np.ascontiguousarray(got[1][:, rows]), v, d)
        else:
            assert np.all(np.abs(got[rows] - v) <= ref.bf16_bound(v, d)), p
            assert rows_ref.rel(got[rows], v) <= rows_ref.REL
    W.w.close()


# ---- rows by themselves ------------------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [2, 40, 300])
def test_a_row_does_not_feel_the_others(ctx, plan, gated, M):  # noqa: F811
    """A kernel gives a row the same bits whatever the rows beside it hold."""
    N, K = 272, 400
    W = Weights(ctx, 9300, 1, N, K, gated)
    x, xs = ref.make_rows(9301, M, K)
    z, zs = ref.make_rows(9302, M, K)
    z[1::2], zs[:, 1::2] = x[1::2], xs[:, 1::2]
    z[0] = ref.NAN
    for p in (-1,) + (ref.PLANS if gated else ref.PLANS + ref.DUO):
        plan(p)
        a, b = call(ctx, W, x, xs), call(ctx, W, z, zs)
        if gated:
            assert np.array_equal(a[0][1::2], b[0][1::2]) and np.array_equal(a[1][:, 1::2], b[1][:, 1::2])
        else:
            assert np.array_equal(a[1::2], b[1::2])
    W.w.close()
