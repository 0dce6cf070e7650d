"""The router, the grouping and the weighted sum around a mixture's expert
products against their plain 64-bit forms. Choices, offsets, orders and places
are whole numbers and equal; weights are f64 values rounded once to f32."""
import numpy as np
import pytest
import torch

import ming_dit_amd as m
import rows_ref as ref
from helpers import bf16, empty_bf16, f32, from_dev, randn, sync, to_dev

pytestmark = pytest.mark.gpu
GUARD = 64


def _i32(n, fill=-7):
    return torch.full((n,), fill, dtype=torch.int32, device="cuda")


# ---- router --------------------------------------------------------------------
def _route(ctx, logits, E, k, f32_in, pad=0, **kw):
    rows = logits.shape[0]
    wide = np.full((rows, E + pad), 9.0, np.float32)
    wide[:, :E] = logits
    src = to_dev(wide if f32_in else bf16(wide))
    ids = _i32(rows * k + GUARD)
    w = torch.full((rows * k + GUARD,), 5.0, dtype=torch.float32, device="cuda")
    bias = kw.pop("bias", None)
    sync()
    ctx.topk_route(src, rows, E, k, ids, w, bias=None if bias is None else to_dev(bias),
                   ld=E + pad, **kw)
    ctx.synchronize()
    ids, w = from_dev(ids), from_dev(w)
    assert np.all(ids[rows * k:] == -7) and np.all(w[rows * k:] == 5.0)
    seen = logits if f32_in else f32(bf16(logits))
    want, ww = ref.route(seen, k, bias=bias, **kw)
    assert np.array_equal(ids[:rows * k].reshape(rows, k), want)
    got = w[:rows * k].reshape(rows, k).astype(np.float64)
    assert np.all(np.abs(got - ww) <= ref.F32 * (1 + 1e-6) * np.abs(ww) + 2.0 ** -149)
    return want


@pytest.mark.parametrize("rows,E,k,G,tg,score,bias,f32_in,normalize", [
    (1, 1, 1, 1, 1, "softmax", False, True, True),
    (1, 2, 2, 2, 2, "sigmoid", True, False, True),
    (3, 60, 6, 1, 1, "softmax", False, True, False),
    (5, 64, 64, 1, 1, "softmax", True, True, True),
    (130, 65, 3, 5, 2, "sigmoid", True, True, True),
    (33, 256, 8, 8, 4, "sigmoid", True, False, True),
    (33, 256, 8, 8, 4, "softmax", False, False, False),
    (7, 512, 16, 64, 7, "sigmoid", False, True, True),
    (4, 1000, 33, 4, 1, "softmax", True, False, True),
    (2, 1024, 64, 64, 64, "sigmoid", True, True, False),
])
def test_route(ctx, rows, E, k, G, tg, score, bias, f32_in, normalize):
    l = randn(9000 + E, (rows, E), 2.0)
    b = randn(9100 + E, (E,), 0.1) if bias else None
    _route(ctx, l, E, k, f32_in, pad=3, bias=b, n_groups=G, top_groups=tg, score=score,
           normalize=normalize, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("G,tg", [(1, 1), (4, 2)])
def test_route_ties_go_to_the_lowest_index(ctx, score, G, tg):
    l = np.round(randn(9200, (40, 96), 1.0))          # a handful of values
    ids = _route(ctx, l, 96, 8, True, n_groups=G, top_groups=tg, score=score)
    l[:] = 0.5
    ids = _route(ctx, l, 96, 8, False, n_groups=G, top_groups=tg, score=score)
    assert np.array_equal(ids, np.tile(np.arange(8, dtype=np.int32), (40, 1)))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("G,tg", [(1, 1), (4, 2)])
def test_route_masked_and_extreme_logits(ctx, score, G, tg):
    l = randn(9300, (12, 40), 1.0)
    l[0] = -np.inf                     # nothing to choose
    l[1, 3:] = -np.inf                 # fewer than k
    l[2, ::2] = np.nan
    l[3, 5] = np.inf
    l[4] = np.nan
    l[5] = np.finfo(np.float32).min    # the type's lowest value is a logit
    l[6] = -1e30
    l[6, 7] = 1e30
    l[7, :20] = -np.inf
    l[8, 9] = l[8, 31] = np.inf
    ids = _route(ctx, l, 40, 6, True, n_groups=G, top_groups=tg, score=score, normalize=True)
    assert np.all(ids[[0, 4]] == -1) and np.all(ids[1, 3:] == -1)
    b = randn(9301, (40,), 0.1)
    b[11], b[12], b[13] = np.nan, -np.inf, np.inf
    ids = _route(ctx, l, 40, 6, True, bias=b, n_groups=G, top_groups=tg, score=score,
                 normalize=False)
    assert not np.isin(ids, (11, 12)).any()


def test_route_many_rows(ctx):
    _route(ctx, randn(9400, (4099, 60), 1.5), 60, 6, True, score="softmax", normalize=True)


def test_route_refusals(ctx):
    l = to_dev(randn(9500, (4, 64)))
    ids, w = _i32(64), torch.zeros(64, device="cuda")
    sync()
    for kw in ({"top_k": 0}, {"top_k": 65}, {"n_experts": 0}, {"n_experts": 1025},
               {"n_groups": 3}, {"n_groups": 0}, {"n_groups": 128}, {"top_groups": 2},
               {"n_groups": 8, "top_groups": 1, "top_k": 9}, {"ld": 63}, {"rows": -1}):
        a = dict(rows=4, n_experts=64, top_k=4)
        a.update(kw)
        with pytest.raises(m.MingError):
            ctx.topk_route(l, a.pop("rows"), a.pop("n_experts"), a.pop("top_k"), ids, w, **a)
    for args in ((None, ids, w), (l, None, w), (l, ids, None)):
        with pytest.raises(m.MingError, match="null|misaligned"):
            m._check(m.lib().ming_topk_route(ctx.h, m._ptr(args[0]), 64, 1, None, 4, 64, 4, 1, 1,
                                             0, 1, 1.0, m._ptr(args[1]), m._ptr(args[2])))
    ctx.topk_route(l, 0, 64, 4, ids, w)               # no rows: nothing to do
    ctx.synchronize()
    assert bool((ids == -7).all())


def test_route_shared_memory_and_sizes(ctx):
    l = to_dev(randn(9501, (16, 64)))
    ids, w = _i32(64), torch.zeros(64, device="cuda")
    sync()
    for kw in ({"ids": l}, {"weights": l}, {"ids": w}, {"bias": w, "weights": w},
               {"rows": 1 << 26}):
        a = dict(logits=l, rows=16, n_experts=64, top_k=4, ids=ids, weights=w)
        a.update(kw)
        with pytest.raises(m.MingError, match="share|2\\^26"):
            ctx.topk_route(**a)
    none = torch.zeros((0, 64), device="cuda")            # has no address
    ctx.topk_route(none, 0, 64, 4, none, none)


@pytest.mark.parametrize("E,k", [(1024, 64), (1000, 64), (65, 64), (1, 1)])
def test_route_largest_and_smallest(ctx, E, k):
    """All of a wave's lanes hold a choice; scores that tie across registers."""
    for rows, seed in ((1, 0), (5, 1)):
        l = np.round(randn(9600 + E + seed, (rows, E), 3.0) * 4) / 4
        l[:, ::7] = l[:, :1]
        ids, w = _i32(rows * k), torch.zeros((rows, k), device="cuda")
        ld = to_dev(l.astype(np.float32))
        sync()
        ctx.topk_route(ld, rows, E, k, ids, w)
        ctx.synchronize()
        wid, ww = ref.route(l.astype(np.float32), k)
        assert np.array_equal(from_dev(ids).reshape(rows, k), wid)
        assert np.allclose(from_dev(w), ww, rtol=ref.F32 * 2, atol=1e-30)


# ---- grouping ------------------------------------------------------------------
def _group(ctx, ids, G):
    n = ids.size
    bufs = [_i32(G + 1 + GUARD), _i32(n + GUARD), _i32(n + GUARD)]
    ws = torch.empty(max(1, m.group_rows_workspace_bytes(n, G)), dtype=torch.uint8, device="cuda")
    src = to_dev(ids if n else np.zeros(1, np.int32))
    sync()
    ctx.group_rows(src, n, G, *bufs, ws)
    ctx.synchronize()
    for b, size, want in zip(bufs, (G + 1, n, n), ref.group(ids, G)):
        b = from_dev(b)
        assert np.array_equal(b[:size], want)
        assert np.all(b[size:] == -7)


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 1000, 1025, 4096, 4097, 20001])
@pytest.mark.parametrize("G", [1, 2, 63, 64, 256, 1024])
def test_group_rows(ctx, n, G):
    rng = np.random.default_rng(n * 7 + G)
    ids = rng.integers(-2, G + 2, n).astype(np.int32)      # some in no group
    _group(ctx, ids, G)


@pytest.mark.parametrize("n", [40, 5000, 300000])
@pytest.mark.parametrize("what", ["one", "none", "last", "sorted", "extreme"])
def test_group_rows_uneven(ctx, n, what):
    G = 77
    ids = {"one": np.full(n, 5), "none": np.full(n, -1), "last": np.full(n, G - 1),
           "sorted": np.sort(np.arange(n) % G),
           "extreme": np.where(np.arange(n) % 2, 2 ** 31 - 1, -2 ** 31)}[what].astype(np.int32)
    _group(ctx, ids, G)


def test_group_rows_refusals(ctx):
    ids, o, p = _i32(5000), _i32(5000), _i32(5000)
    off = _i32(65)
    ws = torch.empty(m.group_rows_workspace_bytes(5000, 64), dtype=torch.uint8, device="cuda")
    for n, G in ((-1, 64), (5000, 0), (5000, 1025)):
        with pytest.raises(m.MingError):
            ctx.group_rows(ids, n, G, off, o, p, ws)
    with pytest.raises(m.MingError):
        ctx.group_rows(ids, 5000, 64, off, o, p, None)
    with pytest.raises(m.MingError, match="workspace"):
        ctx.group_rows(ids, 5000, 64, off, o, p, ws[:-4])
    with pytest.raises(m.MingError):
        ctx.group_rows(None, 10, 64, off, o, p, ws)


def test_group_rows_shared_memory(ctx):
    buf = _i32(20000, 0)
    off, o, p, ids = buf[:100], buf[100:5100], buf[5100:10100], buf[10100:15100]
    ws = buf[15100:].view(torch.uint8)
    ws = ws[(-ws.data_ptr()) % 16:]
    ok = dict(ids=ids, n=5000, n_groups=64, offsets=off, order=o, place=p, ws=ws)
    sync()
    ctx.group_rows(**ok)
    ctx.synchronize()
    for kw in ({"order": p}, {"place": ids}, {"order": ids}, {"offsets": buf[60:160]},
               {"ws": buf[(-buf.data_ptr()) % 16 // 4:].view(torch.uint8)}):
        with pytest.raises(m.MingError, match="share"):
            ctx.group_rows(**dict(ok, **kw))


# ---- the weighted sum -------------------------------------------------------------
@pytest.mark.parametrize("tokens,k,N,pad,add", [
    (1, 1, 8, 0, None), (1, 8, 2048, 0, "own"), (7, 3, 72, 16, "own"), (300, 9, 264, 8, "out"),
    (65, 4, 4096, 0, None), (513, 2, 16, 0, "out"), (10, 33, 2056, 8, "own")])
def test_combine(ctx, tokens, k, N, pad, add):
    rng = np.random.default_rng(tokens * k)
    n = tokens * k + 5
    y = bf16(randn(9600 + N, (n, N + pad)))
    place = rng.permutation(n)[:tokens * k].reshape(tokens, k).astype(np.int32)
    place[rng.random(place.shape) < 0.2] = -1
    place[0, 0] = n + 3                                     # outside: adds nothing
    w = rng.random((tokens, k)).astype(np.float32) * 2 - 0.5
    unread = np.setdiff1d(np.arange(n), place)
    y[unread] = 0x7fc0                                      # NaN in rows no token names
    w[0, 0] = np.inf
    out0 = bf16(randn(9601, (tokens, N + pad)))
    ad = None if add is None else (out0 if add == "out" else bf16(randn(9602, (tokens, N + pad))))
    yd, out = to_dev(y), to_dev(out0)
    addd = None if ad is None else (out if add == "out" else to_dev(ad))
    sync()
    ctx.experts_combine(yd, n, to_dev(place), to_dev(w), tokens, k, out, N, add=addd,
                        ldy=N + pad, ldadd=N + pad, ldo=N + pad)
    ctx.synchronize()
    got = from_dev(out)
    assert np.array_equal(got[:, N:], out0[:, N:])
    want, bound = ref.combine(f32(y)[:, :N], place, w, None if ad is None else f32(ad)[:, :N], n)
    assert np.all(np.abs(f32(got[:, :N]) - want) <= bound)


def test_combine_refusals(ctx):
    y, out = empty_bf16(16, 64), empty_bf16(8, 64)
    place, w = _i32(16, 0), torch.zeros(16, device="cuda")
    ok = dict(y=y, n=16, place=place, weights=w, tokens=8, top_k=2, out=out, N=64)
    for kw in ({"N": 60}, {"N": 72}, {"ldy": 66}, {"ldo": 56}, {"top_k": 0}, {"tokens": -1},
               {"n": -1}, {"y": None}, {"out": None}, {"place": None}, {"weights": None},
               {"out": y}, {"add": out.data_ptr() + 16}, {"out": out.data_ptr() + 2}):
        with pytest.raises(m.MingError):
            ctx.experts_combine(**dict(ok, **kw))
    ctx.experts_combine(**dict(ok, tokens=0))
    ctx.experts_combine(None, 0, None, None, 0, 2, None, 64)


def test_combine_shared_memory_and_sizes(ctx):
    buf, w = empty_bf16(64, 128), torch.zeros(32, device="cuda")
    y, out = buf.data_ptr(), buf.data_ptr() + 2 * 64      # columns beside each other
    place = _i32(32, 0)
    ok = dict(y=y, n=64, place=place, weights=w, tokens=16, top_k=2, out=out, N=64, ldy=128,
              ldo=128)
    sync()
    ctx.experts_combine(**ok)
    ctx.synchronize()
    for kw in ({"out": out - 16}, {"place": out + 128}, {"weights": out}, {"add": out, "ldadd": 64},
               {"add": out + 16, "ldadd": 128}, {"tokens": 2 ** 31 - 1}):
        with pytest.raises(m.MingError, match="share|launch"):
            ctx.experts_combine(**dict(ok, **kw))


def test_empty_arrays(ctx):
    """Calls of no rows take tensors without an address; a grouping of no entries says
    that every group is empty."""
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    off = torch.full((6,), 7, dtype=torch.int32, device="cuda")
    sync()
    ctx.topk_route(e, 0, 8, 2, e, e)
    ctx.group_rows(e, 0, 5, off, e, e)
    ctx.experts_combine(e, 0, e, e, 0, 2, e, 64)
    ctx.synchronize()
    assert not from_dev(off).any()


@pytest.mark.parametrize("rows", [2 ** 26 - 3, 2 ** 26 - 1, 2 ** 31 - 1])
def test_route_of_more_rows_than_a_launch_holds(ctx, rows):
    """Refused by their count, before any array is looked at."""
    far = 1 << 56
    with pytest.raises(m.MingError, match="2\\^26") as e:
        m._check(m.lib().ming_topk_route(ctx.h, far, 8, 1, None, rows, 8, 2, 1, 1, 0, 1, 1.0,
                                         far << 1, far << 2))
    assert e.value.code == 2
