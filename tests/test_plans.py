"""The launch plans, which choose tile heights and K slices by size alone: on the
CPU (without a device they count the MI355X's 256 CUs), through the library's
own symbols."""
import ctypes as C
import random

import pytest

from helpers import dense_plan, plan_rows, xa_tile

SHAPES = [(M, tn, st) for M in (1, 63, 300, 700, 1280, 2085, 4352, 8320, 16640)
          for tn in (1, 8, 15, 40, 60, 80, 129) for st in (1, 4, 16, 60, 165)]


@pytest.mark.parametrize("pair", [False, True])
def test_row_plans_cover_the_rows(pair):
    for M, tn, st in SHAPES:
        p = plan_rows(M, tn, st, pair)
        assert p.rows_main == M or (p.rows_main % 256 == 0 and 0 <= p.rows_main < M), (M, tn, st)
        assert p.rf_rest in ((8, 6, 4) if pair else (8, 6, 4, 2)), (M, tn, st)


def test_row_plans_count_k():
    """A short K leaves a second launch little to gain for its start: plans that
    are two launches at K = 3840 are one at K = 64."""
    two = [s for s in ((5600, 40), (8320, 40), (16640, 40)) if 0 < plan_rows(*s, 60, False).rows_main < s[0]]
    assert two
    for M, tn in two:
        assert plan_rows(M, tn, 1, False).rows_main in (0, M)
    # 4096 rows of [10240, 64]: one launch of a lower height (28.5 us, 36.2 as
    # 256-row tiles and then 192)
    assert plan_rows(4096, 40, 1, False).rows_main == 0
    # 2560 rows of [10240, 3840]: one launch of 256-row tiles (171.8 us, 178.2)
    assert plan_rows(2560, 40, 60, False).rows_main == 2560
    # a paired launch's 4352 rows: five whole rounds, then 128-row tiles
    p = plan_rows(4352, 80, 60, True)
    assert (p.rows_main, p.rf_rest) == (4096, 4)


@pytest.mark.parametrize("M,N,K", [(203, 10240, 256), (1024, 3840, 64), (130, 15360, 128),
                                   (1024, 2560, 256), (40, 10240, 64), (16, 64, 64)])
def test_dense_plans_of_a_short_k(M, N, K):
    """A tall tile's scattered stores are most of an unsplit launch of a few K
    stages: 203 rows of [10240, 256] take 13.2 us on 256 x 128, 7.4 on the dense
    route."""
    rows, cols, slices = dense_plan(M, N, K)
    assert slices == 0 or rows * cols <= 128 * 64


def test_xa_tiles_at_half_a_chip():
    """The adapters' x.A: 256 x 128 tiles from half a chip of them on (512 ranks at
    8320 rows: 65 us, 64-row tiles 74), a block more where K is short."""
    assert xa_tile(8320, 512, 3840, 1) == (256, 128)
    assert xa_tile(16640, 256, 10240, 1) == (256, 128)
    assert xa_tile(16640, 256, 3840, 1) == (64, 128)
    assert xa_tile(16384, 256, 10240, 1) == (64, 128)
    assert xa_tile(4352, 64, 3840, 3) == (64, 64)


def test_a_banks_size_says_where_its_rows_run():
    """The rows' x.A beside a split: a few adapters' chunks, not forty's; none bound
    always, no blocks to spare never."""
    import ming_dit_amd as m
    f = m.lib()._ZN4ming13row_xa_besideEiiiii
    f.restype = C.c_bool
    for ny, M, K in ((5, 200, 3840), (1, 700, 3840), (3, 300, 2048)):
        assert f(ny, M, K, 2, 3) and not f(ny, M, K, 40, 2 + 38 * 4)
        assert f(ny, M, K, 0, 0) and not f(0, M, K, 2, 3)


def test_the_last_rows_that_one_launch_holds():
    """2^32 - 1 threads: a block more than that is refused before it is launched."""
    import ming_dit_amd as m
    route, xa = m.lib()._ZN4ming10route_fitsEx, m.lib()._ZN4ming11row_xa_fitsEii
    route.argtypes, route.restype, xa.restype = [C.c_longlong], C.c_bool, C.c_bool
    assert route(2 ** 26 - 4) and not route(2 ** 26 - 3) and not route(2 ** 31 - 1)
    assert xa(2 ** 28 - 32, 0) and not xa(2 ** 28 - 31, 0) and not xa(2 ** 28 - 32, 1)
    assert xa(767, 100) and not xa(2 ** 31 - 1, 0)


@pytest.mark.parametrize("rows_main,rest", [(0, 64), (0, 256), (256, 128), (2048, 64), (2048, 192)])
def test_a_tiles_list_holds_every_row_its_own_adapter(rows_main, rest):
    """The bound the lists' blocks write under, against tiles counted row by row."""
    import ming_dit_amd as m
    f = m.lib()._ZN4ming15row_tile_chunksEiiiii
    rng = random.Random(rest)
    for M in (rows_main + 1, rows_main + rest - 1, rows_main + rest, rows_main + 5 * rest + 3,
              max(rows_main, 1)):
        for cap, max_rank in ((1, 512), (40, 17), (4096, 64)):
            ldt = (max_rank + 31) // 32 * 32
            ids = [rng.randrange(cap) for _ in range(M)]
            for own in (ids, [i % cap for i in range(M)]):
                edges = list(range(0, rows_main, 256)) + list(range(rows_main, M, rest)) + [M]
                most = max(len(set(own[a:b])) for a, b in zip(edges, edges[1:]))
                assert most * ((max_rank + 31) // 32) <= f(M, rows_main, rest, cap, ldt)
            assert f(M, rows_main, rest, cap, ldt) <= 256 * (ldt // 32)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_the_experts_plan_counts_the_cus(bits):
    """An eighth of a chip is full of tall tiles at an eighth of the groups; 256 CUs are
    what a host without a device plans for."""
    import ming_dit_amd as m
    on, here = m.lib()._ZN4ming14experts_cut_onEiiiiii, m.lib()._ZN4ming11experts_cutEiiiii
    for E in (8, 16, 64, 128):
        for n in (1, 64, 1000, 300 * E, 600 * E):
            assert on(256, E, 2048, 2048, bits, n) == here(E, 2048, 2048, bits, n)
    tall = 8 if bits == 8 else 4
    assert on(256, 2, 2048, 2048, bits, 600) == 2 and on(32, 2, 2048, 2048, bits, 600) == tall


def test_few_row_blocks_of_the_experts():
    """Dense plain ones are narrow where wide ones would leave CUs idle, or K is long."""
    import ming_dit_amd as m
    f = m.lib()._ZN4ming18experts_rows_tilesEiibiiii
    for n, K, co in ((1, 1088, 1), (7, 1472, 1), (8, 1472, 2), (64, 1088, 2), (64, 1536, 1),
                     (1, 1024, 2)):
        assert f(256, 16, False, 64, 1024, K, n) == co, (n, K)
        assert f(256, 4, False, 64, 1024, K, n) == 2 and f(256, 8, True, 64, 1024, K, n) == 1
    assert f(32, 16, False, 64, 1024, 1088, 1) == 2
