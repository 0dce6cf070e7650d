"""What the operators whose rows choose their own weights refuse without a GPU."""
import ctypes as C

import numpy as np

import ming_dit_amd as m
import rows_ref as ref


def test_null_arguments_are_refused_with_a_reason():
    L = m.lib()
    h = C.c_void_p()
    for rc in (L.ming_topk_route(None, None, 0, 1, None, 1, 8, 1, 1, 1, 0, 1, 1.0, None, None),
               L.ming_group_rows(None, None, 1, 1, None, None, None, None, 0),
               L.ming_experts_create(None, 1, 8, 64, 4, 64, None, None, None, 0, C.byref(h)),
               L.ming_experts_create_dense(None, 1, 8, 64, None, 0, C.byref(h)),
               L.ming_experts_shape(None, None, None, None, None),
               L.ming_experts_lin(None, None, None, 0, 0, None, 1, None, 0, None, 0, None, 0),
               L.ming_experts_swiglu(None, None, None, 0, 0, None, 1, None, 0, None, 0, None, 0),
               L.ming_experts_combine(None, None, 0, 0, None, None, 0, 1, None, 0, None, 0, 8),
               L.ming_adapters_create(None, 8, 64, 1, 8, C.byref(h)),
               L.ming_adapters_set(None, 0, 1, None, None, 1.0, 0),
               L.ming_adapters_clear(None, 0),
               L.ming_lin_adapters(None, None, None, None, 0, None, 0, 1, None, None, None, 0)):
        assert rc == 1
        assert b"null" in L.ming_last_error()
    assert L.ming_experts_destroy(None) == 0 and L.ming_adapters_destroy(None) == 0
    assert L.ming_adapters_rank(None, 0) == 0
    assert L.ming_experts_workspace_bytes(None, 4) == 0
    assert L.ming_lin_adapters_workspace_bytes(None, None, None, 4) == 0


def test_group_workspace():
    assert m.group_rows_workspace_bytes(0, 8) == 0
    assert m.group_rows_workspace_bytes(64, 8) == 0
    assert m.group_rows_workspace_bytes(100, 0) == 0
    assert m.group_rows_workspace_bytes(1 << 20, 64) >= 65 * 4
    assert m.group_rows_workspace_bytes(1 << 30, 1024) < 1 << 20


def test_the_plain_forms_agree_with_brute_force():
    """The tests' own references against loops written out."""
    rng = np.random.default_rng(0)
    ids = rng.integers(-1, 5, 40).astype(np.int32)
    off, order, place = ref.group(ids, 4)
    want = [i for g in range(4) for i in range(40) if ids[i] == g]
    assert list(order[:len(want)]) == want and off[-1] == len(want)
    assert all(place[i] == want.index(i) if 0 <= ids[i] < 4 else place[i] == -1
               for i in range(40))
    got, w = ref.route(np.array([[1.0, 3.0, 3.0, -np.inf]], np.float32), 4)
    assert list(got[0]) == [1, 2, 0, -1] and w[0, 3] == 0.0 and abs(w.sum() - 1.0) < 1e-12
