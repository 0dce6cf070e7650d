"""What the operators in 8-bit floating point refuse without a GPU, and their plain
forms against torch's own casts."""
import ctypes as C

import numpy as np
import torch

import f8_ref as ref
import ming_dit_amd as m


def test_null_arguments_are_refused_with_a_reason():
    L = m.lib()
    h = C.c_void_p(1)
    for rc in (L.ming_f8_quantize(None, None, 0, 1, 16, None, 0, None, 0),
               L.ming_f8_rmsnorm(None, None, 0, None, 0, None, 0, None, None, 0, None, 0, None, 0,
                                 1, 16, 1e-6),
               L.ming_f8_quantize_weight(None, None, 8, 16, None, None),
               L.ming_f8_create(None, 1, 8, 16, 0, None, None, 0, C.byref(h)),
               L.ming_f8_shape(None, None, None, None, None),
               L.ming_f8_lin(None, None, None, 0, None, 0, None, 0, 1, None, None, 0),
               L.ming_f8_swiglu(None, None, None, 0, None, 0, None, 0, None, 0, 1, None, 0),
               L.ming_f8_experts_lin(None, None, None, 0, None, 0, 1, None, 1, None, 1, None, 0,
                                     None, 0),
               L.ming_f8_experts_swiglu(None, None, None, 0, None, 0, 1, None, 1, None, 1, None, 0,
                                        None, 0, None, 0)):
        assert rc == 1
        assert b"null" in L.ming_last_error()
    assert not h.value
    assert L.ming_f8_create(None, 1, 8, 16, 0, None, None, 0, None) == 1
    assert L.ming_f8_destroy(None) == 0
    assert L.ming_f8_workspace_bytes(None, 4) == 0


def test_codes_agree_with_torch():
    """The tests' own table and rounding against torch's e4m3."""
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.decode(codes), want, equal_nan=True)
    rng = np.random.default_rng(0)
    fine = ref.VALUES[np.isfinite(ref.VALUES)]
    mids = (np.sort(fine)[1:] + np.sort(fine)[:-1]) / 2
    v = np.concatenate([fine, mids, rng.uniform(-448, 448, 4000), rng.normal(0, 0.02, 4000),
                        [448.0, -448.0, 0.0, -0.0]]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(v.astype(np.float64)), want)


def test_quantized_rows_by_hand():
    v = np.zeros((2, 130))
    v[0, :4] = [448.0, 1.0, -0.0625, 17.0]      # 17 lies between 16 and 18: to even, 16
    v[1, 128:] = [3.0, -1.5]
    codes, scales = ref.quantize(v)
    assert np.array_equal(ref.decode(codes)[0, :4], [448.0, 1.0, -0.0625, 16.0])
    assert scales[0, 0] == 0x3f80
    # 3 / 448 = 1.714.. 2^-8: up to 220 / 128 2^-8; 3 over that is 446.8, a 448
    assert scales[1, 1] == 0x3bdc
    assert np.array_equal(ref.decode(codes)[1, 128:], [448.0, -224.0])
    # 2^-100 / 448 = 1.142.. 2^-109: up to 147 / 128 2^-109
    assert scales[0, 1] == ((127 - 109) << 7) + 147 - 128
