"""The 8-bit operators' refusals that need no GPU, and the reference of their codes against itself."""
import ctypes

import pytest
import torch

import act8_ref as ref


def test_codes_by_counting():
    """The reference's codes are the nearest whole numbers, ties to even, by exhaustive fractions."""
    from fractions import Fraction
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.randint(-300, 301, (4, 40), generator=g).double() / 8, torch.randn(4, 40, generator=g).to(torch.bfloat16).double(),
                   torch.zeros(1, 40, dtype=torch.float64)])
    q, s = ref.codes(v)
    for i in range(v.shape[0]):
        m = max(abs(Fraction(float(t))) for t in v[i])
        for t, k in zip(v[i], q[i]):
            want = 0 if m == 0 else round(Fraction(float(t)) * 127 / m)          # round(Fraction): half to even
            assert int(k) == want
        assert float(s[i]) == pytest.approx(float(m) / 127, rel=1e-15)


def test_norm_create_refusals(ek):
    from ek_hip import _capi as C
    lib, h = ek.load(), ctypes.c_void_p()
    gain = torch.ones(64, dtype=torch.bfloat16)
    base = dict(hidden=64, act_dtype=C.EK_BF16, eps=1e-6, device_id=0, flags=0)
    for patch in (dict(hidden=0), dict(hidden=60), dict(hidden=-8), dict(hidden=1 << 25), dict(act_dtype=C.EK_F32), dict(eps=0.0), dict(eps=-1.0),
                  dict(eps=float("inf")), dict(eps=float("nan")), dict(flags=1)):
        cfg = C.ek_norm_cfg(**{**base, **patch})
        assert lib.ek_norm_create(ctypes.byref(cfg), gain.data_ptr(), C.EK_HOST, ctypes.byref(h)) == C.EK_INVALID_INPUT, patch
        assert lib.ek_last_error() and not h.value
    cfg = C.ek_norm_cfg(**base)
    assert lib.ek_norm_create(ctypes.byref(cfg), None, C.EK_HOST, ctypes.byref(h)) == C.EK_WEIGHT_NOT_FOUND
    assert lib.ek_norm_create(ctypes.byref(cfg), gain.data_ptr(), 7, ctypes.byref(h)) == C.EK_INVALID_INPUT
    assert lib.ek_norm_create(None, gain.data_ptr(), C.EK_HOST, ctypes.byref(h)) == C.EK_INVALID_INPUT
    assert lib.ek_norm_create(ctypes.byref(cfg), gain.data_ptr(), C.EK_HOST, None) == C.EK_INVALID_INPUT
    cfg = C.ek_norm_cfg(**{**base, "device_id": 99})
    assert lib.ek_norm_create(ctypes.byref(cfg), gain.data_ptr(), C.EK_HOST, ctypes.byref(h)) == C.EK_HIP_ERROR
    assert lib.ek_norm_forward(None, None, None, 0, None, None, None, None, 0, None) == C.EK_INVALID_INPUT
    assert lib.ek_norm_shape(None, None, None) == C.EK_INVALID_INPUT
    assert lib.ek_norm_destroy(None) == C.EK_INVALID_INPUT


def test_linear_create_refusals(ek):
    from ek_hip import _capi as C
    lib, h = ek.load(), ctypes.c_void_p()
    w, s = torch.zeros(32, 128, dtype=torch.int8), torch.ones(32)
    base = dict(in_features=128, out_features=32, max_rows=16, act_dtype=C.EK_BF16, device_id=0, flags=0)

    def desc(**kw):
        d = C.ek_weight_desc()
        d.ptr, d.rows, d.cols, d.dtype, d.mem = w.data_ptr(), 32, 128, C.EK_I8, C.EK_HOST
        d.scale, d.scale_dtype, d.scale_kind = s.data_ptr(), C.EK_F32, C.EK_SCALE_PER_CHANNEL
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    def create(cfg_patch, desc_patch, bias=None, bias_dtype=0):
        cfg, d = C.ek_linear_cfg(**{**base, **cfg_patch}), desc(**desc_patch)
        return lib.ek_linear_create(ctypes.byref(cfg), ctypes.byref(d), bias, bias_dtype, ctypes.byref(h))

    for patch in (dict(in_features=0), dict(in_features=131073), dict(out_features=0), dict(out_features=1 << 25), dict(max_rows=0),
                  dict(max_rows=65535 * 64 + 1), dict(act_dtype=C.EK_I8), dict(flags=2), dict(in_features=64), dict(out_features=31)):
        assert create(patch, {}) == C.EK_INVALID_INPUT, patch
    for patch in (dict(dtype=C.EK_BF16), dict(dtype=C.EK_F8E4M3), dict(scale_kind=C.EK_SCALE_NONE), dict(scale_kind=C.EK_SCALE_BLOCK128),
                  dict(scale_dtype=C.EK_I8), dict(mem=5)):
        assert create({}, patch) == C.EK_INVALID_INPUT, patch
    assert create({}, dict(ptr=None)) == C.EK_WEIGHT_NOT_FOUND
    assert create({}, dict(scale=None)) == C.EK_WEIGHT_NOT_FOUND
    assert create({}, {}, s.data_ptr(), C.EK_I8) == C.EK_INVALID_INPUT
    assert create(dict(device_id=99), {}) == C.EK_HIP_ERROR
    assert lib.ek_linear_forward(None, None, None, 0, None, 0, None) == C.EK_INVALID_INPUT
    assert lib.ek_linear_shape(None, None, None) == C.EK_INVALID_INPUT
    assert lib.ek_linear_destroy(None) == C.EK_INVALID_INPUT
