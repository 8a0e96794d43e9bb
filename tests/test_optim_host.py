"""Refusals of the optimiser that need no GPU, and the random rounding of its 8-bit states restated on the host."""
import ctypes

import numpy as np
import pytest
import torch


def test_adamw_refuses_what_it_cannot_do():
    import spmm_cpp
    p = torch.nn.Parameter(torch.ones(3))
    for bad in (dict(lr=-1.0), dict(eps=-1e-8), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1.0), dict(state_bits=16), dict(max_norm=0.0),
                dict(max_norm=float('nan')), dict(lr=float('nan')), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            spmm_cpp.AdamW([p], **bad)
    opt = spmm_cpp.AdamW([p])
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match='no CPU path'):
        opt.step()
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(2))], betas=(2.0, 0.9)))


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ('p', 'g', 'm', 'v', 'm_scale', 'v_scale', 'step')] + \
               [('n', ctypes.c_int64), ('place', ctypes.c_int64), ('type', ctypes.c_int32), ('pad', ctypes.c_int32)]


class Options(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ('lr', 'beta1', 'beta2', 'eps', 'weight_decay')] + [('seed', ctypes.c_uint32), ('bits', ctypes.c_int32)]


def test_c_entries_check_before_they_launch():
    import spmm_cpp
    L = spmm_cpp.lib()
    step, norm, need = L.dg_adamw_step, L.dg_grad_norm, L.dg_adamw_workspace
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    step.argtypes, norm.argtypes = [vp, i32, vp, vp, vp, i64, vp], [vp, i32, ctypes.c_double, vp, vp, i64, vp]
    need.argtypes, need.restype = [vp, i32], i64
    fine = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, seed=0, bits=32)

    def call(t, workspace=0x1000, size=1 << 20, **changes):
        return step(ctypes.byref(t), 1, ctypes.byref(Options(**dict(fine, **changes))), None, workspace, size, None)

    def tensor(**changes):
        return Tensor(**dict(dict(p=0x1000, g=0x1000, m=0x1000, v=0x1000, step=0x1000, n=8, type=0), **changes))

    assert call(tensor(p=None)) == -1 and call(tensor(step=None)) == -1 and call(tensor(g=None)) == -1
    assert call(tensor(), bits=8) == -1                                        # no scales
    assert call(tensor(n=-1)) == -2 and call(tensor(type=3)) == -2 and call(tensor(p=0x1002)) == -2 and call(tensor(), bits=16) == -2
    assert call(tensor(), beta1=1.0) == -2 and call(tensor(), lr=-1.0) == -2 and call(tensor(), lr=float('nan')) == -2
    assert call(tensor(), workspace=None) == -1 and call(tensor(), workspace=0x1004) == -2 and call(tensor(), size=8) != 0
    assert norm(ctypes.byref(tensor()), 1, 0.0, 0x1000, 0x1000, 1 << 20, None) == -2
    assert norm(ctypes.byref(tensor()), 1, 1.0, None, 0x1000, 1 << 20, None) == -1
    assert norm(ctypes.byref(tensor()), 1, 1.0, 0x1000, 0x1000, 16, None) != 0
    assert need(None, 3) < 0 and need(None, 0) >= 16
    assert step(None, 0, ctypes.byref(Options(**fine)), None, 0x1000, 16, None) == 0


def _mix(h):
    h = h.astype(np.uint32)
    h = (h ^ (h >> np.uint32(16))) * np.uint32(0x6A09E667)
    h = (h ^ (h >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return h ^ (h >> np.uint32(16))


def test_noise_is_even():
    """The 16-bit numbers of the roundings, over 2^20 places and three steps: every one of 16 classes has its share within six standard deviations, and
    neighbours, and the same place in the next step, are uncorrelated within six of theirs."""
    n = 1 << 20
    places = np.arange(n // 2, dtype=np.uint32) * np.uint32(0x9E3779B1)
    with np.errstate(over='ignore'):
        rows = []
        for step in (1, 2, 1000):
            key = _mix(np.array([7 + step * 0x3C6EF373], dtype=np.uint64).astype(np.uint32))
            h = _mix(places + key)
            rows.append(np.stack([h & 0xFFFF, h >> 16], 1).reshape(-1).astype(np.float64))
    for u in rows:
        counts = np.bincount((u // 4096).astype(int), minlength=16)
        assert np.abs(counts - n / 16).max() < 6 * np.sqrt(n / 16)
        assert abs(np.corrcoef(u[:-1], u[1:])[0, 1]) < 6 / np.sqrt(n)
    assert abs(np.corrcoef(rows[0], rows[1])[0, 1]) < 6 / np.sqrt(n)
