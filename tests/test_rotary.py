# SPDX-License-Identifier: Apache-2.0
"""Rotary positions on the CPU: frequencies, and the refusals of the Python
layer and of the C ABI (before any launch)."""
import math

import pytest
import torch

from kotflash_b200 import _ext, apply_rotary, rotary_frequencies

F16 = torch.float16


def test_frequencies():
    f, magnitude = rotary_frequencies(8, base=16.0)
    assert f.dtype == torch.float64 and f.tolist() == [1.0, 0.5, 0.25, 0.125] and magnitude == 1.0
    f, magnitude = rotary_frequencies(8, base=16.0, scaling="linear", factor=4.0)
    assert f.tolist() == [0.25, 0.125, 0.0625, 0.03125] and magnitude == 1.0
    plain, _ = rotary_frequencies(64)
    f, magnitude = rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert f[0] == 1.0 and math.isclose(f[-1].item(), plain[-1].item() / 8, rel_tol=1e-12) and magnitude == 1.0
    f, magnitude = rotary_frequencies(64, scaling="yarn", factor=8.0, trained_length=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(f[turns >= 32], plain[turns >= 32])
    assert torch.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((f < plain) & (f > plain / 8))[between].all()
    assert math.isclose(magnitude, 0.1 * math.log(8) + 1)
    assert rotary_frequencies(2, scaling="ntk", factor=2.0)[0].tolist() == [1.0]


@pytest.mark.parametrize("args,match", [
    (dict(rotated=7), "even"), (dict(rotated=0), "even"), (dict(rotated=True), "even"), (dict(rotated=8, base=0.0), "base"),
    (dict(rotated=8, factor=0.5), "factor"), (dict(rotated=8, scaling="cubic"), "scaling"), (dict(rotated=8, scaling="yarn"), "trained_length"),
    (dict(rotated=8, scaling="yarn", trained_length=100, slow=2.0, fast=1.0), "slow"),
])
def test_frequency_refusals(args, match):
    with pytest.raises(ValueError, match=match):
        rotary_frequencies(**args)


@pytest.mark.parametrize("changes,error,match", [
    (dict(q=None), TypeError, "torch.Tensor"), (dict(q=torch.zeros(2, 3, 64, dtype=F16)), ValueError, "4-D"),
    (dict(q=torch.zeros(2, 4, 5, 64)), ValueError, "dtypes must match"), (dict(k=torch.zeros(2, 2, 6, 64, dtype=F16)), ValueError, "agree"),
    (dict(k=torch.zeros(2, 2, 5, 72, dtype=F16)), ValueError, "agree"), (dict(q=torch.zeros(2, 4, 5, 64), k=None), TypeError, "float16 and bfloat16"),
    (dict(positions=torch.zeros(5)), TypeError, "positions"), (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions"),
    (dict(positions=torch.zeros(1, 5, dtype=torch.int32)), ValueError, "positions"),
    (dict(frequencies=torch.zeros(32)), TypeError, "float64"), (dict(frequencies=torch.zeros(33, dtype=torch.float64)), ValueError, "frequencies"),
    (dict(frequencies=torch.zeros(0, dtype=torch.float64)), ValueError, "frequencies"),
    (dict(frequencies=torch.zeros(64, dtype=torch.float64)[::2]), ValueError, "frequencies"),
    (dict(frequencies=torch.zeros(32, dtype=torch.float64, requires_grad=True)), RuntimeError, "gradient"),
    (dict(), RuntimeError, "sm_100"),
])
def test_refusals(changes, error, match):
    a = dict(q=torch.zeros(2, 4, 5, 64, dtype=F16), k=torch.zeros(2, 2, 5, 64, dtype=F16), positions=torch.zeros(2, 5, dtype=torch.int32),
             frequencies=torch.zeros(32, dtype=torch.float64))
    a.update(changes)
    with pytest.raises(error, match=match):
        apply_rotary(**a)


def test_c_abi_refuses_before_any_launch():
    lib, p = _ext.load(), 0x1000

    def t(shape, ptr=p, last=1):
        return (0,) * 9 if shape is None else (ptr, *shape, shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], last)

    def rotary(q=(2, 4, 5, 64), k=(2, 2, 5, 64), qo=None, ko=None, pos=p, bits=32, freqs=p, rotated=64, magnitude=1.0, dtype=0, last=1, q_ptr=p):
        return lib.kf_rotary(_ext.pack_rotary(*t(q, q_ptr, last), *t(k), *t(qo or q), *t(ko or k), pos, bits, 5, 1, freqs, rotated, 0, 0, magnitude, dtype, 0))

    for kw, code, match in [
        (dict(dtype=3), _ext.KF_ERR_INVALID, "dtype"), (dict(q=(2, 4, 0, 64)), _ext.KF_ERR_INVALID, "non-zero"),
        (dict(k=(2, 2, 6, 64)), _ext.KF_ERR_INVALID, "agree"), (dict(qo=(2, 4, 5, 72)), _ext.KF_ERR_INVALID, "output shapes"),
        (dict(rotated=63), _ext.KF_ERR_INVALID, "even"), (dict(rotated=66), _ext.KF_ERR_INVALID, "at most"), (dict(rotated=0), _ext.KF_ERR_INVALID, "at least"),
        (dict(bits=16), _ext.KF_ERR_INVALID, "32 or 64"), (dict(pos=0), _ext.KF_ERR_INVALID, "null"), (dict(freqs=0), _ext.KF_ERR_INVALID, "null"),
        (dict(q_ptr=0), _ext.KF_ERR_INVALID, "null"), (dict(magnitude=1e39), _ext.KF_ERR_INVALID, "magnitude"), (dict(last=2), _ext.KF_ERR_INVALID, "contiguous"),
        (dict(q=(2, 4, 2 ** 31, 64), k=None), _ext.KF_ERR_UNSUPPORTED, "too large"),
    ]:
        assert rotary(**kw) == code, (kw, _ext.last_error())
        assert match in _ext.last_error(), (kw, _ext.last_error())
    assert lib.kf_rotary(None) == _ext.KF_ERR_INVALID
