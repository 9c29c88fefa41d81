# SPDX-License-Identifier: Apache-2.0
"""K7, rotary positions, in forward mode: the rotation is linear, so a tangent
is rotated as its primal is, bit for bit (GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from kotflash_b200 import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def _rand(shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("grads", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("duals", [(True, True), (True, False), (False, True)])
def test_tangents_are_rotated(interleaved, grads, duals):
    freqs, _ = rotary_frequencies(48, device="cuda")
    positions = torch.arange(11, device="cuda")
    x = [_rand((2, h, 11, 64), h).requires_grad_(g) for h, g in zip((4, 2), grads)]
    t = [_rand((2, h, 11, 64), 10 + h) for h in (4, 2)]
    with torch.no_grad():
        want = apply_rotary(*x, positions, freqs, interleaved=interleaved, magnitude=1.25)
        turned = apply_rotary(*t, positions, freqs, interleaved=interleaved, magnitude=1.25)
    with fwd.dual_level():
        ins = [fwd.make_dual(a, b) if dual else a for a, b, dual in zip(x, t, duals)]
        outs = [fwd.unpack_dual(y) for y in apply_rotary(*ins, positions, freqs, interleaved=interleaved, magnitude=1.25)]
        for got, w, tangent, dual in zip(outs, want, turned, duals):
            assert torch.equal(got.primal, w)
            assert torch.equal(got.tangent, tangent) if dual else got.tangent is None
        if any(grads):  # and the gradient beside it
            chosen = [a for a, g in zip(x, grads) if g]
            given = [_rand(a.shape, 20 + i) for i, a in enumerate(chosen)]
            got = torch.autograd.grad([o.primal for o, g in zip(outs, grads) if g], chosen, given)
            for grad, dy, a in zip(got, given, chosen):
                # <dy, f(a)> = <f'(dy), a>, to the roundings of both
                left = (dy.double() * want[0 if a is x[0] else 1].double()).sum()
                right = (grad.double() * a.detach().double()).sum()
                slack = 2.0 ** -8 * ((dy.double() * want[0 if a is x[0] else 1].double()).abs().sum() + (grad.double() * a.detach().double()).abs().sum())
                assert (left - right).abs() <= slack


def test_one_tensor_and_no_gradients():
    freqs, _ = rotary_frequencies(64, device="cuda")
    positions = torch.arange(5, device="cuda")
    x, t = _rand((1, 3, 5, 64), 1), _rand((1, 3, 5, 64), 2)
    want = apply_rotary(t, None, positions, freqs)
    with fwd.dual_level(), torch.no_grad():
        got = fwd.unpack_dual(apply_rotary(fwd.make_dual(x, t), None, positions, freqs))
        assert torch.equal(got.tangent, want) and torch.equal(got.primal, apply_rotary(x, None, positions, freqs))


def test_a_gradient_is_differentiated_forwards():
    """The tangent of a gradient with respect to what comes in from behind."""
    freqs, _ = rotary_frequencies(64, device="cuda")
    positions = torch.arange(5, device="cuda")
    x, dy, t = _rand((1, 3, 5, 64), 1).requires_grad_(True), _rand((1, 3, 5, 64), 2), _rand((1, 3, 5, 64), 3)
    y = apply_rotary(x, None, positions, freqs)
    with torch.no_grad():
        want, = torch.autograd.grad(y, x, t, retain_graph=True)
    with fwd.dual_level():
        for create_graph in (False, True):
            got, = torch.autograd.grad(y, x, fwd.make_dual(dy, t), retain_graph=True, create_graph=create_graph)
            assert torch.equal(fwd.unpack_dual(got).tangent, want)


def test_a_tangent_is_differentiated_backwards():
    freqs, _ = rotary_frequencies(64, device="cuda")
    positions = torch.arange(5, device="cuda")
    x, t = _rand((1, 3, 5, 64), 1).requires_grad_(True), _rand((1, 3, 5, 64), 3).requires_grad_(True)
    dy = _rand((1, 3, 5, 64), 2)
    y = apply_rotary(t, None, positions, freqs)
    want, = torch.autograd.grad(y, t, dy)
    with fwd.dual_level():
        tangent = fwd.unpack_dual(apply_rotary(fwd.make_dual(x, t), None, positions, freqs)).tangent
        got, = torch.autograd.grad(tangent, t, dy)
    assert torch.equal(got, want)
