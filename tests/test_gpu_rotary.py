# SPDX-License-Identifier: Apache-2.0
"""K7, rotary positions, against the formula in 64 bits (GPU)."""
import math

import pytest
import torch

from kotflash_b200 import apply_rotary, attention, rotary_frequencies

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _want(x, positions, freqs, interleaved, magnitude, sign=1.0):
    """The formula in 64 bits, and each pair's length."""
    x = x.detach().double()
    R = 2 * freqs.numel()
    at = (positions if positions.ndim == 2 else positions[None]).double()[:, None, :, None] * freqs
    c, s = torch.cos(at) * magnitude, torch.sin(at) * magnitude * sign
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2: R])
    y, size = x.clone(), x.abs()
    for t, (u, v) in ((y, (a * c - b * s, b * c + a * s)), (size, (torch.hypot(a, b) * abs(magnitude),) * 2)):
        if interleaved:
            t[..., 0:R:2], t[..., 1:R:2] = u, v
        else:
            t[..., : R // 2], t[..., R // 2: R] = u, v
    return y, size


def _check(got, x, positions, freqs, interleaved, magnitude, sign=1.0):
    """cos and sin are off by the reduced angle's rounding (2^-24 of at most pi)
    and the function's (2 units of 2^-24), the magnitude and the two products
    and their sum by 2^-24 each: 8 x 2^-24 of the pair's length in all; the
    result is rounded once.  Passing columns are copied."""
    want, size = _want(x, positions, freqs, interleaved, magnitude, sign)
    R = 2 * freqs.numel()
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert torch.equal(got[..., R:], x[..., R:])
    err = (got.double() - want).abs()[..., :R]
    bound = (UNIT[x.dtype] * want.abs() + 8 * 2.0 ** -24 * size + 2.0 ** -24 * (x.dtype == F16))[..., :R]
    assert (err <= bound).all(), f"off by {err.max():.3e}"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,R,far", [
    (1, 1, 1, 1, 16, 16, 10), (64, 1, 32, 8, 128, 128, 131072), (2, 300, 8, 2, 128, 64, 5000), (1, 77, 5, 5, 72, 72, 1 << 20),
    (3, 19, 6, 1, 72, 18, 2 ** 31 - 20), (1, 1000, 4, 4, 96, 24, 1000), (2, 33, 3, 1, 104, 104, 40000), (1, 50, 2, 2, 40, 10, 999),
    (1, 9, 40, 8, 20, 6, 100), (2, 17, 1, 3, 7, 2, 100), (1, 2500, 16, 4, 64, 64, 8192), (1, 3, 2, 1, 256, 192, 77),
])
def test_rotates_as_the_formula(interleaved, dtype, B, S, Hq, Hkv, D, R, far):
    freqs, magnitude = rotary_frequencies(R, base=500000.0, scaling="yarn", factor=8.0, trained_length=4096, device="cuda")
    first = torch.randint(0, far - S + 1, (B, 1), generator=torch.Generator().manual_seed(S)).cuda()
    positions = (first + torch.arange(S, device="cuda")).to(torch.int32)
    rows = _rand((B, S, Hq + 2 * Hkv, D), dtype, 1).transpose(1, 2)
    q, k, _ = rows.split([Hq, Hkv, Hkv], 1)
    got_q, got_k = apply_rotary(q, k, positions, freqs, interleaved=interleaved, magnitude=magnitude)
    _check(got_q, q, positions, freqs, interleaved, magnitude)
    _check(got_k, k, positions, freqs, interleaved, magnitude)
    # one tensor alone, 64-bit positions, others' strides: the same values
    wide = torch.empty(B, 2 * S, device="cuda", dtype=torch.int64)[:, ::2].copy_(positions)
    alone = apply_rotary(k.contiguous(), None, wide, freqs, interleaved=interleaved, magnitude=magnitude)
    assert torch.equal(alone, got_k)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_rows_off_their_alignment(interleaved, offset):
    """Views that begin inside 16 bytes take narrower pieces."""
    freqs, _ = rotary_frequencies(32, device="cuda")
    base = _rand((2, 3, 21, 64 + offset), BF16, 2)
    q, positions = base[..., offset:], torch.arange(21, device="cuda")
    _check(apply_rotary(q, None, positions, freqs, interleaved=interleaved), q, positions, freqs, interleaved, 1.0)
    t = q.transpose(-1, -2).contiguous().transpose(-1, -2)  # columns outside
    assert torch.equal(apply_rotary(t, None, positions, freqs, interleaved=interleaved), apply_rotary(q, None, positions, freqs, interleaved=interleaved))


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_positions_shared_by_the_batch(scaling):
    freqs, magnitude = rotary_frequencies(128, scaling=scaling, factor=4.0, trained_length=2048, device="cuda")
    q, k = _rand((3, 4, 60, 128), F16, 3), _rand((3, 2, 60, 128), F16, 4)
    positions = torch.arange(100, 160, device="cuda")
    got = apply_rotary(q, k, positions, freqs, magnitude=magnitude)
    want = apply_rotary(q, k, positions.expand(3, 60), freqs, magnitude=magnitude)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check(got[0], q, positions, freqs, False, magnitude)


def test_negative_positions_and_magnitudes():
    freqs, _ = rotary_frequencies(64, device="cuda")
    q = _rand((1, 2, 40, 64), F16, 5)
    positions = torch.arange(-20, 20, device="cuda")
    for magnitude in (1.0, -0.5, 0.0):
        _check(apply_rotary(q, None, positions, freqs, magnitude=magnitude), q, positions, freqs, False, magnitude)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,R", [(128, 128), (72, 18), (96, 64)])
def test_gradients(interleaved, dtype, D, R):
    """Against the formula (the rotation back), and against differences: the map
    is linear, so <g, f(x + e) - f(x)> is <grad, e>, to the roundings of f."""
    freqs, magnitude = rotary_frequencies(R, scaling="yarn", factor=2.0, trained_length=100, device="cuda")
    positions = torch.randint(0, 9000, (2, 37), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    q, k = _rand((2, 6, 37, D), dtype, 1).requires_grad_(True), _rand((2, 37, 2, D), dtype, 2).transpose(1, 2).requires_grad_(True)
    gq, gk = _rand((2, 37, 6, D), dtype, 3).transpose(1, 2), _rand((2, 2, 37, D), dtype, 4)
    out = apply_rotary(q, k, positions, freqs, interleaved=interleaved, magnitude=magnitude)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk))
    _check(dq, gq, positions, freqs, interleaved, magnitude, -1.0)
    _check(dk, gk, positions, freqs, interleaved, magnitude, -1.0)
    for x, y, g, grad, i in ((q, out[0], gq, dq, 0), (k, out[1], gk, dk, 1)):
        e = _rand(x.shape, dtype, 9).detach()
        moved = (x.detach() + e)                      # rounded: the difference is what it is
        e = moved.double() - x.detach().double()
        args = (moved, None)
        z = apply_rotary(*args, positions, freqs, interleaved=interleaved, magnitude=magnitude)
        by_difference = ((z.double() - y.detach().double()) * g.double()).sum().item()
        by_gradient = (grad.double() * e).sum().item()
        slack = (UNIT[dtype] * (z.abs().double() + y.detach().abs().double()) * g.abs().double()).sum() + (UNIT[dtype] * grad.abs().double() * e.abs()).sum()
        # roundings are independent and of either sign; their worst sum is the bound
        assert abs(by_difference - by_gradient) <= slack.item() * 1.01


def test_gradients_of_one_of_two_and_expanded_ones():
    freqs, _ = rotary_frequencies(64, device="cuda")
    positions = torch.arange(11, device="cuda")
    q, k = _rand((1, 2, 11, 64), BF16, 1), _rand((1, 1, 11, 64), BF16, 2).requires_grad_(True)
    oq, ok = apply_rotary(q, k, positions, freqs)
    assert ok.requires_grad and not oq.requires_grad
    (dk,) = torch.autograd.grad(ok.sum(), (k,))       # a gradient of stride 0
    _check(dk, torch.ones_like(k), positions, freqs, False, 1.0, -1.0)
    q.requires_grad_(True)
    oq, ok = apply_rotary(q, k, positions, freqs)
    dq, dk = torch.autograd.grad(oq.float().square().sum(), (q, k), allow_unused=True)
    assert dk is None and torch.isfinite(dq).all()
    oq = apply_rotary(q, None, positions, freqs)
    (dq,) = torch.autograd.grad(oq, (q,), torch.ones_like(oq), create_graph=True)
    _check(dq.detach(), torch.ones_like(q), positions, freqs, False, 1.0, -1.0)
    with torch.no_grad():
        assert not apply_rotary(q, None, positions, freqs).requires_grad


def test_positions_that_change_before_the_backward_pass_are_refused():
    freqs, _ = rotary_frequencies(64, device="cuda")
    positions, q = torch.arange(5, device="cuda"), _rand((1, 1, 5, 64), F16, 1).requires_grad_(True)
    out = apply_rotary(q, None, positions, freqs)
    positions += 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_nothing_to_rotate():
    freqs, _ = rotary_frequencies(16, device="cuda")
    q, k = torch.empty(2, 3, 0, 16, device="cuda", dtype=F16), torch.empty(2, 1, 0, 16, device="cuda", dtype=F16)
    oq, ok = apply_rotary(q, k, torch.empty(2, 0, device="cuda", dtype=torch.int32), freqs)
    assert oq.shape == q.shape and ok.shape == k.shape
    k = _rand((2, 1, 4, 16), F16, 1)
    oq, ok = apply_rotary(k[:, :0], k, torch.arange(4, device="cuda"), freqs)
    assert oq.shape == (2, 0, 4, 16) and torch.equal(ok, apply_rotary(k, None, torch.arange(4, device="cuda"), freqs))


def test_infinities_and_nan_stay_in_their_pair():
    freqs, _ = rotary_frequencies(32, device="cuda")
    q = _rand((1, 1, 8, 64), F16, 1)
    q[0, 0, 3, 5], q[0, 0, 4, 50] = math.nan, math.inf
    out = apply_rotary(q, None, torch.arange(8, device="cuda"), freqs)
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[0, 0, 3, 5] = want[0, 0, 3, 21] = want[0, 0, 4, 50] = True
    assert torch.equal(bad, want)


def test_training_through_attention_as_a_captured_step():
    """Rotary, then causal attention, forward and backward: relative positions
    alone count, and the step replays as a graph."""
    freqs, _ = rotary_frequencies(64, device="cuda")
    q, k, v = (_rand((1, h, 130, 64), BF16, i) for i, h in ((1, 4), (2, 2), (3, 2)))
    do = _rand((1, 4, 130, 64), BF16, 4)
    positions = torch.arange(130, device="cuda")

    def step(q, k, v):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        rq, rk = apply_rotary(*leaves[:2], positions, freqs)
        out = attention(rq, rk, leaves[2], causal=True, backend="triton")
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    want = step(q, k, v)
    ins = [t.clone() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*ins)
    for t in ins:
        t.zero_()
    graph.replay()
    for t, x in zip(ins, (q, k, v)):
        t.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    # dQ is summed by atomics in an order of its own
    for got, ref in zip(outs, want):
        assert (got.double() - ref.double()).abs().max() <= 2.0 ** -7 * ref.double().abs().max()
    # moved by 1000 positions: the same attention, to the roundings of q and k
    positions += 1000
    moved = step(q, k, v)
    assert (moved[0].double() - want[0].double()).abs().max() <= 2e-2 * (1 + want[0].double().abs().max())
    del graph
