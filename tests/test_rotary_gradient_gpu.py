"""Gradients through rotary: the transposed map of what comes back, against the formula in 64 bits and against differences."""
import pytest
import torch

import dtb200
from paged_reference import turn
from test_rotary_gpu import _check, _freq

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("shape, Hk, rotary, dtype, interleaved, scaling", [
    ((1, 1, 128), 1, 128, F32, False, None), ((77, 6, 128), 2, 64, BF, False, "yarn"), ((2, 50, 4, 80), 4, 40, HF, True, None), ((33, 3, 30), 1, 6, F32, True, "ntk"),
])
def test_gradients(shape, Hk, rotary, dtype, interleaved, scaling):
    g = torch.Generator("cuda").manual_seed(0)
    table = dtb200.make_rotary_table(rotary, layout="interleaved" if interleaved else "half", scaling=scaling, factor=4.0)
    freq = (table.turns * 6.283185307179586).tolist()
    positions = torch.randint(0, 5000, (shape[-3],), generator=g, device="cuda")

    def normal(heads):
        return torch.randn(*shape[:-2], heads, shape[-1], generator=g, device="cuda").to(dtype)

    q, k, dq, dk = normal(shape[-2]).requires_grad_(), normal(Hk).requires_grad_(), normal(shape[-2]), normal(Hk)
    a, b = dtb200.rotary(q, k, table=table, positions=positions)
    with torch.no_grad():
        plain = dtb200.rotary(q, k, table=table, positions=positions)
    assert torch.equal(a, plain[0]) and torch.equal(b, plain[1])
    got = torch.autograd.grad((a, b), (q, k), (dq, dk), retain_graph=True)
    for x, up in zip(got, (dq, dk)):
        _check(x, turn(up, positions, freq, interleaved, table.amplitude, transpose=True), up, table.amplitude)
    only, = torch.autograd.grad(b, k, dk, retain_graph=True)
    assert torch.equal(only, got[1])
    # a sum's gradient comes as one number in all places
    ones, = torch.autograd.grad(a.sum(), q)
    _check(ones, turn(torch.ones_like(q), positions, freq, interleaved, table.amplitude, transpose=True), torch.ones_like(q), table.amplitude)


def test_gradient_is_the_difference():
    """The map is linear, so the difference quotient over any step is the derivative, but for f32's products: of each of the 4200
    numbers 2^-21 of its pair's size, which stays below 16."""
    g = torch.Generator("cuda").manual_seed(1)
    table = dtb200.make_rotary_table(48, axes=[8, 8, 8])
    positions = torch.randint(0, 900, (3, 25), generator=g, device="cuda")
    x, step, up = (torch.randn(25, 3, 56, generator=g, device="cuda") for _ in range(3))
    x.requires_grad_()
    y = dtb200.rotary(x, table=table, positions=positions)
    grad, = torch.autograd.grad(y, x, up)
    with torch.no_grad():
        moved = dtb200.rotary(x + step, table=table, positions=positions)
    left, right = ((moved - y).double() * up.double()).sum(), (grad.double() * step.double()).sum()
    assert (left - right).abs() <= 4200 * 2.0 ** -20 * 16


def test_gradient_of_the_gradient():
    table = dtb200.make_rotary_table(32)
    positions = torch.arange(9, device="cuda")
    x, up, w = (torch.randn(9, 2, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) for i in range(3))
    x.requires_grad_(), up.requires_grad_()
    y = dtb200.rotary(x, table=table, positions=positions)
    grad, = torch.autograd.grad(y, x, up, create_graph=True)
    again, = torch.autograd.grad(grad, up, w)
    assert torch.equal(again, dtb200.rotary(w, table=table, positions=positions))
