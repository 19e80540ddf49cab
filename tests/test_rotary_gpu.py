"""Rotary positions, and keys and values written into pages, against their definitions in 64 bits."""
import math

import pytest
import torch

import dtb200
from paged_reference import Batch, turn

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _freq(pairs, base=10000.0):
    return [base ** (-j / pairs) for j in range(pairs)]


def _check(got, want, x, amplitude=1.0):
    # two f32 products of factors that are off by 2^-22 at most, their sum, one rounding to the result's type; |pair| bounds both
    size = amplitude * 2 * x.double().abs().amax(-1, keepdim=True)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -21 * size + torch.finfo(got.dtype).tiny
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max().item()


CASES = [  # shape, key heads, rotary, dtype, interleaved
    ((1, 1, 128), 1, 128, BF, False),
    ((5, 24, 128), 8, 64, BF, False),
    ((333, 3, 128), 0, 128, HF, True),
    ((2, 77, 4, 64), 2, 64, F32, False),
    ((3, 50, 5, 80), 5, 40, BF, True),
    ((40, 2, 96), 2, 20, HF, False),
    ((9, 7, 30), 1, 6, F32, True),
    ((9, 7, 31), 2, 10, BF, False),
    ((4, 2, 512), 1, 512, F32, False),
    ((2, 16, 200, 2), 1, 2, BF, True),
    ((1000, 1, 256), 1, 256, BF, False),
]


@pytest.mark.parametrize("shape,Hk,rotary,dtype,interleaved", CASES)
@pytest.mark.parametrize("transpose", [False, True])
def test_rotary(shape, Hk, rotary, dtype, interleaved, transpose):
    g = torch.Generator("cuda").manual_seed(rotary)
    q = torch.randn(shape, generator=g, device="cuda").to(dtype)
    k = torch.randn(*shape[:-2], Hk, shape[-1], generator=g, device="cuda").to(dtype) if Hk else None
    table = dtb200.make_rotary_table(rotary, layout="interleaved" if interleaved else "half")
    tokens = shape[-3]
    for positions in (torch.arange(tokens, device="cuda", dtype=torch.int32), torch.randint(0, 10 ** 7, (tokens,), generator=g, device="cuda"),
                      torch.rand(tokens, generator=g, device="cuda") * 1e4 - 5e3):
        got = dtb200.rotary(q, k, table=table, positions=positions, transpose=transpose)
        for x, y in zip((q, k), got if Hk else (got,)):
            _check(y, turn(x, positions, _freq(rotary // 2), interleaved, transpose=transpose), x)
            assert torch.equal(y[..., rotary:], x[..., rotary:])


def test_positions_of_each_sequence_axes_and_strides():
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(2, 6, 50, 128, generator=g, device="cuda").to(BF)             # [B, heads, tokens, dim]
    table = dtb200.make_rotary_table(128, axes=[16, 24, 24], layout="interleaved")
    positions = torch.randint(0, 500, (3, 2, 50), generator=g, device="cuda").transpose(1, 2).contiguous().transpose(1, 2)
    axis = [0] * 16 + [1] * 24 + [2] * 24
    freq = _freq(16) + _freq(24) + _freq(24)
    got = dtb200.rotary(x.transpose(1, 2), table=table, positions=positions)
    _check(got, turn(x.transpose(1, 2), positions, freq, True, axis=axis), x.transpose(1, 2))
    out = torch.empty_like(x)
    dtb200.rotary(x.transpose(1, 2), table=table, positions=positions[:, 0], out=out.transpose(1, 2))
    _check(out.transpose(1, 2), turn(x.transpose(1, 2), positions[:, 0, None].expand(3, 2, 50), freq, True, axis=axis), x.transpose(1, 2))
    odd = torch.randn(50, 3, 131, generator=g, device="cuda").to(BF)[:, :, 1:129]  # rows off 16-byte boundaries
    got = dtb200.rotary(odd, table=table, positions=positions[:, 0])
    _check(got, turn(odd, positions[:, 0], freq, True, axis=axis), odd)
    spread = torch.randn(50, 3, 128, 2, generator=g, device="cuda").to(BF)[..., 0]  # channels apart, and a broadcast
    got = dtb200.rotary(spread, spread[:, :1].expand(50, 4, 128), table=table, positions=positions[:, 0])
    _check(got[0], turn(spread, positions[:, 0], freq, True, axis=axis), spread)
    assert torch.equal(got[1][:, 3], got[0][:, 0])
    want = dtb200.rotary(x.transpose(1, 2), table=table, positions=positions)
    y = x.clone().transpose(1, 2)
    assert dtb200.rotary(y, table=table, positions=positions, out=y) is y and torch.equal(y, want)


def test_transpose_is_the_gradient():
    g = torch.Generator("cuda").manual_seed(0)
    x, up = (torch.randn(20, 3, 48, generator=g, device="cuda") for _ in range(2))
    table = dtb200.make_rotary_table(32, scaling="yarn", factor=4.0)
    positions = torch.arange(20, device="cuda") * 1000
    y = dtb200.rotary(x, table=table, positions=positions)
    back = dtb200.rotary(up, table=table, positions=positions, transpose=True)
    # <up, R x> = <R^T up, x>; the map is linear, so a difference quotient of any length is the derivative
    left, right = (up.double() * y.double()).sum(-1), (back.double() * x.double()).sum(-1)
    assert ((left - right).abs() <= 48 * 2.0 ** -20 * up.abs().amax() * x.abs().amax()).all()
    step = torch.randn(20, 3, 48, generator=g, device="cuda")
    moved = dtb200.rotary(x + step, table=table, positions=positions)
    assert ((((moved - y).double() * up.double()).sum() - (back.double() * step.double()).sum()).abs() <= 20 * 3 * 48 * 2.0 ** -19 * 16).all()


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 4.0), ("yarn", 16.0)])
def test_scaling(scaling, factor):
    n, base, original = 32, 10000.0, 4096
    table = dtb200.make_rotary_table(64, scaling=scaling, factor=factor, original_length=original)
    freq, gain = _freq(n), 1.0
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "ntk":
        freq = _freq(n, base * factor ** (n / (n - 1)))
        assert math.isclose(freq[-1] * factor, _freq(n)[-1]) and freq[0] == 1.0
    else:
        gain = 0.1 * math.log(factor) + 1
        at = [n * math.log(original / (t * 2 * math.pi)) / math.log(base) for t in (32.0, 1.0)]
        low, high = math.floor(at[0]), math.ceil(at[1])
        keep = [1 - min(max((j - low) / (high - low), 0), 1) for j in range(n)]
        freq = [f * k + f / factor * (1 - k) for f, k in zip(freq, keep)]
    x = torch.randn(100, 2, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    positions = torch.arange(100, device="cuda") * 997
    _check(dtb200.rotary(x, table=table, positions=positions), turn(x, positions, freq, False, gain), x, gain)


@pytest.mark.parametrize("dtype,layout,page,D,rope", [(BF, "hnd", 16, 128, "half"), (HF, "nhd", 32, 64, "interleaved"), (BF, "nhd", 5, 40, None),
                                                      (BF, "hnd", 1, 128, "interleaved")])
def test_append(dtype, layout, page, D, rope):
    new, kv = [1, 0, 40, 7, 12, 3], [33, 10, 60, 7, 9, 0]        # sequence 4 counts fewer tokens than it brings, 5 none
    batch = Batch(new, kv, Hkv=3, D=D, page=page, dtype=dtype, layout=layout, tail=4, extra_width=0)
    g = torch.Generator("cuda").manual_seed(0)
    q, k, v = (torch.randn(batch.tokens, h, D, generator=g, device="cuda").to(dtype) for h in (6, 3, 3))
    table = dtb200.make_rotary_table(D // 2, layout=rope) if rope else None
    kc, vc = batch.key_cache.clone(), batch.value_cache.clone()
    assert kc.stride() == batch.key_cache.stride()
    out = torch.full_like(q, 5.0)
    got = dtb200.paged_append_(kc, vc, k, v, table=table, query=q, query_out=out, **batch.where)
    assert got is out and (out[sum(new):] == 5.0).all()
    freq = _freq(D // 4)
    want_k, want_v = batch.key_cache.double(), batch.value_cache.double()
    for b, n in enumerate(new):
        slots = torch.arange(kv[b] - n, kv[b], device="cuda")
        rows = batch.rows(b)
        qt, kt = (turn(x[rows], slots, freq, rope == "interleaved") if rope else x[rows].double() for x in (q, k))
        _check(out[rows], qt, q[rows])
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                p, r = int(batch.page_table[b, s // page]), s % page
                _check(kc[p, :, r], kt[i], k[rows][i])
                assert torch.equal(vc[p, :, r], v[rows][i])
                want_k[p, :, r], want_v[p, :, r] = kc[p, :, r].double(), vc[p, :, r].double()
    assert torch.equal(kc.double().nan_to_num(99.0), want_k.nan_to_num(99.0))          # nothing else is written
    assert torch.equal(vc.double().nan_to_num(99.0), want_v.nan_to_num(99.0))
    kc2, vc2 = batch.key_cache.clone(), batch.value_cache.clone()
    assert dtb200.paged_append_(kc2, vc2, k, v, table=table, **batch.where) is None
    assert torch.equal(kc2.nan_to_num(99.0), kc.nan_to_num(99.0))


def test_append_takes_positions_and_drops_what_has_no_page():
    batch = Batch([3, 2], [40, 20], Hkv=2, D=128, page=16, extra_width=0)
    g = torch.Generator("cuda").manual_seed(0)
    q, k, v = (torch.randn(5, h, 128, generator=g, device="cuda").to(BF) for h in (4, 2, 2))
    table = dtb200.make_rotary_table(128, axes=[16, 24, 24])
    positions = torch.randint(0, 1000, (3, 5), generator=g, device="cuda")
    batch.page_table[0, 2] = -1
    batch.page_table[1, 1] = batch.pages
    kc, vc = batch.key_cache.clone(), batch.value_cache.clone()
    got = dtb200.paged_append_(kc, vc, k, v, table=table, positions=positions, query=q, **batch.where)
    assert torch.equal(got, dtb200.rotary(q, table=table, positions=positions))
    assert torch.equal(kc.nan_to_num(9.0), batch.key_cache.nan_to_num(9.0)) and torch.equal(vc.nan_to_num(9.0), batch.value_cache.nan_to_num(9.0))
    batch.kv_len.fill_(10 ** 9)                                  # past the table
    dtb200.paged_append_(kc, vc, k, v, **batch.where)
    assert torch.equal(kc.nan_to_num(9.0), batch.key_cache.nan_to_num(9.0))
    empty = torch.empty(0, 2, 16, 128, dtype=BF, device="cuda")
    got = dtb200.paged_append_(empty, empty.clone(), k, v, table=table, positions=positions, query=q, **batch.where)
    assert torch.equal(got, dtb200.rotary(q, table=table, positions=positions))


@pytest.mark.parametrize("starts", [[0, 5, 3, 9], [-4, 2, 100, 6], [9, 9, 9, 9]])
def test_append_with_starts_out_of_order_stays_in_bounds(starts):
    batch = Batch([3, 3, 3], [40, 50, 60], Hkv=2, D=128, page=16)
    batch.query_start.copy_(torch.tensor(starts))
    k = torch.randn(9, 2, 128, device="cuda").to(BF)
    dtb200.paged_append_(batch.key_cache, batch.value_cache, k, k, query=k, **batch.where)
    torch.cuda.synchronize()


def test_rotary_under_capture():
    table = dtb200.make_rotary_table(64)
    q, k = torch.randn(7, 4, 128, device="cuda").to(BF), torch.randn(7, 2, 128, device="cuda").to(BF)
    positions = torch.arange(7, device="cuda", dtype=torch.int32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = dtb200.rotary(q, k, table=table, positions=positions)
    positions += 1000
    graph.replay()
    want = dtb200.rotary(q, k, table=table, positions=positions)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
