"""Rotary positions, alone and with the write into the paged cache, against 64-bit numbers.

Bound: the result's rounding (half a step), and in front of it the cosine's and sine's error (an angle within one turn rounded to
32 bits, 2^-24 of a turn's pi, and two units in the last place of the functions: 2^-21 together) and three fp32 roundings, all relative to the
pair's absolute values."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import tpu_mlir_b200._lib as L  # noqa: E402
from decode_model import TORCH, frequencies, rotate, smallest, step  # noqa: E402
from decode_util import DT, Cache, f64, i32, rope_plan  # noqa: E402

SCALED = [("none", 1.0, 0, 0, 0), ("linear", 4.0, 0, 0, 0), ("stretched", 8.0, 0, 0, 0), ("yarn", 16.0, 4096.0, 1.0, 32.0), ("banded", 8.0, 8192.0, 1.0, 4.0)]


def close(y, want, size, dtype):
    assert bool(np.isfinite(y).all())
    bound = step(dtype) * np.abs(want) + (1 + step(dtype)) * 2.0**-21 * size + smallest(dtype)
    worst = (np.abs(y - want) - bound).max() if y.size else 0
    assert worst <= 0, worst


def call(plan, x, y, positions, dtype, stream=None):
    L.check(L.lib().b200q_rope_dev(C.byref(plan), x.data_ptr(), y.data_ptr(), positions.data_ptr(), x.shape[0], x.shape[1], x.stride(0), x.stride(1),
                                   y.stride(0), y.stride(1), DT[dtype], stream))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (80, 32), (64, 22), (256, 256), (96, 96), (6, 4), (8, 2), (64, 0), (130, 130)])
@pytest.mark.parametrize("rows,heads,dtype", [(1, 1, "bf16"), (1, 40, "f16"), (3, 7, "f16"), (1201, 5, "bf16")])
def test_rope(interleaved, dim, rotary, rows, heads, dtype):
    g = torch.Generator().manual_seed(rows + dim + rotary)
    x = torch.randn((rows, heads, dim), generator=g).to(TORCH[dtype]).cuda()
    positions = torch.randint(0, 131072, (rows,), generator=g, dtype=torch.int32).cuda()
    y = torch.full_like(x, float("nan"))
    call(rope_plan(dim, rotary, interleaved), x, y, positions, dtype)
    f, m = frequencies(rotary, 10000.0) if rotary else ([], 1.0)
    want, size = rotate(f64(x), positions.tolist(), f, m, interleaved)
    close(f64(y), want, size, dtype)
    assert torch.equal(y[..., rotary:], x[..., rotary:])
    call(rope_plan(dim, rotary, interleaved), x, x, positions, dtype)      # in place
    assert torch.equal(x.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("kind,factor,span,low,high", SCALED)
@pytest.mark.parametrize("base", [10000.0, 1000000.0])
def test_rope_scaled(kind, factor, span, low, high, base):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((50, 2, 128), generator=g).to(torch.float16).cuda()
    positions = i32([0, 1, 2**31 - 1, 2**24 + 1, -5] + [int(p) for p in torch.randint(0, 1 << 20, (45,), generator=g)])
    y = torch.empty_like(x)
    call(rope_plan(128, 128, False, base, kind, factor, span, low, high), x, y, positions, "f16")
    f, m = frequencies(128, base, kind, factor, span, low, high)
    want, size = rotate(f64(x), positions.tolist(), f, m, False)
    # a position of 2^31 times a frequency carries 2^31 * 2^-53 of relative rounding: 2^-22 of a radian for each of two 64-bit roundings
    size = size * np.where(np.abs(np.array(positions.tolist())) > 2**24, 4.0, 1.0)[:, None, None]
    close(f64(y), want, size, "f16")


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides_and_alignment(shift, interleaved):
    """Heads outside rows, gaps between heads, rows that start off 16 bytes: only the elements themselves are written."""
    g = torch.Generator().manual_seed(shift)
    raw = torch.randn((6, 33, 80), generator=g).to(torch.bfloat16).cuda()
    x = raw.permute(1, 0, 2)[:, :, shift:shift + 64]
    back = torch.full((33, 6, 77), 7.0, dtype=torch.bfloat16, device="cuda")
    y = back[:, 1:, :64][:, :5]
    positions = i32(list(range(33)))
    call(rope_plan(64, 48, interleaved), x[:, :5], y, positions, "bf16")
    f, m = frequencies(48, 10000.0)
    want, size = rotate(f64(x[:, :5]), range(33), f, m, interleaved)
    close(f64(y), want, size, "bf16")
    assert bool((back[:, 0] == 7).all()) and bool((back[:, 1:, 64:] == 7).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout,page_size,dim,rotary,dtype", [("nhd", 16, 128, 128, "bf16"), ("hnd", 5, 80, 20, "f16"), ("nhd", 1, 64, 64, "f16"), ("hnd", 64, 256, 128, "bf16")])
@pytest.mark.parametrize("counts", [[1], [1, 0, 1, 1], [0, 37, 5, 0, 64, 1, 200], [0, 0]])
@pytest.mark.parametrize("tree", [False, True])
def test_append(interleaved, layout, page_size, dim, rotary, dtype, counts, tree):
    rng = np.random.default_rng(dim + len(counts))
    n, hq, hk, layers = len(counts), 6, 3, 2
    lengths = [int(x) for x in rng.integers(0, 90, n)]
    width = -(-300 // page_size)
    c = Cache(sequences=n, width=width, pages=n * width + 2, page_size=page_size, heads=hk, dim=dim, layers=layers, dtype=dtype, layout=layout, pad=8, seed=n)
    assert c.model.reserve([x + t for x, t in zip(lengths, counts)]) == 0
    c.model.length = lengths
    c.up()
    before, rows, after = 3, sum(counts), 4          # rows in front of the first sequence and behind the last
    start = np.cumsum([before] + counts).tolist()
    total = before + rows + after
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn((total, hq + 2 * hk, dim), generator=g).to(TORCH[dtype]).cuda()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    out = torch.full((total, hq, dim), 5.0, dtype=TORCH[dtype], device="cuda")
    where = [lengths[s] + i for s in range(n) for i in range(counts[s])]
    positions = [0] * before + [int(p) for p in rng.integers(0, 9000, rows)] + [0] * after if tree else None
    want_k, want_v, old_k, old_v = f64(c.k), c.v.clone(), c.k.clone(), c.v.clone()
    c.append(rope_plan(dim, rotary, interleaved), q, out, k, v, i32(start), None if positions is None else i32(positions), layer=1)
    torch.cuda.synchronize()
    turn = positions[before:before + rows] if tree else where
    f, m = frequencies(rotary, 10000.0)
    inside = slice(before, before + rows)
    want, size = rotate(f64(q[inside]), turn, f, m, interleaved)
    close(f64(out[inside]), want, size, dtype)
    assert bool((out[:before] == 5).all()) and bool((out[before + rows:] == 5).all())
    wk, size = rotate(f64(k[inside]), turn, f, m, interleaved)
    written = np.zeros(c.k.shape[:4], bool)
    at = 0
    for s in range(n):
        for i in range(counts[s]):
            p, t = c.model.place(s, lengths[s] + i)
            written[1, p, t] = True
            close(f64(c.k[1, p, t]), wk[at], size[at], dtype)
            want_v[1, p, t] = v[before + at]
            at += 1
    assert torch.equal(c.v, want_v)
    untouched = torch.from_numpy(~written).cuda()
    assert torch.equal(c.k[untouched], old_k[untouched])


def test_append_where_there_is_no_page():
    """Positions past the held pages, past the table and in a page that is none: the queries are rotated, nothing is written."""
    c = Cache(sequences=4, width=2, pages=4, page_size=4, heads=1, dim=64)
    c.model.table = [[0, -1], [1, 7], [2, 3], [-9, 2**31 - 1]]
    c.model.length, c.model.held = [3, 3, 7, 2**31 - 1], [2, 2, 2, 2]
    c.up()
    q = torch.randn((8, 2, 64)).to(torch.bfloat16).cuda()
    k = torch.randn((8, 1, 64)).to(torch.bfloat16).cuda()
    out, old_k, old_v = torch.zeros_like(q), c.k.clone(), c.v.clone()
    c.append(rope_plan(64, 64, True), q, out, k, k, i32([0, 2, 4, 6, 8]), i32([1] * 8))
    torch.cuda.synchronize()
    f, m = frequencies(64, 10000.0)
    want, size = rotate(f64(q), [1] * 8, f, m, True)
    close(f64(out), want, size, "bf16")
    changed = [(s, 0) for s in (0, 1, 2)]            # only the first row of these has a place
    old_v[0, 0, 3], old_v[0, 1, 3], old_v[0, 3, 3] = k[0], k[2], k[4]
    assert torch.equal(c.v, old_v) and len(changed) == 3
    assert (c.k != old_k).flatten(3).any(-1).sum() == 3


def test_rope_infinities_stay_in_their_pair():
    x = torch.randn((2, 1, 64)).to(torch.bfloat16).cuda()
    x[0, 0, 3] = float("inf")
    x[1, 0, 40] = float("nan")
    y = torch.empty_like(x)
    call(rope_plan(64, 64, False), x, y, i32([7, 9]), "bf16")
    bad = (~torch.isfinite(y)).nonzero().tolist()
    assert bad == [[0, 0, 3], [0, 0, 35], [1, 0, 8], [1, 0, 40]]
