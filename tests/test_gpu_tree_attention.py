"""Attention of drafted trees over the paged cache against 64-bit numbers, with bounds derived in decode_model.attention."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from decode_model import TORCH, attention  # noqa: E402
from decode_util import Cache, f64, i32, random_tree, words  # noqa: E402


def setup(counts, lengths, *, page_size=16, heads=2, group=2, dim=64, dtype="bf16", layout="nhd", layers=1, seed=0, tree=True, before=0, after=0, spare=3,
          size=1.0):
    rng = np.random.default_rng(seed)
    n = len(counts)
    width = max(1, -(-max(a + b for a, b in zip(counts, lengths)) // page_size)) + 1
    c = Cache(sequences=n, width=width, pages=sum(-(-(a + b) // page_size) for a, b in zip(counts, lengths)) + spare, page_size=page_size, heads=heads, dim=dim,
              layers=layers, dtype=dtype, layout=layout, pad=8, seed=seed)
    assert c.model.reserve([a + b for a, b in zip(counts, lengths)]) == 0
    order = rng.permutation(len(c.model.refcount))
    c.model.table = [[int(order[p]) if p >= 0 else -1 for p in row] for row in c.model.table]
    c.model.length = list(lengths)
    c.up()
    rows = before + sum(counts) + after
    start = np.cumsum([before] + list(counts)).tolist()
    g = torch.Generator().manual_seed(seed + 1)
    q = (size * torch.randn((rows, heads * group, dim), generator=g)).to(TORCH[dtype]).cuda()
    bits = None
    if tree:
        most = max(max(counts), 1)
        bits = np.zeros((rows, most), bool)
        for s, t in enumerate(counts):
            bits[start[s]:start[s] + t, :t] = random_tree(rng, t)
        # what stands in the mask past a sequence's own nodes is not looked at
        bits[:, :] |= np.array([[m >= counts[max(0, np.searchsorted(start, r, side="right") - 1)] if before <= r < rows - after else True for m in range(most)]
                                for r in range(rows)], bool).reshape(rows, most)
    return c, q, start, bits


def check(c, q, start, bits, scale=0.125, layer=0):
    out = torch.full_like(q, 9.0)
    space = c.attend(q, out, i32(start), None if bits is None else words(bits), scale=scale, layer=layer)
    torch.cuda.synchronize()
    assert bool((space[-64:] == 0xA5).all()), "bytes behind the workspace were written"
    rows = [(start[s], start[s + 1]) for s in range(len(start) - 1)]
    use = None
    if bits is not None:
        use = bits.copy()
        for s, (b, e) in enumerate(rows):
            use[max(b, 0):max(e, 0), max(e - b, 0):] = False
    want, bound = attention(f64(q), c.model, f64(c.k[layer]), f64(c.v[layer]), start, use, scale, c.dtype)
    got = f64(out)
    outside = np.array([not any(b <= r < e for b, e in rows) for r in range(q.shape[0])])
    assert (got[outside] == 9).all(), "a row outside every sequence was written"
    w, g, b = want[~outside], got[~outside], bound[~outside]
    nan = np.isnan(w)
    assert (np.isnan(g) == nan).all()
    inf = np.isinf(w)
    assert (g[inf] == w[inf]).all()
    ok = ~nan & ~inf
    over = np.abs(g[ok] - w[ok]) - b[ok]
    assert over.size == 0 or over.max() <= 0, (over.max(), b[ok].max())
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 63, 64, 65, 127, 128, 500, 1100])
def test_one_token(length, dtype):
    check(*setup([1], [length], dtype=dtype, tree=False, seed=length))


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 16), (3, 2), (2, 7), (8, 4), (1, 33), (1, 71), (2, 5)])
@pytest.mark.parametrize("dim,page_size,layout", [(128, 16, "nhd"), (64, 24, "hnd"), (80, 1, "nhd"), (96, 7, "hnd"), (256, 64, "nhd"), (8, 16, "hnd"), (136, 128, "hnd")])
def test_heads_and_pages(heads, group, dim, page_size, layout):
    check(*setup([1, 3, 2], [130, 0, 61], heads=heads, group=group, dim=dim, page_size=page_size, layout=layout, seed=dim + group, dtype="f16" if dim % 3 else "bf16"),
          scale=dim ** -0.5)


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("counts,lengths", [([1, 0, 5, 31, 2], [70, 40, 0, 333, 129]), ([64], [200]), ([65, 1], [63, 64]), ([130, 33], [0, 10]), ([0, 0, 3], [5, 0, 700]),
                                            ([2] * 40, [11 * i for i in range(40)])])
@pytest.mark.parametrize("group", [1, 4])
def test_trees_and_chains(tree, counts, lengths, group):
    check(*setup(counts, lengths, tree=tree, group=group, before=2, after=3, layers=2, page_size=8, seed=sum(counts)), layer=1)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1], [7], [40]])
def test_split_contexts(dim, counts):
    """One long context, cut into parts over the whole GPU."""
    check(*setup(counts, [5000], dim=dim, heads=1, group=3, page_size=32, seed=dim), scale=dim ** -0.5)


def test_rows_that_see_nothing_are_zeros():
    c, q, start, bits = setup([3, 2], [0, 20], seed=4)
    bits[:] = False
    bits[1, 0] = True
    out = check(c, q, start, bits)
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all()) and bool((out[1] != 0).any()) and bool((out[3] != 0).any())


def test_masks_of_any_width_and_with_all_bits():
    c, q, start, bits = setup([5], [9], seed=6)
    check(c, q, start, np.zeros((5, 5), bool))
    check(c, q, start, np.ones((5, 5), bool))       # a node may see later ones: the mask alone counts
    check(c, q, start, np.ones((5, 3), bool))       # fewer bits than nodes: the others are not seen
    check(c, q, start, np.ones((5, 200), bool))


def test_no_page_no_contribution():
    """Pages that the pool does not have, in the middle of a context, at its end, everywhere."""
    for holes in ([1], [0, 3], [0, 1, 2, 3, 4]):
        c, q, start, bits = setup([4, 2], [70, 40], page_size=16, seed=8)
        for h in holes:
            c.model.table[0][h] = [-1, 10**6, -2**31][h % 3]
        c.up()
        check(c, q, start, bits)
    c, q, start, bits = setup([4, 2], [70, 40], page_size=16, seed=8)
    c.model.length = [10**6, 2**31 - 1]             # lengths that the table does not hold
    c.up()
    out = torch.full_like(q, 9.0)
    c.attend(q, out, i32(start), words(bits))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group,counts", [(1, [9]), (4, [9, 40]), (2, [16])])
def test_what_is_not_seen_does_not_matter(dtype, group, counts):
    """Infinities and NaN in drafted nodes that some rows do not see, in slots past the last node and in pages of others."""
    c, q, start, bits = setup(counts, [61] * len(counts), group=group, dtype=dtype, dim=128, seed=12, spare=6)
    held = np.zeros((len(c.model.refcount), 16), bool)
    for s, t in enumerate(counts):
        for p in range(61 + t):
            held[c.model.place(s, p)] = True
    free = torch.from_numpy(~held).cuda()
    for t in (c.k, c.v):
        for bad in (float("nan"), float("inf")):
            t[0][free] = bad
    plain = check(c, q, start, bits)
    assert bool(torch.isfinite(plain).all())
    for s, t in enumerate(counts):
        for node, (kbad, vbad) in {1: (float("nan"), 1.0), 3: (1.0, float("nan")), 5: (1.0, float("inf")), 6: (1.0, -float("inf")), 8: (float("inf"), float("nan"))}.items():
            p, slot = c.model.place(s, 61 + node)
            c.k[0, p, slot, :, 3] = kbad
            c.v[0, p, slot, :, 5] = vbad
            if node == 5:
                c.v[0, p, slot, :, 70:75] = vbad
    out = check(c, q, start, bits)
    for s, t in enumerate(counts):
        clean = [r for r in range(start[s], start[s] + t) if not any(bits[r, m] for m in (1, 3, 5, 6, 8))]
        assert clean and torch.equal(out[clean], plain[clean])


def test_large_scores():
    """Weights that underflow, and a maximum that moves from unit to unit."""
    c, q, start, bits = setup([3], [900], size=30.0, seed=2)
    c.k *= torch.linspace(0.1, 3, c.k.shape[1], device="cuda").to(c.k.dtype)[None, :, None, None, None]
    check(c, q, start, bits, scale=1.0)


def test_strides():
    """Queries inside a wider row, heads outside rows in the output."""
    c, q, start, bits = setup([4, 1], [33, 90], heads=2, group=3, seed=3)
    wide = torch.zeros((q.shape[0], 10, 80), dtype=q.dtype, device="cuda")
    wide[:, 2:8, 8:72] = q
    view = wide[:, 2:8, 8:72]
    back = torch.full((6, q.shape[0] + 2, 72), 9.0, dtype=q.dtype, device="cuda")
    out = back.permute(1, 0, 2)[1:-1, :, :64]
    want = torch.empty_like(q)
    c.attend(q, want, i32(start), words(bits))
    c.attend(view, out, i32(start), words(bits))
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert bool((back[:, 0] == 9).all()) and bool((back[:, -1] == 9).all()) and bool((back[:, :, 64:] == 9).all())


def test_row_starts_that_are_not_ascending_stay_inside():
    c, q, start, bits = setup([3, 4, 2], [10, 40, 80], seed=5)
    out = torch.full_like(q, 9.0)
    for wrong in ([0, 100, -3, 9], [5, 2, 9, 4], [-4, 3, 7, 9], [2**31 - 1, -2**31, 9, 9]):
        c.attend(q, out, i32(wrong), words(bits))
    torch.cuda.synchronize()


def test_same_result_every_time_and_on_two_streams():
    a = setup([9, 20, 1], [3000, 50, 700], group=4, dim=128, seed=31)
    b = setup([17], [1500], group=2, dim=128, seed=32)
    outs = []
    for c, q, start, bits in (a, b):
        o = torch.empty_like(q)
        c.attend(q, o, i32(start), words(bits))
        outs.append(o)
    torch.cuda.synchronize()
    again = [torch.empty_like(o) for o in outs]
    streams = [torch.cuda.Stream() for _ in outs]
    held = [(i32(start), words(bits), c.workspace(q.shape[1])) for c, q, start, bits in (a, b)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, q, start, bits), o, s, (st, w, space) in zip((a, b), again, streams, held):
            c.attend(q, o, st, w, stream=s.cuda_stream, space=space)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, again))


def test_captured_lengths_may_change():
    c, q, start, bits = setup([6], [400], group=4, dim=128, seed=40)
    st, w, space, out = i32(start), words(bits), c.workspace(q.shape[1]), torch.zeros_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.attend(q, out, st, w, stream=side.cuda_stream, space=space)
    for length in (400, 0, 64, 7, 399):
        c.length.fill_(length)
        c.model.length = [length]
        graph.replay()
        want = check(c, q, start, bits)
        assert torch.equal(out, want)


def test_many_sequences():
    rng = np.random.default_rng(1)
    n = 1024
    check(*setup([int(x) for x in rng.integers(0, 3, n)], [int(x) for x in rng.integers(0, 40, n)], heads=1, group=1, dim=16, seed=50))


@pytest.mark.parametrize("group,counts,lengths", [(1, [1, 5], [70, 3000]), (4, [6, 2], [2000, 0]), (4, [20, 9], [1500, 64]), (4, [64], [1100])])
def test_in_place(group, counts, lengths):
    c, q, start, bits = setup(counts, lengths, group=group, dim=128, seed=60)
    out = torch.empty_like(q)
    c.attend(q, out, i32(start), words(bits))
    c.attend(q, q, i32(start), words(bits))
    torch.cuda.synchronize()
    assert torch.equal(q, out)


@pytest.mark.parametrize("nodes,dim", [(1, 64), (6, 64), (12, 64), (40, 64), (1, 256)])
def test_many_small_weights_beside_a_large_one(nodes, dim):
    """8000 weights of 2^-25.5, each less than half the smallest half precision number, beside one of 1 whose value is 0: together they are
    the result.  All sequences read the same pages; there are enough of them that most contexts are not cut."""
    n, length, ps, group = 600, 8000, 16, 4
    pages = length // ps
    c = Cache(sequences=n, width=pages + 4, pages=pages, page_size=ps, heads=1, dim=dim, dtype="f16", seed=70)
    c.model.table = [list(range(pages)) + [-1] * 4 for _ in range(n)]      # the nodes have no pages: only the context is seen
    c.model.length, c.model.held = [length] * n, [pages] * n
    c.up()
    c.k.zero_()
    c.v.fill_(1.0)
    c.k[0, 0, 0, 0, 0] = 4.0
    c.v[0, 0, 0].zero_()
    q = torch.zeros((n * nodes, group, dim), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 25.5 * np.log(2) / 4
    out = torch.full_like(q, 9.0)
    c.attend(q, out, torch.arange(0, (n + 1) * nodes, nodes, dtype=torch.int32, device="cuda"), None, scale=1.0)
    torch.cuda.synchronize()
    w = np.exp(-4.0 * float(q[0, 0, 0]))
    want = (length - 1) * w / (1 + (length - 1) * w)
    # weights are multiples of 2^-24 / 2^7: half of that each; the score in fp32 (|score| 2^-22); the sum's 2^-23 a term; the result's rounding
    bound = (length - 1) * 2.0**-32 + want * (17.7 * 2.0**-22 + length * 2.0**-23 + 2.0**-11)
    assert float((out.double() - want).abs().max()) <= bound, (float(out.min()), float(out.max()), want, bound)


@pytest.mark.parametrize("group", [1, 40])
def test_positions_up_to_the_last_of_31_bits(group):
    """A context whose last unit starts at 2^31 - 64 (of two pages: one of them stands in the table over and over).  With queries of zero
    all weights are 1 and the sums are whole numbers below 2^24 in every block."""
    ps, width = 16, 2**27 - 1
    c = Cache(sequences=1, width=1, pages=2, page_size=ps, heads=1, dim=64, seed=80)
    c.model.length, c.model.held = [width * ps - 3], [width]
    c.up()
    c.table = torch.zeros((1, width), dtype=torch.int32, device="cuda")
    c.table[0, -1] = 1
    c.v.zero_()
    c.v[0, 0, :, 0, 0] = 1.0
    c.v[0, 0, 0, 0, 1] = 8.0
    c.v[0, 1, -1, 0, :] = float("nan")        # the last node: only itself sees it
    q = torch.zeros((3, group, 64), dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 9.0)
    c.attend(q, out, i32([0, 3]), None, scale=1.0)
    torch.cuda.synchronize()
    assert bool(out[2].isnan().all())
    # 16 of 2^31 positions have other values than those below: nothing beside half a step of bf16
    assert bool((out[:2, :, 0] == 1.0).all()) and bool((out[:2, :, 1] == 0.5).all()) and bool((out[:2, :, 2:] == 0).all())


@pytest.mark.parametrize("dim,group,counts,lengths", [(64, 4, [700, 3, 129], [0, 500, 70]), (128, 1, [300, 513], [0, 63]), (64, 7, [200, 90], [130, 0]),
                                                      (256, 2, [150], [40]), (64, 1, [1], [0]), (16, 3, [17, 40, 11], [65, 0, 64]), (128, 40, [30], [100])])
def test_long_chains(dim, group, counts, lengths):
    """Chains of many row tiles, each of which ends at its own last node."""
    check(*setup(counts, lengths, dim=dim, group=group, heads=2, tree=False, before=1, after=2, seed=dim + group), scale=dim ** -0.5)


def test_long_chain_without_all_of_its_pages():
    c, q, start, _ = setup([400], [100], dim=64, group=4, tree=False, seed=90)
    c.model.held[0] = 20                            # 320 positions: later nodes see no more than these
    c.model.table[0][9] = -1
    c.up()
    check(c, q, start, None)


def test_what_is_not_seen_in_a_long_chain():
    """Infinities and NaN that only later nodes of a chain see, in the same unit and in later ones."""
    c, q, start, _ = setup([300], [50], dim=64, group=4, tree=False, seed=91)
    plain = check(c, q, start, None)
    for node, bad in ((40, float("nan")), (130, float("inf")), (131, -float("inf"))):
        p, slot = c.model.place(0, 50 + node)
        c.v[0, p, slot, :, 5] = bad
        c.k[0, p, slot, :, 7] = bad if node == 40 else 1.0
    out = check(c, q, start, None)
    assert torch.equal(out[:40], plain[:40]) and not bool(torch.isfinite(out[40:]).all())
