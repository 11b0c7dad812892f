"""What the decoding operators' contract says for inputs at its edge: values that are not finite in stages that are filled again, lengths and
pages that the pool does not hold, scores past fp32's range, rows that no sequence names."""
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from decode_model import TORCH, attention, frequencies, rotate, smallest, step  # noqa: E402
from decode_util import Cache, f64, i32, random_tree, rope_plan, words  # noqa: E402
from test_gpu_tree_attention import setup  # noqa: E402


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nodes,group,dim", [(4, 4, 64), (4, 4, 128), (8, 4, 64), (8, 4, 128), (4, 4, 256), (24, 2, 128)])
def test_stages_that_are_filled_again_after_infinities_were_taken_out(nodes, group, dim, dtype):
    """Enough short contexts that every block goes through more units than it has stages, each context's last unit with infinite and NaN values
    of nodes that nobody sees: the values that the same stage holds next are the right ones, every time."""
    n, heads, page_size = 320, 2, 16
    rng = np.random.default_rng(nodes + dim)
    lengths = [int(x) for x in rng.integers(20, 150, n)]
    width = -(-(150 + nodes) // page_size)
    c = Cache(sequences=n, width=width, pages=n * width, page_size=page_size, heads=heads, dim=dim, dtype=dtype, seed=nodes)
    assert c.model.reserve([x + nodes for x in lengths]) == 0
    c.model.length = lengths
    c.up()
    hidden = nodes - 2                                 # two nodes that nobody sees: values of NaN and of both infinities
    bits = np.concatenate([random_tree(rng, nodes) for _ in range(n)])
    bits[:, hidden:] = False
    places = torch.tensor([c.model.place(s, lengths[s] + hidden + i) for s in range(n) for i in range(2)], device="cuda").T
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").repeat(dim)[:dim].to(TORCH[dtype])
    c.v[0, places[0], places[1]] = bad
    q = torch.randn((n * nodes, heads * group, dim), generator=torch.Generator().manual_seed(dim)).to(TORCH[dtype]).cuda()
    start, mask, space = i32(list(range(0, (n + 1) * nodes, nodes))), words(bits), c.workspace(heads * group)
    out, again = torch.empty_like(q), torch.empty_like(q)
    c.attend(q, out, start, mask, scale=dim ** -0.5, space=space)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all())
    for _ in range(10):
        c.attend(q, again, start, mask, scale=dim ** -0.5, space=space)
        torch.cuda.synchronize()
        assert torch.equal(out, again)
    some = list(range(0, n, 16))                       # against 64-bit numbers: every sixteenth sequence, the others left without rows
    c.model.table, c.model.length, c.model.held = ([m[s] for s in some] for m in (c.model.table, c.model.length, c.model.held))
    rows = np.concatenate([np.arange(s * nodes, (s + 1) * nodes) for s in some])
    want, bound = attention(f64(q[rows]), c.model, f64(c.k[0]), f64(c.v[0]), list(range(0, len(rows) + 1, nodes)), bits[rows], dim ** -0.5, dtype)
    assert (np.abs(f64(out[rows]) - want) <= bound).all()


@pytest.mark.parametrize("bad", [-1, 40, 2**31 - 1, -2**31])
def test_fork_of_a_ragged_page_that_is_none(bad):
    """The child has no page where its parent has none: no free page is taken for it, and attention sees the same positions of both."""
    c = Cache(sequences=4, width=4, pages=12, page_size=16, heads=2, dim=64, layers=2, seed=3)
    c.model.table = [[3, 5, bad, -1], [7, -1, -1, -1], [9, bad, 4, 8], [1, -1, -1, -1]]
    c.model.length, c.model.held = [40, 9, 45, 16], [3, 1, 4, 1]
    c.model.refcount = [0, 1, 0, 1, 1, 1, 0, 1, 1, 1, 0, 0]
    c.up()
    k, v = c.k.clone(), c.v.clone()
    c.fork([-1, 0, -1, 2])
    torch.cuda.synchronize()
    # the second sequence has no page at column 2, the fourth a hole at column 1 and a copy of page 4 (13 slots) in page 0
    assert c.status.item() == 0
    assert c.length.tolist() == [40, 40, 45, 45] and c.held.tolist() == [3, 3, 4, 3]
    assert c.table.tolist() == [[3, 5, bad, -1], [3, 5, -1, -1], [9, bad, 4, 8], [9, bad, 0, -1]]
    assert c.refcount.tolist() == [1, 0, 0, 2, 1, 2, 0, 0, 1, 2, 0, 0]
    k[:, 0, :13], v[:, 0, :13] = k[:, 4, :13], v[:, 4, :13]
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    q = torch.randn((1, 4, 64), device="cuda").to(torch.bfloat16).repeat(4, 1, 1)
    out = torch.empty_like(q)
    c.attend(q, out, i32([0, 1, 2, 3, 4]))           # (a chain of one node whose position has no page)
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1])
    c.free([1, 1, 1, 1])
    torch.cuda.synchronize()
    assert c.refcount.tolist() == [0] * 12


def test_fork_of_a_missing_page_needs_no_free_one():
    c = Cache(sequences=2, width=2, pages=2, page_size=4, heads=1, dim=8)
    c.model.table, c.model.length, c.model.held, c.model.refcount = [[0, -1], [1, -1]], [6, 3], [2, 1], [1, 1]
    c.up()
    c.fork([-1, 0])
    torch.cuda.synchronize()
    assert c.status.item() == 0
    assert c.table.tolist() == [[0, -1], [0, -1]] and c.length.tolist() == [6, 6] and c.held.tolist() == [2, 2] and c.refcount.tolist() == [2, 0]


@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_past_the_table_are_turned_by_where_they_belong(interleaved):
    """Lengths past what a row of the table holds: nothing is written, the queries are turned by length + node all the same.

    Bound of tests/test_gpu_rope.py; an angle of 2^31 turns carries two 64-bit roundings of 2^-53 * 2^31 each, 2^-21 together."""
    c = Cache(sequences=5, width=2, pages=10, page_size=4, heads=1, dim=64)
    c.model.table = [[0, 1], [2, 3], [4, 5], [6, 7], [8, 9]]
    c.model.length, c.model.held = [8, 1000, 2**31 - 1, 2**31 - 2, -7], [2] * 5
    c.up()
    q = torch.randn((10, 2, 64), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    k = torch.randn((10, 1, 64), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    out, want_v, old_k = torch.zeros_like(q), c.v.clone(), c.k.clone()
    c.append(rope_plan(64, 64, interleaved), q, out, k, k, i32([0, 2, 4, 6, 8, 10]))
    torch.cuda.synchronize()
    at = [8, 9, 1000, 1001, 2**31 - 1, 2**31, 2**31 - 2, 2**31 - 1, 0, 1]       # (a length below zero is an empty sequence)
    f, m = frequencies(64, 10000.0)
    want, size = rotate(f64(q), at, f, m, interleaved)
    size *= np.where(np.array(at) > 2**24, 4.0, 1.0)[:, None, None]
    bound = step("bf16") * np.abs(want) + (1 + step("bf16")) * 2.0**-21 * size + smallest("bf16")
    assert (np.abs(f64(out) - want) <= bound).all()
    want_v[0, 8, 0], want_v[0, 8, 1] = k[8], k[9]
    assert torch.equal(c.v, want_v)
    untouched = torch.ones(c.k.shape[:3], dtype=torch.bool, device="cuda")
    untouched[0, 8, :2] = False
    assert torch.equal(c.k[untouched], old_k[untouched])


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("nodes,group,sequences", [(1, 4, 1), (1, 4, 400), (6, 4, 3), (40, 1, 3), (40, 1, 300), (64, 4, 3), (64, 4, 200), (150, 4, 200)])
def test_scores_past_fp32_make_their_rows_nan(nodes, group, sequences, tree):
    """Finite scores whose product with scale * log2(e) is not: no weights can be formed, and zeros would say that nothing was seen.  Items that
    are cut and whole ones, every form; rows of other heads and sequences are as without them."""
    lengths = [70] * sequences
    c = Cache(sequences=sequences, width=16, pages=16 * sequences, page_size=16, heads=2, dim=64, seed=11)
    assert c.model.reserve([x + nodes for x in lengths]) == 0
    c.model.length = lengths
    c.up()
    q = torch.randn((sequences * nodes, 2 * group, 64), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    start, space = i32(list(range(0, (sequences + 1) * nodes, nodes))), c.workspace(2 * group)
    mask = words(np.concatenate([random_tree(np.random.default_rng(s), nodes) for s in range(sequences)])) if tree else None
    plain, out = torch.empty_like(q), torch.empty_like(q)
    c.attend(q, plain, start, mask, scale=1.0, space=space)
    wild = q.clone()
    wild[0, 1] = 0
    wild[0, 1, 3] = 2.0**62                       # 2^62 * 2^64 * 3 * log2(e) is past 2^128, the products alone are not
    p, slot = c.model.place(0, 5)
    c.k[0, p, slot, 0, 3] = 2.0**64
    wild[1:, :group, 3] = 0                       # (what the other rows of this cache head see there does not change)
    wild[0, [h for h in range(group) if h != 1], 3] = 0
    quiet = wild.clone()
    quiet[0, 1] = 0
    c.attend(quiet, plain, start, mask, scale=3.0, space=space)
    c.attend(wild, out, start, mask, scale=3.0, space=space)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(plain).all())
    assert bool(out[0, 1].isnan().all())
    same = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    same[0, 1] = False
    assert torch.equal(out[same], plain[same])


def guarded(q):
    """An output for q's rows inside a wider buffer of nines, and that buffer."""
    back = torch.full((q.shape[0] + 8, q.shape[1] + 2, q.shape[2] + 8), 9.0, dtype=q.dtype, device="cuda")
    return back[4:-4, 1:-1, :q.shape[2]], back


def only(back, out, named):
    """Nothing but the named rows of the output was written."""
    rest = back.clone()
    view = rest[4:-4, 1:-1, :out.shape[2]]
    view[named] = 9.0
    return bool((rest == 9).all())


@pytest.mark.parametrize("group,tree", [(2, True), (2, False), (8, True), (12, True), (50, True), (100, False)])
@pytest.mark.parametrize("wrong,same_as", [([0, 100, -3, 9], [0, 9, 9, 9]), ([5, 2, 9, 4], [2, 2, 9, 9]), ([-4, 3, 7, 9], [3, 3, 7, 9]),
                                           ([2**31 - 1, -2**31, 9, 9], [9, 9, 9, 9])])
def test_row_starts_that_do_not_ascend(wrong, same_as, group, tree):
    """A sequence whose start is negative or not below its end has no rows, ends are cut to the rows there are; no other row is written, nor a byte
    behind the workspace."""
    c, q, start, bits = setup([3, 4, 2], [10, 40, 80], group=group, seed=5, tree=tree)
    out, back = guarded(q)
    space = c.attend(q, out, i32(wrong), None if bits is None else words(bits))
    torch.cuda.synchronize()
    assert bool((space[-64:] == 0xA5).all())
    want, bound = attention(f64(q), c.model, f64(c.k[0]), f64(c.v[0]), same_as, bits, 0.125, c.dtype)
    named = ~np.isnan(want).any((1, 2))
    assert named.sum() == same_as[-1] - same_as[0]
    assert only(back, out, torch.from_numpy(named).cuda())
    assert (np.abs(f64(out)[named] - want[named]) <= bound[named]).all()


@pytest.mark.parametrize("group,tree", [(2, True), (2, False), (8, True), (12, True), (50, True), (100, False)])
def test_lengths_past_the_table(group, tree):
    """The positions of the held pages are seen, no drafted node is: none has a page."""
    c, q, start, bits = setup([4, 2], [70, 40], page_size=16, group=group, seed=8, tree=tree)
    c.model.length = [10**6, 2**31 - 1]
    c.up()
    out, back = guarded(q)
    space = c.attend(q, out, i32(start), None if bits is None else words(bits))
    torch.cuda.synchronize()
    assert bool((space[-64:] == 0xA5).all()) and only(back, out, slice(None))
    c.model.length = [c.model.width * 16] * 2
    want, bound = attention(f64(q), c.model, f64(c.k[0]), f64(c.v[0]), start, bits, 0.125, c.dtype)
    assert (np.abs(f64(out) - want) <= bound).all()


def test_keys_are_written_only_where_their_rows_have_a_page():
    """Rows past the held pages, past the table and in pages that are none; keys are turned, values are copied, everything else stays."""
    c = Cache(sequences=4, width=2, pages=4, page_size=4, heads=2, dim=64, layers=2)
    c.model.table = [[0, -1], [1, 7], [2, 3], [-9, 2**31 - 1]]
    c.model.length, c.model.held = [3, 3, 7, 2], [2, 2, 2, 2]
    c.up()
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn((8, h, 64), generator=g).to(torch.bfloat16).cuda() for h in (4, 2, 2))
    out, want_k, want_v = torch.zeros_like(q), c.k.clone(), c.v.clone()
    at = [1, 5, 2, 9, 0, 3, 7, 8]
    c.append(rope_plan(64, 64, True), q, out, k, v, i32([0, 2, 4, 6, 8]), i32(at), layer=1)
    torch.cuda.synchronize()
    f, m = frequencies(64, 10000.0)
    for got, x in ((out, q), (torch.stack([c.k[1, 0, 3], c.k[1, 1, 3], c.k[1, 3, 3]]), k[[0, 2, 4]])):
        want, size = rotate(f64(x), at if x is q else [at[0], at[2], at[4]], f, m, True)
        assert (np.abs(f64(got) - want) <= step("bf16") * np.abs(want) + (1 + step("bf16")) * 2.0**-21 * size + smallest("bf16")).all()
    for row, (page, slot) in {0: (0, 3), 2: (1, 3), 4: (3, 3)}.items():
        want_k[1, page, slot], want_v[1, page, slot] = c.k[1, page, slot], v[row]
    assert torch.equal(c.k, want_k) and torch.equal(c.v, want_v)


@pytest.mark.parametrize("tree", [True, False])
def test_a_run_of_a_pools_sequences_is_a_pool(tree):
    """Sequences of different kinds in calls of their own (a prompt, single tokens): pool and row starts begin at the run's first sequence, rows keep
    their numbers.  Together they are the one call's rows."""
    counts, lengths = [1, 1, 180, 1], [300, 90, 40, 7]
    c, q, start, bits = setup(counts, lengths, group=4, heads=2, dim=128, seed=21, tree=tree)
    mask = None if bits is None else words(bits)
    pool, starts = c.pool(), i32(start)
    out, back = guarded(q)
    for first, n in ((0, 2), (2, 1), (3, 1)):
        view = c.pool()
        view.sequences = n
        view.table, view.length, view.held = pool.table + 4 * first * pool.table_stride, pool.length + 4 * first, pool.held + 4 * first
        c.pool = lambda view=view: view
        c.attend(q, out, starts[first:first + n + 1], mask)
        torch.cuda.synchronize()
        assert only(back, out, slice(0, start[first + n]))
        del c.pool
    use = bits
    if bits is not None:
        use = bits.copy()
        for s, t in enumerate(counts):
            use[start[s]:start[s + 1], t:] = False
    want, bound = attention(f64(q), c.model, f64(c.k[0]), f64(c.v[0]), start, use, 0.125, c.dtype)
    assert (np.abs(f64(out) - want) <= bound).all()


@pytest.mark.parametrize("counts,lengths,group,tree", [([3, 1, 7], [40, 100, 5], 2, True), ([40, 9, 0], [300, 20, 70], 4, True), ([200, 150], [20, 300], 4, False)])
def test_rows_of_the_table_inside_wider_ones(counts, lengths, group, tree):
    """A table_stride above table_width: every call stays within the rows.  And attention in place, chains whose tiles end at their last node too."""
    c, q, start, bits = setup(counts, lengths, group=group, tree=tree, seed=3)
    n, width = c.table.shape
    wide = torch.full((n, width + 5), 77, dtype=torch.int32, device="cuda")
    wide[:, :width] = c.table
    c.table = wide[:, :width]
    mask, out = None if bits is None else words(bits), torch.empty_like(q)
    use = None if bits is None else bits.copy()
    if use is not None:
        for s, t in enumerate(counts):
            use[start[s]:start[s + 1], t:] = False
    want, bound = attention(f64(q), c.model, f64(c.k[0]), f64(c.v[0]), start, use, 0.125, c.dtype)
    c.attend(q, out, i32(start), mask)
    c.attend(q, q, i32(start), mask)
    torch.cuda.synchronize()
    assert torch.equal(q, out) and (np.abs(f64(out) - want) <= bound).all()
    for call in (lambda x: x.fork([-1] + [0] * (n - 1)), lambda x: x.free([0] + [1] * (n - 1)), lambda x: x.reserve([30] * n)):
        call(c)
        call(c.model)
        c.same_state()
    assert c.status.item() == 0
    assert bool((wide[:, width:] == 77).all())


def test_calls_from_several_host_threads():
    """A stream and a workspace each: the same results as one after the other."""
    work = [setup([5 + s], [900], group=4, dim=128, seed=s) for s in range(4)]
    alone, together = [torch.empty_like(q) for _, q, *_ in work], [torch.empty_like(q) for _, q, *_ in work]
    held = [(i32(start), words(bits), c.workspace(q.shape[1]), torch.cuda.Stream()) for c, q, start, bits in work]
    for (c, q, *_), o, (st, w, space, _) in zip(work, alone, held):
        c.attend(q, o, st, w, space=space)
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            (c, q, *_), (st, w, space, stream) = work[i], held[i]
            for _ in range(100):
                c.attend(q, together[i], st, w, stream=stream.cuda_stream, space=space)
            stream.synchronize()
        except Exception as e:
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and all(torch.equal(a, b) for a, b in zip(alone, together))
