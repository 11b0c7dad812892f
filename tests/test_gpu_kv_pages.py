"""Pages of the key / value cache: tables, counts and moved entries against a plain Python pool, exactly."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from decode_model import Pool, attention  # noqa: E402
from decode_util import Cache, f64, i32, rope_plan, words  # noqa: E402


def filled(c, lengths):
    """Sequences of these lengths, pages handed out by the model."""
    assert c.model.reserve(lengths) == 0
    c.model.length = list(lengths)
    c.up()


@pytest.mark.parametrize("sequences,width,pages,page_size", [(1, 1, 1, 1), (3, 5, 17, 4), (7, 40, 260, 3), (130, 9, 1000, 16), (1024, 4, 4099, 2),
                                                             (5, 200, 70001, 8), (2, 5000, 1 << 20, 16)])
def test_reserve_and_free(sequences, width, pages, page_size):
    rng = np.random.default_rng(pages)
    c = Cache(sequences=sequences, width=width, pages=pages, page_size=page_size, heads=1, dim=8, layers=1) if pages < 1 << 17 else \
        Cache(sequences=sequences, width=width, pages=pages, page_size=page_size, heads=1, dim=8, layers=1, pad=0)
    most = min(width * page_size, pages * page_size // max(1, sequences))
    for turn in range(5):
        extra = [int(e) for e in rng.integers(-1, max(1, most // 2) + 1, sequences)]
        c.status.zero_()
        c.reserve(extra)
        code = c.model.reserve(extra)
        c.same_state()
        assert c.status.item() == code
        if turn % 2:
            which = [int(w) for w in rng.integers(0, 2, sequences)]
            c.free(which)
            c.model.free(which)
            c.same_state()
        else:
            c.model.length = [h * page_size - int(rng.integers(0, page_size)) if h else 0 for h in c.model.held]
            c.up()


def test_reserve_is_all_or_nothing():
    c = Cache(sequences=3, width=4, pages=6, page_size=4, heads=1, dim=8)
    c.reserve([8, 8, 12])                       # seven pages of six
    assert c.status.item() == 1
    c.same_state()
    c.status.zero_()
    c.reserve([4, 17, -5])                      # a row of five entries in a table of four
    assert c.status.item() == 2
    c.same_state()
    c.status.zero_()
    c.reserve([8, 0, 16])
    assert c.model.reserve([8, 0, 16]) == 0 and c.status.item() == 0
    c.same_state()
    c.reserve([2**31 - 1, -1, -1])              # far past 32 bits of positions
    assert c.status.item() == 2
    c.same_state()


@pytest.mark.parametrize("layout,heads,dim,dtype", [("nhd", 2, 64, "bf16"), ("hnd", 3, 80, "f16"), ("nhd", 1, 8, "f16"), ("hnd", 1, 256, "bf16")])
@pytest.mark.parametrize("page_size", [1, 5, 16])
def test_fork(layout, heads, dim, dtype, page_size):
    rng = np.random.default_rng(dim + page_size)
    n = 9
    c = Cache(sequences=n, width=12, pages=150, page_size=page_size, heads=heads, dim=dim, layers=3, dtype=dtype, layout=layout, pad=8)
    filled(c, [int(x) for x in rng.integers(0, 11 * page_size, n)])
    for parent in ([-1] * n,
                   list(range(n)),                           # itself: left alone
                   [1, 0] + list(range(2, n)),               # a swap
                   [0] * n,                                  # all from one
                   [0, 0, 1, 2, 3, 4, 5, 6, 7],              # a chain of children that are parents
                   [8, n, -2, 2**31 - 1, 0, 0, 8, 1, 1]):    # values that name nobody
        k, v = c.k.clone(), c.v.clone()
        c.fork(parent)
        code, copies = c.model.fork(parent)
        for src, dst, slots in copies:
            k[:, dst, :slots], v[:, dst, :slots] = k[:, src, :slots].clone(), v[:, src, :slots].clone()
        assert code == 0 and c.status.item() == 0
        c.same_state()
        assert torch.equal(c.k, k) and torch.equal(c.v, v)
        c.model.length = [max(0, x - int(rng.integers(0, 2))) if x % page_size else x for x in c.model.length]
        c.up()


def test_fork_of_many_sequences():
    rng = np.random.default_rng(5)
    n = 1024
    c = Cache(sequences=n, width=7, pages=6000, page_size=2, heads=1, dim=8, layers=2)
    filled(c, [int(x) for x in rng.integers(0, 9, n)])
    parent = [int(p) for p in rng.integers(0, n, n)]
    k, v = c.k.clone(), c.v.clone()
    c.fork(parent)
    code, copies = c.model.fork(parent)
    assert code == 0
    for src, dst, slots in copies:
        k[:, dst, :slots], v[:, dst, :slots] = k[:, src, :slots], v[:, src, :slots]
    c.same_state()
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


def test_fork_without_pages_changes_nothing():
    c = Cache(sequences=3, width=3, pages=3, page_size=4, heads=1, dim=8)
    filled(c, [6, 0, 0])
    c.fork([0, 0, 0])                            # two ragged children, one free page
    assert c.status.item() == 1
    c.same_state()
    c.status.zero_()
    c.fork([0, 0, -1])
    assert c.model.fork([0, 0, -1])[0] == 0 and c.status.item() == 0
    c.same_state()


@pytest.mark.parametrize("layout,heads,dim,dtype,page_size,layers", [("nhd", 2, 64, "bf16", 16, 3), ("hnd", 3, 80, "f16", 5, 2), ("nhd", 8, 128, "bf16", 1, 1),
                                                                     ("hnd", 1, 8, "f16", 64, 4)])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact(layout, heads, dim, dtype, page_size, layers, in_place):
    rng = np.random.default_rng(dim)
    n, drafts = 7, 40
    c = Cache(sequences=n, width=-(-90 // page_size), pages=n * (-(-90 // page_size)) + 2, page_size=page_size, heads=heads, dim=dim, layers=layers, dtype=dtype,
              layout=layout, pad=8)
    lengths = [0, 1, 17, 30, 44, 49, 50]
    assert c.model.reserve([x + drafts for x in lengths]) == 0
    c.model.length = lengths
    c.up()
    paths = [sorted(int(x) for x in rng.choice(drafts, m, replace=False)) for m in (0, 1, 7, 8, 9, 40, 25)]
    paths[1] = [39]
    paths[4] = [0, 1, 2, 5, 5, 9, 11, 12, 13]     # a node twice: the path ends there
    paths[6] = [3, 4, 2, 8] + [9] * 21            # not ascending
    width = 41
    rows = [p + [77] * (width - len(p)) for p in paths]
    want_k, want_v, after = c.k.clone(), c.v.clone(), []
    for s, p in enumerate(paths):
        moves = c.model.path(s, p)
        for (pa, ta), (pb, tb) in moves:
            want_k[:, pb, tb], want_v[:, pb, tb] = want_k[:, pa, ta].clone(), want_v[:, pa, ta].clone()
        after.append(lengths[s] + len(moves))
    out = c.length if in_place else torch.full((n,), -1, dtype=torch.int32, device="cuda")
    c.compact(rows, [len(p) for p in paths], out=out)
    torch.cuda.synchronize()
    assert out.tolist() == after
    assert after == [0, 2, 24, 38, 48, 89, 52]
    if not in_place:
        assert c.length.tolist() == lengths
    assert torch.equal(c.k, want_k) and torch.equal(c.v, want_v)


def test_compact_of_paths_that_leave_the_pool():
    c = Cache(sequences=4, width=3, pages=8, page_size=4, heads=1, dim=16)
    c.model.table = [[0, 1, -1], [2, 99, 3], [4, 5, 6], [7, -1, -1]]
    c.model.length, c.model.held = [3, 1, 10, 2], [2, 3, 3, 1]
    c.up()
    k = c.k.clone()
    # past the held pages; a page that is none; past the table; a count above the row's width and one below zero
    c.compact([[2, 4, 6], [1, 4, 5], [1, 2, 3], [1, 2, 3]], [3, 3, 999, -4])
    torch.cuda.synchronize()
    assert c.length.tolist() == [3 + 2, 1 + 1, 10 + 1, 2]
    for s, (a, b) in ((0, (5, 3)), (0, (7, 4)), (1, (2, 1)), (2, (11, 10))):
        pa, pb = c.model.place(s, a), c.model.place(s, b)
        k[:, pb[0], pb[1]] = k[:, pa[0], pa[1]].clone()
    assert torch.equal(c.k, k)


def test_compact_of_nothing_and_of_the_longest_path():
    c = Cache(sequences=1, width=70, pages=70, page_size=16, heads=1, dim=8)
    assert c.model.reserve([1100]) == 0
    c.model.length = [40]
    c.up()
    path = list(range(7, 7 + 1024))
    k = c.k.clone()
    c.compact([path], [0])
    assert c.length.tolist() == [40] and torch.equal(c.k, k)
    c.compact([path], [1024])
    torch.cuda.synchronize()
    for i, node in enumerate(path):
        (pa, ta), (pb, tb) = c.model.place(0, 40 + node), c.model.place(0, 40 + i)
        k[:, pb, tb] = k[:, pa, ta].clone()
    assert c.length.tolist() == [1064] and torch.equal(c.k, k)


def test_a_captured_step_on_another_stream():
    """Reserve, compact, fork and free captured once and replayed: the state goes on from replay to replay."""
    c = Cache(sequences=4, width=30, pages=120, page_size=4, heads=2, dim=64, layers=2)
    filled(c, [5, 9, 3, 1])
    ready = i32([8, 8, 8, 8])
    path, count = i32([[0, 2, 5]] * 4), i32([3, 1, 2, 0])
    parent, which = i32([-1, -1, 0, -1]), i32([0, 0, 0, 1])
    import ctypes as C

    import tpu_mlir_b200._lib as L
    lib, cache, pool = L.lib(), c.cache(), c.pool()

    def step(stream):
        L.check(lib.b200q_kv_reserve_dev(C.byref(pool), ready.data_ptr(), c.status.data_ptr(), stream))
        L.check(lib.b200q_kv_compact_dev(C.byref(cache), C.byref(pool), path.data_ptr(), 3, 3, count.data_ptr(), c.length.data_ptr(), stream))
        L.check(lib.b200q_kv_fork_dev(C.byref(cache), C.byref(pool), parent.data_ptr(), c.status.data_ptr(), stream))
        L.check(lib.b200q_kv_free_dev(C.byref(pool), which.data_ptr(), stream))

    k = c.k.clone()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for _ in range(4):
        graph.replay()
        assert c.model.reserve([8] * 4) == 0
        for s, n in enumerate([3, 1, 2, 0]):
            moves = c.model.path(s, [0, 2, 5][:n])
            for (pa, ta), (pb, tb) in moves:
                k[:, pb, tb] = k[:, pa, ta].clone()
            c.model.length[s] += n
        code, copies = c.model.fork([-1, -1, 0, -1])
        assert code == 0
        for src, dst, slots in copies:
            k[:, dst, :slots] = k[:, src, :slots].clone()
        c.model.free([0, 0, 0, 1])
        c.same_state()
        assert torch.equal(c.k, k) and c.status.item() == 0


def test_counts_off_sixteen_bytes_and_a_pool_that_fills_the_default_shared_memory():
    c = Cache(sequences=2, width=40000, pages=262144, page_size=8, heads=1, dim=8)
    c.reserve([300000, 17])
    assert c.model.reserve([300000, 17]) == 0
    c.same_state()
    back = torch.zeros(70, dtype=torch.int32, device="cuda")
    for shift in (1, 2, 3):
        c = Cache(sequences=2, width=30, pages=61, page_size=4, heads=1, dim=8)
        back.zero_()
        back[:shift] = back[shift + 61:] = -9
        c.refcount = back[shift:shift + 61]
        for extra in ([50, 70], [80, 90], [400, 1]):
            c.reserve(extra)
            c.model.reserve(extra)
            c.same_state()
        assert (back[:shift] == -9).all() and (back[shift + 61:] == -9).all()


def test_without_a_status_word():
    import ctypes as C

    import tpu_mlir_b200._lib as L
    c = Cache(sequences=2, width=2, pages=3, page_size=4, heads=1, dim=8)
    lib = L.lib()
    for extra in ([9, 0], [8, 8], [8, 1]):       # too wide, too many, just right
        e = i32(extra)
        L.check(lib.b200q_kv_reserve_dev(C.byref(c.pool()), e.data_ptr(), None, None))
        c.model.reserve(extra)
        c.same_state()
    c.model.length = [7, 0]
    c.up()
    p = i32([0, 0])
    L.check(lib.b200q_kv_fork_dev(C.byref(c.cache()), C.byref(c.pool()), p.data_ptr(), None, None))    # no page is free
    c.same_state()


def test_entries_past_the_held_pages_are_not_looked_at():
    """A table whose rows were never cleared: what stands past the held pages names pages of others."""
    c = Cache(sequences=3, width=6, pages=10, page_size=4, heads=1, dim=8, layers=2)
    c.model.table = [[0, 1, 4, 5, 6, 7], [4, 5, 0, 0, 0, 0], [0, 1, 2, 3, 4, 5]]
    c.model.held, c.model.length = [2, 2, 0], [30, 7, 11]       # lengths past the held pages, too
    c.model.refcount = [1, 1, 0, 0, 1, 1, 0, 0, 0, 0]
    c.up()
    k = c.k.clone()
    c.compact([[0, 2], [0, 3], [1, 2]], [2, 2, 2])
    torch.cuda.synchronize()
    assert c.length.tolist() == [30, 8, 11] and torch.equal(c.k, k)      # (node 0 of the second sequence stays where it is)
    c.model.length = [30, 8, 11]
    c.fork([-1, 2, 0])                           # a parent without pages, and one whose length is past its pages
    torch.cuda.synchronize()
    assert c.length.tolist() == [30, 0, 8] and c.held.tolist() == [2, 0, 2]
    assert c.table.tolist()[1:] == [[-1] * 6, [0, 1, -1, -1, -1, -1]]
    assert c.refcount.tolist() == [2, 2, 0, 0, 0, 0, 0, 0, 0, 0]


def test_offsets_past_32_bits():
    """Pages whose elements lie past 2^31: appended to, attended, compacted and forked."""
    heads, dim, ps, pages = 8, 128, 64, 36000    # 65536 elements a page: the last ones lie past 2.3e9
    c = Cache(sequences=2, width=4, pages=4, page_size=ps, heads=heads, dim=dim, layers=1)
    c.model = Pool(2, 4, pages, ps)
    c.k, c.v = (torch.empty((1, pages, ps, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    used = [35999, 7, 35990, 32768]
    for t in (c.k, c.v):
        for p in used:
            t[0, p] = torch.randn((ps, heads, dim), device="cuda")
    c.model.table = [[35999, 7, 35990, 32768], [-1] * 4]
    c.model.held, c.model.length = [4, 0], [150, 0]
    c.model.refcount = [1] * (pages - 1) + [0]
    c.model.refcount[35999], c.model.refcount[35995] = 1, 0
    c.up()
    nodes = 40
    q = torch.randn((nodes, heads + 2 * heads, dim), device="cuda").to(torch.bfloat16)
    out, start = torch.empty((nodes, heads, dim), dtype=torch.bfloat16, device="cuda"), i32([0, nodes, nodes])
    c.append(rope_plan(dim, 0, False), q[:, :heads], out, q[:, heads:2 * heads], q[:, 2 * heads:], start)
    torch.cuda.synchronize()
    assert torch.equal(out, q[:, :heads])        # (no pair is turned)
    for i in range(nodes):
        p, t = c.model.place(0, 150 + i)
        assert torch.equal(c.k[0, p, t], q[i, heads:2 * heads]) and torch.equal(c.v[0, p, t], q[i, 2 * heads:])
    bits = np.tril(np.ones((nodes, nodes), bool))
    got = torch.empty_like(out)
    c.attend(out, got, start, words(bits), scale=dim ** -0.5)
    torch.cuda.synchronize()

    small = Pool(2, 4, 4, ps)                    # the pages that are used, for the 64-bit numbers
    small.table, small.held, small.length = [[0, 1, 2, 3], [-1] * 4], [4, 0], [150, 0]
    want, bound = attention(f64(out), small, f64(c.k[0][used]), f64(c.v[0][used]), [0, nodes, nodes], bits, dim ** -0.5, "bf16")
    assert (np.abs(f64(got) - want) <= bound).all()
    c.compact([[0, 5, 9], [0, 0, 0]], [3, 0])
    torch.cuda.synchronize()
    for i, n in enumerate((0, 5, 9)):
        p, t = c.model.place(0, 150 + i)
        assert torch.equal(c.k[0, p, t], q[n, heads:2 * heads])
    c.model.length = [153, 0]
    c.fork([-1, 0])                              # the ragged page lands in page 35995
    torch.cuda.synchronize()
    assert c.table.tolist()[1] == [35999, 7, 35995, -1]
    assert torch.equal(c.k[0, 35995, :25], c.k[0, 35990, :25]) and torch.equal(c.v[0, 35995, :25], c.v[0, 35990, :25])
