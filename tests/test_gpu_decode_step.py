"""A decoder's steps as they are run: projections with 4-bit weights, rotary positions and the cache's pages, attention of a drafted tree,
the accepted path kept, beams forked, sequences freed - against 64-bit numbers for every step, captured and not."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import tpu_mlir_b200._lib as L  # noqa: E402
from decode_model import attention, frequencies, rotate, step  # noqa: E402
from decode_util import Cache, f64, i32, random_tree, rope_plan, words  # noqa: E402

HQ, HK, DIM, HIDDEN, GROUP = 4, 2, 64, 256, 64


class Projection:
    """tpu.A16MatMul through a device handle: hidden -> queries, keys and values side by side."""

    def __init__(self, n, k, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.wq = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
        self.sc = (torch.rand(n * k // GROUP, device="cuda", generator=g) * 0.01 + 0.002).to(torch.bfloat16)
        self.zp = torch.full((n * k // GROUP,), 8, dtype=torch.uint8, device="cuda")
        self.n, self.h = n, C.c_void_p()
        L.check(L.lib().b200q_a16_dev_create_dt(self.wq.data_ptr(), self.sc.data_ptr(), self.zp.data_ptr(), None, n, k, GROUP, L.DT_BF16, C.byref(self.h)))

    def __call__(self, x, y, stream=None):
        L.check(L.lib().b200q_a16_dev_run(self.h, x.data_ptr(), y.data_ptr(), x.shape[0], stream))

    def __del__(self):
        L.lib().b200q_a16_dev_destroy(C.byref(self.h))


@pytest.mark.parametrize("captured", [False, True])
def test_drafted_steps(captured):
    rng = np.random.default_rng(7)
    n, nodes, steps = 3, 6, 4
    c = Cache(sequences=n, width=12, pages=40, page_size=8, heads=HK, dim=DIM, layers=2, seed=1)
    c.model.length = [13, 0, 30]
    c.held.fill_(0)
    assert c.model.reserve([0, 0, 0]) == 0
    c.up()
    proj = Projection((HQ + 2 * HK) * DIM, HIDDEN, 3)
    plan = rope_plan(DIM, DIM, False, kind="linear", factor=2.0)
    f, m = frequencies(DIM, 10000.0, "linear", 2.0)
    rows = n * nodes
    x = torch.zeros((rows, HIDDEN), dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros((rows, HQ + 2 * HK, DIM), dtype=torch.bfloat16, device="cuda")
    q, out = (torch.zeros((rows, HQ, DIM), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    start, extra = i32([s * nodes for s in range(n + 1)]), i32([nodes] * n)
    mask, positions = torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    path, count = torch.zeros((n, 4), dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    space = c.workspace(HQ)
    lib, cache, pool = L.lib(), c.cache(), c.pool()

    def verify(stream):
        L.check(lib.b200q_kv_reserve_dev(C.byref(pool), extra.data_ptr(), c.status.data_ptr(), stream))
        proj(x, qkv, stream)
        for layer in (0, 1):
            c.append(plan, qkv[:, :HQ], q, qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:], start, positions, layer=layer, stream=stream)
        c.attend(q, out, start, mask, scale=DIM ** -0.5, layer=1, stream=stream, space=space)

    def accept(stream):
        L.check(lib.b200q_kv_compact_dev(C.byref(cache), C.byref(pool), path.data_ptr(), 4, 4, count.data_ptr(), c.length.data_ptr(), stream))

    stream, graphs = None, []
    if captured:
        side = torch.cuda.Stream()
        verify(None)                                     # (first calls outside a capture; the state is put back below)
        torch.cuda.synchronize()
        for call in (verify, accept):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call(side.cuda_stream)
            graphs.append(g)
        for t, v in ((c.table, c.model.table), (c.length, c.model.length), (c.held, c.model.held), (c.refcount, c.model.refcount)):
            t.copy_(i32(v))
    for turn in range(steps):
        assert c.model.reserve([nodes] * n) == 0
        trees = [random_tree(rng, nodes) for _ in range(n)]
        bits = np.concatenate(trees)
        at = [c.model.length[s] + int(trees[s][i].sum()) - 1 for s in range(n) for i in range(nodes)]
        x.copy_(torch.from_numpy(rng.standard_normal((rows, HIDDEN))).to(torch.bfloat16))
        mask.copy_(words(bits))
        positions.copy_(i32(at))
        # the longest path of each tree, cut to four nodes
        paths = []
        for t in trees:
            deepest = max(range(nodes), key=lambda i: t[i].sum())
            paths.append([int(j) for j in np.nonzero(t[deepest])[0]][:4])
        path.copy_(i32([p + [0] * (4 - len(p)) for p in paths]))
        count.copy_(i32([len(p) for p in paths]))
        graphs[0].replay() if captured else verify(stream)
        torch.cuda.synchronize()
        c.same_state()
        assert c.status.item() == 0
        y = f64(qkv)
        turned, size = rotate(y[:, :HQ], at, f, m, False)
        assert (np.abs(f64(q) - turned) <= step("bf16") * np.abs(turned) + 2.0**-20 * size + 1e-30).all()
        keys, size = rotate(y[:, HQ:HQ + HK], at, f, m, False)
        for r in range(rows):
            p, t = c.model.place(r // nodes, c.model.length[r // nodes] + r % nodes)
            for layer in (0, 1):
                assert (np.abs(f64(c.k[layer, p, t]) - keys[r]) <= step("bf16") * np.abs(keys[r]) + 2.0**-20 * size[r] + 1e-30).all()
                assert (f64(c.v[layer, p, t]) == y[r, HQ + HK:]).all()
        want, bound = attention(f64(q), c.model, f64(c.k[1]), f64(c.v[1]), start.tolist(), bits, DIM ** -0.5, "bf16")
        assert (np.abs(f64(out) - want) <= bound).all()
        k, v = c.k.clone(), c.v.clone()
        for s, p in enumerate(paths):
            for a, b in c.model.path(s, p):
                k[:, b[0], b[1]], v[:, b[0], b[1]] = k[:, a[0], a[1]].clone(), v[:, a[0], a[1]].clone()
            c.model.length[s] += len(p)
        graphs[1].replay() if captured else accept(stream)
        c.same_state()
        assert torch.equal(c.k, k) and torch.equal(c.v, v)
    # the first sequence goes on as two beams, the second ends
    c.fork([-1, 0, -1])
    code, copies = c.model.fork([-1, 0, -1])
    assert code == 0
    for src, dst, slots in copies:
        assert torch.equal(c.k[:, dst, :slots], c.k[:, src, :slots]) and torch.equal(c.v[:, dst, :slots], c.v[:, src, :slots])
    c.same_state()
    # both beams attend to the same past
    c.reserve([1, 1, -1])
    c.model.reserve([1, 1, -1])
    one = torch.randn((1, HQ + 2 * HK, DIM), device="cuda").to(torch.bfloat16).repeat(2, 1, 1)
    got = torch.empty((2, HQ, DIM), dtype=torch.bfloat16, device="cuda")
    rot = torch.empty_like(got)
    c.append(plan, one[:, :HQ], rot, one[:, HQ:HQ + HK], one[:, HQ + HK:], i32([0, 1, 2, 2]), layer=1)
    c.attend(rot, got, i32([0, 1, 2, 2]), scale=DIM ** -0.5, layer=1)
    torch.cuda.synchronize()
    assert torch.equal(got[0], got[1])
    want, bound = attention(f64(rot), c.model, f64(c.k[1]), f64(c.v[1]), [0, 1, 2, 2], None, DIM ** -0.5, "bf16")
    assert (np.abs(f64(got) - want) <= bound).all()
    for which in ([0, 1, 0], [1, 0, 1]):
        c.free(which)
        c.model.free(which)
        c.same_state()
    assert sum(c.model.refcount) == 0


def test_a_chain_of_tokens_and_the_same_tokens_as_one_prompt_agree():
    """Token by token and all at once: the cache gets the same bits, the outputs differ by roundings only."""
    n = 70
    qkv = torch.randn((n, HQ + 2 * HK, DIM), generator=torch.Generator().manual_seed(5)).to(torch.float16).cuda()
    results, caches = [], []
    for at_once in (True, False):
        c = Cache(sequences=1, width=6, pages=6, page_size=16, heads=HK, dim=DIM, dtype="f16", seed=2)
        c.reserve([n])
        plan, out, q = rope_plan(DIM, 32, True), torch.empty((n, HQ, DIM), dtype=torch.float16, device="cuda"), torch.empty((n, HQ, DIM), dtype=torch.float16, device="cuda")
        for lo in range(0, n, n if at_once else 1):
            hi = n if at_once else lo + 1
            rows, start = qkv[lo:hi], i32([0, hi - lo])
            c.append(plan, rows[:, :HQ], q[lo:hi], rows[:, HQ:HQ + HK], rows[:, HQ + HK:], start)
            c.attend(q[lo:hi], out[lo:hi], start, scale=DIM ** -0.5)
            c.length.fill_(hi)
        torch.cuda.synchronize()
        results.append((f64(out), f64(q)))
        caches.append(c)
    assert np.array_equal(results[0][1], results[1][1])
    assert all(torch.equal(caches[0].k[0, p], caches[1].k[0, p]) for p in range(4))
    c = caches[0]
    c.model.reserve([n])
    want, bound = attention(results[0][1], c.model, f64(c.k[0]), f64(c.v[0]), [0, n], None, DIM ** -0.5, "f16")
    for got, _ in results:
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("nodes,group", [(1, 1), (40, 2), (100, 4)])
def test_a_wait_that_runs_out_is_reported(nodes, group):
    """Stages that wait for bytes that never come (no fault, no hang): the status says so within the budget, and the next call is right."""
    c = Cache(sequences=1, width=20, pages=20, page_size=16, heads=1, dim=64, seed=4)
    assert c.model.reserve([200 + nodes]) == 0
    c.model.length = [200]
    c.up()
    q = torch.randn((nodes, group, 64), device="cuda").to(torch.bfloat16)
    out, start, space, status = torch.empty_like(q), i32([0, nodes]), c.workspace(group), torch.zeros(1, dtype=torch.int32, device="cuda")
    lib = L.lib()

    def call():
        a = L.TreeAttention(q=q.data_ptr(), out=out.data_ptr(), row_start=start.data_ptr(), mask=None, workspace=space.data_ptr(), workspace_bytes=space.numel() - 64,
                            q_row_stride=q.stride(0), q_head_stride=q.stride(1), out_row_stride=out.stride(0), out_head_stride=out.stride(1), mask_stride=0, rows=nodes,
                            q_heads=group, layer=0, scale=0.125, status=status.data_ptr())
        L.check(lib.b200q_tree_attention_dev(C.byref(c.cache()), C.byref(c.pool()), C.byref(a), None))
        torch.cuda.synchronize()
    try:
        lib.b200q_debug_set_wait_fault(16, 1000000)
        call()
        assert status.item() != 0
    finally:
        lib.b200q_debug_set_wait_fault(0, 0)
    status.zero_()
    call()
    assert status.item() == 0
    want, bound = attention(f64(q), c.model, f64(c.k[0]), f64(c.v[0]), [0, nodes], None, 0.125, "bf16")
    assert (np.abs(f64(out) - want) <= bound).all()


def test_two_captured_graphs_with_a_workspace_each():
    made = []
    for seed, nodes, length in ((1, 30, 900), (2, 3, 2500)):
        c = Cache(sequences=1, width=50, pages=50, page_size=64, heads=2, dim=128, seed=seed)
        assert c.model.reserve([length + nodes]) == 0
        c.model.length = [length]
        c.up()
        q = torch.randn((nodes, 8, 128), device="cuda").to(torch.bfloat16)
        out, start, space = torch.zeros_like(q), i32([0, nodes]), c.workspace(8)
        alone = torch.empty_like(q)
        c.attend(q, alone, start, space=space)
        torch.cuda.synchronize()
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=side):
            for _ in range(5):
                c.attend(q, out, start, stream=side.cuda_stream, space=space)
        made.append((g, side, out, alone, c, q, start, space))
    for _ in range(10):
        for g, side, *_ in made:
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone) for _, _, out, alone, *_ in made)
