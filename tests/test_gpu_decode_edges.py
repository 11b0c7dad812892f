"""What the decoding operators' contract says for inputs at its edge: values that are not finite in stages that are filled again, lengths and
pages that the pool does not hold, scores past fp32's range, rows that no sequence names."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from decode_model import TORCH, attention  # noqa: E402
from decode_util import Cache, f64, i32, random_tree, words  # noqa: E402


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
