"""The operators of a decoding step over a paged key / value cache, as cases that can be measured one by one.

  rope       rotary positions on one tensor of heads
  append     rotary positions on queries and keys, the keys and values written into the pages of the cache
  attention  attention of a tree of drafted tokens (or of one token) over the pages of every sequence
  fork       sequences that become copies of others (beams reordered): full pages shared, the ragged last one copied
  compact    the accepted path of a drafted tree moved to the front, in every layer
  admit      finished sequences give their pages back, pages are reserved for new prompts and for the next drafts

With ``own`` false, ``run`` computes them from elementary torch operations; with ``own`` true it makes the library's calls.
Lengths are spread over a case's range by a fixed rule, so that ``work`` knows them; everything else comes from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # rotary positions of a prompt's queries, a head size and a head count that are no powers of two
        dict(name="rope_prompt_d80", kind="rope", rows=4001, heads=20, dim=80, rotary=32, interleaved=True, base=10000.0, scaling="none",
             far=4001, dtype="f16"),
        # one sequence, one token: a chat that is being answered, latency is all there is
        dict(name="append_b1_t1", kind="append", seqs=1, drafts=1, drafts_min=1, ctx=700, ctx_min=700, q_heads=32, kv_heads=8, dim=128,
             rotary=128, interleaved=False, base=500000.0, scaling="banded", page=16, layout="nhd", dtype="bf16", tree=False),
        # a served batch whose sequences all verify a drafted tree, long contexts, part of the head rotated
        dict(name="append_b64_tree", kind="append", seqs=64, drafts=24, drafts_min=8, ctx=30000, ctx_min=100, q_heads=32, kv_heads=8, dim=128,
             rotary=64, interleaved=True, base=10000.0, scaling="yarn", page=16, layout="nhd", dtype="f16", tree=True),
        # three prompts in one batch
        dict(name="append_prompts", kind="append", seqs=3, drafts=3900, drafts_min=1300, ctx=0, ctx_min=0, q_heads=32, kv_heads=8, dim=128,
             rotary=128, interleaved=False, base=10000.0, scaling="linear", page=64, layout="hnd", dtype="bf16", tree=False),
        # one sequence, one token, a short context: latency
        dict(name="attention_b1_t1", kind="attention", seqs=1, drafts=1, drafts_min=1, ctx=430, ctx_min=430, q_heads=32, kv_heads=8, dim=128,
             page=16, layout="nhd", dtype="bf16", tree=False),
        # token by token decoding of a served batch of uneven contexts
        dict(name="attention_b48_t1", kind="attention", seqs=48, drafts=1, drafts_min=1, ctx=8000, ctx_min=200, q_heads=32, kv_heads=8, dim=128,
             page=16, layout="nhd", dtype="bf16", tree=False),
        # drafted trees of a served batch
        dict(name="attention_b16_t24", kind="attention", seqs=16, drafts=24, drafts_min=9, ctx=5000, ctx_min=700, q_heads=32, kv_heads=8, dim=128,
             page=32, layout="hnd", dtype="bf16", tree=True),
        # one very long document, a few drafted tokens, seven queries to a key head
        dict(name="attention_b1_t7_long", kind="attention", seqs=1, drafts=7, drafts_min=7, ctx=131000, ctx_min=131000, q_heads=28, kv_heads=4,
             dim=64, page=64, layout="nhd", dtype="f16", tree=True),
        # large trees over long contexts: the products count, not the bytes
        dict(name="attention_b8_t64", kind="attention", seqs=8, drafts=64, drafts_min=48, ctx=16000, ctx_min=9000, q_heads=32, kv_heads=8, dim=128,
             page=16, layout="nhd", dtype="bf16", tree=True),
        # sixteen beams of four requests reordered, every layer's ragged page copied
        dict(name="fork_beams16", kind="fork", seqs=16, beams=4, ctx=1500, ctx_min=200, kv_heads=8, dim=128, layers=32, page=16, layout="nhd",
             dtype="bf16"),
        # the accepted paths of a verified batch
        dict(name="compact_b64_t32", kind="compact", seqs=64, drafts=32, accepted=7, ctx=600, ctx_min=40, kv_heads=8, dim=128, layers=32, page=16,
             layout="nhd", dtype="bf16"),
        # a third of a batch has ended and new prompts come in: tables and counts only
        dict(name="admit_b192", kind="admit", seqs=192, ctx=8000, ctx_min=30, prompt=5000, prompt_min=20, drafts=16, pages=65536, page=16),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8), (32, 8), (32, 32), (28, 4), (40, 8), (16, 1), (12, 2), (8, 8), (64, 8), (6, 3)]
_PAGES = [8, 16, 16, 24, 32, 64, 128]


def _rotary(rng, dim):
    return dict(rotary=dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2), interleaved=rng.random() < 0.5,
                base=rng.choice([10000.0, 500000.0, 1000000.0]), scaling=rng.choice(["none", "linear", "stretched", "yarn", "banded"]))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attention", "attention", "attention", "attention", "fork", "compact", "admit"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 128, 128, 128, 80, 96, 256])
    layout = rng.choice(["nhd", "hnd"])
    page = rng.choice(_PAGES)
    q_heads, kv_heads = rng.choice(_HEADS)
    if kind == "rope":
        return dict(kind=kind, rows=_log(rng, 1, 8000), heads=rng.randint(1, 40), dim=dim, far=_log(rng, 100, 200000), dtype=dtype, **_rotary(rng, dim))
    if kind == "append":
        seqs = _log(rng, 1, 96)
        most = _log(rng, 1, max(2, min(4000, 9000 // seqs)))
        return dict(kind=kind, seqs=seqs, drafts=most, drafts_min=rng.randint(1, most), ctx=_log(rng, 30, max(60, 400000 // seqs)), ctx_min=rng.randint(0, 30),
                    q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, layout=layout, dtype=dtype, tree=most <= 64, **_rotary(rng, dim))
    if kind == "attention":
        seqs = _log(rng, 1, 64)
        most = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 64)])
        room = 600_000_000 // (kv_heads * dim * 4)                        # positions whose keys and values take 600 MB
        room = min(room, 34_000_000_000 // (most * q_heads * dim))        # and that the largest listed case's products cover
        ctx = _log(rng, 20, max(30, min(131000, room // seqs)))
        return dict(kind=kind, seqs=seqs, drafts=most, drafts_min=rng.randint(1, most), ctx=ctx, ctx_min=rng.randint(0, min(ctx, 200)), q_heads=q_heads,
                    kv_heads=kv_heads, dim=dim, page=page, layout=layout, dtype=dtype, tree=rng.random() < 0.7)
    if kind == "fork":
        beams = rng.randint(2, 6)
        return dict(kind=kind, seqs=beams * rng.randint(1, 6), beams=beams, ctx=_log(rng, 40, 1500), ctx_min=rng.randint(1, 40),
                    kv_heads=kv_heads if kv_heads < 32 else 8, dim=dim if dim < 256 else 128, layers=rng.randint(1, 32), page=page if page < 128 else 16,
                    layout=layout, dtype=dtype)
    if kind == "compact":
        drafts = _log(rng, 2, 64)
        return dict(kind=kind, seqs=_log(rng, 1, 64), drafts=drafts, accepted=rng.randint(1, min(drafts, 8)), ctx=_log(rng, 20, 500), ctx_min=rng.randint(0, 20),
                    kv_heads=kv_heads if kv_heads < 32 else 8, dim=dim if dim < 256 else 128, layers=rng.randint(1, 24), page=page, layout=layout, dtype=dtype)
    seqs = _log(rng, 1, 192)
    return dict(kind="admit", seqs=seqs, ctx=_log(rng, 50, 8000), ctx_min=rng.randint(0, 50), prompt=_log(rng, 20, 5000), prompt_min=rng.randint(1, 20),
                drafts=rng.randint(1, 64), pages=seqs * 900 + rng.randint(1, 4000), page=rng.choice([16, 24, 32, 64]))


# ------------------------------------------------------------------------------------------------ sizes that go by the case alone
def _spread(lo, hi, n, turn=0.6180339887498949):
    """n whole numbers between lo and hi, spread over their logarithm; the first is hi."""
    return [int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * (1 - (i * turn) % 1.0)))) - 1 for i in range(n)]


def _lengths(case):
    return _spread(case["ctx_min"], case["ctx"], case["seqs"])


def _drafts(case):
    if case["kind"] == "compact":
        return [case["drafts"]] * case["seqs"]
    return _spread(case["drafts_min"], case["drafts"], case["seqs"], turn=0.41421356237309515)


def _accepted(case):
    return [min(case["drafts"], i * 5 % (case["accepted"] + 1)) if i else case["accepted"] for i in range(case["seqs"])]


def _prompts(case):
    return _spread(case["prompt_min"], case["prompt"], case["seqs"], turn=0.7320508075688772)


def _parents(case):
    """Every request keeps its first beam, the others become copies of the first or the second."""
    b = case["beams"]
    return [i if i % b == 0 else i - i % b + (i % b) // 2 % 2 for i in range(case["seqs"])]


def _up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------------------------ prepare
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = dict(case=case, kind=case["kind"])
    if case["kind"] == "rope":
        dt = _DT[case["dtype"]]
        s["x"] = torch.randn((case["rows"], case["heads"], case["dim"]), device=DEV, generator=g).to(dt)
        s["y"] = torch.empty_like(s["x"])
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), dtype=torch.int32, device=DEV, generator=g)
        return s
    _prepare_pool(s, case, g)
    if case["kind"] == "admit":
        ends = [i % 3 == 0 for i in range(case["seqs"])]
        s["which"] = torch.tensor([int(e) for e in ends], dtype=torch.int32, device=DEV)
        s["extra"] = torch.tensor([p if e else case["drafts"] for e, p in zip(ends, _prompts(case))], dtype=torch.int32, device=DEV)
        return s
    if case["kind"] == "fork":
        s["parent"] = torch.tensor(_parents(case), dtype=torch.int32, device=DEV)
    elif case["kind"] == "compact":
        count = _accepted(case)
        order = torch.rand((case["seqs"], case["drafts"]), device=DEV, generator=g).argsort(dim=1)
        most = max(max(count), 1)
        kept = torch.arange(most, device=DEV)[None, :] < torch.tensor(count, device=DEV)[:, None]
        path = torch.where(kept, order[:, :most], 1 << 20).sort(dim=1).values
        s["path"] = torch.where(kept, path, -1).to(torch.int32).contiguous()
        s["path_length"] = torch.tensor(count, dtype=torch.int32, device=DEV)
        s["length_out"] = torch.zeros_like(s["length"])
    else:
        _prepare_rows(s, case, g)
    return s


def _prepare_pool(s, case, g):
    """The pages that the sequences hold, handed out in random order, and what the cache holds in them."""
    n, ps, lens = case["seqs"], case["page"], _lengths(case)
    if case["kind"] == "admit":
        held = [_up(l, ps) for l in lens]
        width = _up(max(case["ctx"] + case["drafts"], case["prompt"] + 1), ps) + 1
        pages = max(case["pages"], sum(held) + 1)
    else:
        ahead = [0] * n if case["kind"] == "fork" else _drafts(case)
        held = [_up(l + t, ps) for l, t in zip(lens, ahead)]
        width = max(held) + 1
        pages = sum(held) + (n if case["kind"] == "fork" else 0) + 3
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    held_t = torch.tensor(held, dtype=torch.int64, device=DEV)
    col = torch.arange(width, device=DEV)[None, :]
    used = col < held_t[:, None]
    first = (held_t.cumsum(0) - held_t)[:, None]
    s["table"] = torch.where(used, order[(first + col).clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    s["length"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["held"] = held_t.to(torch.int32)
    s["refcount"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
    s["refcount"][s["table"][used].long()] = 1
    s["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    s["scratch"] = torch.zeros(64 + 8 * n, dtype=torch.int32, device=DEV)
    s["pages"] = pages
    if case["kind"] != "admit":
        layers, h, d, dt = case.get("layers", 1), case["kv_heads"], case["dim"], _DT[case["dtype"]]
        shape = (layers, pages, ps, h, d) if case["layout"] == "nhd" else (layers, pages, h, ps, d)
        for name in ("k", "v"):
            t = torch.empty(shape, dtype=dt, device=DEV)
            for one in t:                       # layer by layer: the numbers' 32-bit form is not held for all of them
                one.copy_(torch.randn(shape[1:], device=DEV, generator=g))
            # always seen as [layers, pages, slots, heads, dim]
            s[name] = t if case["layout"] == "nhd" else t.permute(0, 1, 3, 2, 4)


def _prepare_rows(s, case, g):
    """What a projection leaves: queries, keys and values of a row side by side; and the rows' trees."""
    counts = _drafts(case)
    rows, hq, hk, d = sum(counts), case["q_heads"], case["kv_heads"], case["dim"]
    qkv = torch.randn((rows, hq + 2 * hk, d), device=DEV, generator=g)
    qkv[:, :hq] *= 1.5
    qkv = qkv.to(_DT[case["dtype"]])
    s["q"], s["key"], s["value"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    s["out"] = torch.zeros((rows, hq, d), dtype=qkv.dtype, device=DEV)
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    s["row_start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
    s["most"] = max(counts)
    s["most_positions"] = max(l + c for l, c in zip(_lengths(case), counts))
    s["mask"], s["positions"] = None, None
    if case["tree"]:
        # node i hangs below one of the nodes before it, most often a late one; it sees its ancestors and itself
        gc = torch.Generator()
        gc.manual_seed(int(torch.randint(0, 2**31, (1,), device=DEV, generator=g).item()))
        n, words = case["seqs"], _up(s["most"], 32)
        sees = torch.zeros((n, s["most"], 32 * words), dtype=torch.bool)
        depth = torch.zeros((n, s["most"]), dtype=torch.int64)
        each = torch.arange(n)
        for i in range(s["most"]):
            if i:
                up = (torch.rand(n, generator=gc).sqrt() * i).long()
                sees[:, i] = sees[each, up]
                depth[:, i] = depth[each, up] + 1
            sees[:, i, i] = True
        bits = (sees.view(n, s["most"], words, 32).long() << torch.arange(32)).sum(-1)
        bits = torch.where(bits >= 2**31, bits - 2**32, bits).to(torch.int32)
        take = torch.arange(s["most"])[None, :] < torch.tensor(counts)[:, None]
        s["mask"] = bits[take].contiguous().to(DEV)
        at = depth + torch.tensor(_lengths(case))[:, None]
        s["positions"] = at[take].to(torch.int32).to(DEV)


# ------------------------------------------------------------------------------------------------ run
def run(state):
    if own:
        if "call" not in state:                 # the argument blocks, filled once as a program does
            state["call"] = _BIND[state["kind"]](state)
        return state["call"]()
    return _PLAIN[state["kind"]](state)


# ---- plain forms
def _frequencies(case):
    """Angle per position of every pair, in 64 bits, and the factor on what is rotated."""
    r, base, kind = case["rotary"], case["base"], case["scaling"]
    i = torch.arange(0, r, 2, dtype=torch.float64, device=DEV)
    f = base ** (-i / r)
    factor, span = 8.0, 8192.0
    if kind == "linear":
        return f / factor, 1.0
    if kind == "stretched":
        return (base * factor ** (r / (r - 2.0))) ** (-i / r) if r > 2 else f, 1.0
    if kind == "yarn":
        def pair(turns):
            return r * math.log(span / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if kind == "banded":
        turns = span * f / (2 * math.pi)
        share = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * ((1 - share) / factor + share), 1.0
    return f, 1.0


def _rotated(x, positions, case):
    f, m = _frequencies(case)
    a = positions.double()[:, None, None] * f
    c, n = (a.cos() * m).float(), (a.sin() * m).float()
    r = case["rotary"]
    x = x.float()
    part, rest = x[..., :r], x[..., r:]
    if case["interleaved"]:
        p, q = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((p * c - q * n, q * c + p * n), dim=-1).flatten(-2)
    else:
        p, q = part[..., :r // 2], part[..., r // 2:]
        turned = torch.cat((p * c - q * n, q * c + p * n), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rope(s):
    s["y"].copy_(_rotated(s["x"], s["positions"], s["case"]))
    return s["y"]


def _plain_append(s):
    case, ps = s["case"], s["case"]["page"]
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["row_start"].long(), row, right=True) - 1
    at = s["length"].long()[seq] + row - s["row_start"].long()[seq]
    turn = at if s["positions"] is None else s["positions"]
    s["out"].copy_(_rotated(s["q"], turn, case))
    page, slot = s["table"].long()[seq, at // ps], at % ps
    s["k"][0].index_put_((page, slot), _rotated(s["key"], turn, case).to(s["k"].dtype))
    s["v"][0].index_put_((page, slot), s["value"])
    return s["out"], s["k"], s["v"]


def _plain_attention(s):
    case, ps = s["case"], s["case"]["page"]
    hq, hk, d, t, n = case["q_heads"], case["kv_heads"], case["dim"], s["most"], case["seqs"]
    start, length = s["row_start"].long(), s["length"].long()
    count = start[1:] - start[:-1]
    pos = torch.arange(s["most_positions"], device=DEV)
    page = s["table"].long()[:, pos // ps]
    there = (pos < (length + count)[:, None]) & (page >= 0)
    page, slot = page.clamp(min=0), (pos % ps)[None, :]
    k = torch.where(there[..., None, None], s["k"][0][page, slot], 0).float()
    v = torch.where(there[..., None, None], s["v"][0][page, slot], 0).float()
    node = torch.arange(t, device=DEV)
    row = (start[:-1, None] + node).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().view(n, t, hk, hq // hk, d)
    ahead = pos[None, :] - length[:, None]                                # which drafted node stands at a position
    if s["mask"] is None:
        sees = ahead[:, None, :] <= node[None, :, None]
    else:
        words = s["mask"].long()[row]                                     # [seqs, nodes, words]
        last = words.shape[-1] * 32 - 1
        word = words.gather(2, (ahead.clamp(0, last) // 32)[:, None, :].expand(-1, t, -1))
        bit = (word >> (ahead.clamp(0, last) % 32)[:, None, :]) & 1
        sees = (ahead[:, None, :] < 0) | ((bit != 0) & (ahead[:, None, :] <= last))
    sees = (sees & there[:, None, :])[:, None, None]
    score = torch.einsum("nthgd,nkhd->nhgtk", q, k) * (1.0 / math.sqrt(d))
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    o = torch.einsum("nhgtk,nkhd->nthgd", e, v)
    total = e.sum(-1).permute(0, 3, 1, 2)[..., None]
    o = (o / torch.where(total == 0, 1.0, total)).reshape(n, t, hq, d)
    real = node[None, :] < count[:, None]
    s["out"][row[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def _plain_fork(s):
    ps, n = s["case"]["page"], s["case"]["seqs"]
    each = torch.arange(n, device=DEV)
    parent = s["parent"].long()
    child = (parent >= 0) & (parent < n) & (parent != each)
    of = torch.where(child, parent, each)
    old, length, held = s["table"].long(), s["length"].long(), s["held"].long()
    count, full = length[of], length[of] // ps
    ragged = child & (count % ps != 0)
    free = (s["refcount"] == 0).nonzero().flatten()
    if int(ragged.sum()) > free.numel():
        s["status"].fill_(1)
        return _fork_outputs(s)
    new = torch.where(ragged, free[(ragged.cumsum(0) - 1).clamp(min=0)], -1)
    col = torch.arange(old.shape[1], device=DEV)[None, :]
    shared = child[:, None] & (col < full[:, None])
    dropped = child[:, None] & (col < held[:, None])
    row = torch.where(col < full[:, None], old[of], -1)
    row = torch.where((col == full[:, None]) & ragged[:, None], new[:, None], row)
    s["table"].copy_(torch.where(child[:, None], row, old))
    one = torch.ones((), dtype=torch.int32, device=DEV)
    s["refcount"].index_add_(0, old[of][shared], one.expand(int(shared.sum())))
    s["refcount"].index_add_(0, old[dropped], -one.expand(int(dropped.sum())))
    s["refcount"][new[ragged]] = 1
    src, dst = old[of, full.clamp(max=old.shape[1] - 1)], new
    slot = torch.arange(ps, device=DEV)[None, :]
    moved = ragged[:, None] & (slot < (count % ps)[:, None])
    a, b, at = src[:, None].expand(-1, ps)[moved], dst[:, None].expand(-1, ps)[moved], slot.expand(n, -1)[moved]
    s["k"][:, b, at] = s["k"][:, a, at]
    s["v"][:, b, at] = s["v"][:, a, at]
    s["held"].copy_(torch.where(child, full + ragged.long(), held))
    s["length"].copy_(count)
    return _fork_outputs(s)


def _fork_outputs(s):
    return s["table"], s["length"], s["held"], s["refcount"], s["status"], s["k"], s["v"]


def _plain_compact(s):
    ps = s["case"]["page"]
    step = torch.arange(s["path"].shape[1], device=DEV)[None, :]
    moved = step < s["path_length"].long()[:, None]
    length, table = s["length"].long(), s["table"].long()
    src = (length[:, None] + s["path"].long().clamp(min=0))
    dst = length[:, None] + step
    last = table.shape[1] * ps - 1
    a, b = src.clamp(max=last), dst.clamp(max=last)
    pa, pb = table.gather(1, a // ps)[moved], table.gather(1, b // ps)[moved]
    sa, sb = (a % ps)[moved], (b % ps)[moved]
    s["k"][:, pb, sb] = s["k"][:, pa, sa]
    s["v"][:, pb, sb] = s["v"][:, pa, sa]
    s["length_out"].copy_(length + s["path_length"])
    return s["length_out"], s["k"], s["v"]


def _plain_admit(s):
    ps = s["case"]["page"]
    col = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    ends = s["which"] != 0
    given = ends[:, None] & (col < s["held"].long()[:, None])
    one = torch.ones((), dtype=torch.int32, device=DEV)
    s["refcount"].index_add_(0, s["table"].long()[given], -one.expand(int(given.sum())))
    s["table"].masked_fill_(given, -1)
    s["length"].masked_fill_(ends, 0)
    s["held"].masked_fill_(ends, 0)
    want = (s["length"].long() + s["extra"].long() + ps - 1) // ps
    need = (want - s["held"].long()).clamp(min=0)
    need = torch.where(s["extra"] >= 0, need, 0)
    total = int(need.sum())
    free = (s["refcount"] == 0).nonzero().flatten()
    if total > free.numel() or bool((want > s["table"].shape[1]).any()):
        s["status"].fill_(1)
    else:
        end = need.cumsum(0)
        k = torch.arange(total, device=DEV)
        seq = torch.searchsorted(end, k, right=True)
        s["table"][seq, s["held"].long()[seq] + k - (end - need)[seq]] = free[:total].to(torch.int32)
        s["refcount"][free[:total]] = 1
        s["held"] += need.to(torch.int32)
    return s["table"], s["length"], s["held"], s["refcount"], s["status"]


_PLAIN = dict(rope=_plain_rope, append=_plain_append, attention=_plain_attention, fork=_plain_fork, compact=_plain_compact, admit=_plain_admit)


# ---- the library's calls
def _library():
    import ctypes
    import tpu_mlir_b200._lib as L
    return ctypes, L, L.lib()


def _plan(case):
    C, L, lib = _library()
    kind = {"none": L.ROPE_SCALING_NONE, "linear": L.ROPE_SCALING_LINEAR, "stretched": L.ROPE_SCALING_STRETCHED, "yarn": L.ROPE_SCALING_YARN,
            "banded": L.ROPE_SCALING_BANDED}[case["scaling"]]
    low, high = (1.0, 32.0) if case["scaling"] == "yarn" else (1.0, 4.0)
    scaling = L.RopeScaling(kind=kind, factor=8.0, original_positions=8192.0, low_turns=low, high_turns=high)
    plan = L.RopePlan()
    L.check(lib.b200q_rope_plan_init(C.byref(plan), case["dim"], case["rotary"], int(case["interleaved"]), case["base"], C.byref(scaling)))
    return plan


def _dtype(case):
    _, L, _ = _library()
    return L.DT_F16 if case["dtype"] == "f16" else L.DT_BF16


def _cache(s):
    _, L, _ = _library()
    k = s["k"]
    return L.KvCache(k=k.data_ptr(), v=s["v"].data_ptr(), layer_stride=k.stride(0), page_stride=k.stride(1), slot_stride=k.stride(2),
                     head_stride=k.stride(3), layers=k.shape[0], heads=k.shape[3], head_dim=k.shape[4], dtype=_dtype(s["case"]))


def _pool(s):
    _, L, _ = _library()
    return L.KvPool(table=s["table"].data_ptr(), length=s["length"].data_ptr(), held=s["held"].data_ptr(), refcount=s["refcount"].data_ptr(),
                    scratch=s["scratch"].data_ptr(), table_stride=s["table"].stride(0), sequences=s["case"]["seqs"], table_width=s["table"].shape[1],
                    pages=s["pages"], page_size=s["case"]["page"], scratch_words=s["scratch"].numel())


def _caller(keep, outputs, *calls):
    """One pass: the calls on the current stream, in order."""
    C, L, _ = _library()
    check = L.check

    def call():
        stream = torch.cuda.current_stream().cuda_stream
        for f, args in calls:
            rc = f(*args, stream)
            if rc:
                check(rc)
        return outputs
    call.keep = keep
    return call


def _bind_rope(s):
    C, L, lib = _library()
    x, y, plan = s["x"], s["y"], _plan(s["case"])
    args = (C.byref(plan), x.data_ptr(), y.data_ptr(), s["positions"].data_ptr(), x.shape[0], x.shape[1], x.stride(0), x.stride(1), y.stride(0),
            y.stride(1), _dtype(s["case"]))
    return _caller((plan,), y, (lib.b200q_rope_dev, args))


def _bind_append(s):
    C, L, lib = _library()
    plan, cache, pool = _plan(s["case"]), _cache(s), _pool(s)
    q, k, v, o = s["q"], s["key"], s["value"], s["out"]
    a = L.RopeAppend(q=q.data_ptr(), q_out=o.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), row_start=s["row_start"].data_ptr(),
                     positions=None if s["positions"] is None else s["positions"].data_ptr(), q_row_stride=q.stride(0), q_head_stride=q.stride(1),
                     q_out_row_stride=o.stride(0), q_out_head_stride=o.stride(1), k_row_stride=k.stride(0), k_head_stride=k.stride(1),
                     v_row_stride=v.stride(0), v_head_stride=v.stride(1), rows=q.shape[0], q_heads=q.shape[1], layer=0)
    args = tuple(C.byref(b) for b in (plan, cache, pool, a))
    return _caller((plan, cache, pool, a), (o, s["k"], s["v"]), (lib.b200q_rope_append_dev, args))


def _bind_attention(s):
    C, L, lib = _library()
    cache, pool, q, o = _cache(s), _pool(s), s["q"], s["out"]
    need = C.c_int64()
    L.check(lib.b200q_tree_attention_workspace(C.byref(cache), q.shape[1], C.byref(need)))
    space = torch.empty(need.value, dtype=torch.uint8, device=DEV)
    m = s["mask"]
    a = L.TreeAttention(q=q.data_ptr(), out=o.data_ptr(), row_start=s["row_start"].data_ptr(), mask=None if m is None else m.data_ptr(),
                        workspace=space.data_ptr(), workspace_bytes=need.value, q_row_stride=q.stride(0), q_head_stride=q.stride(1),
                        out_row_stride=o.stride(0), out_head_stride=o.stride(1), mask_stride=0 if m is None else m.stride(0), rows=q.shape[0],
                        q_heads=q.shape[1], layer=0, scale=1.0 / math.sqrt(q.shape[2]))
    args = tuple(C.byref(b) for b in (cache, pool, a))
    return _caller((cache, pool, a, space), o, (lib.b200q_tree_attention_dev, args))


def _bind_fork(s):
    C, L, lib = _library()
    cache, pool = _cache(s), _pool(s)
    args = (C.byref(cache), C.byref(pool), s["parent"].data_ptr(), s["status"].data_ptr())
    return _caller((cache, pool), _fork_outputs(s), (lib.b200q_kv_fork_dev, args))


def _bind_compact(s):
    C, L, lib = _library()
    cache, pool, path = _cache(s), _pool(s), s["path"]
    args = (C.byref(cache), C.byref(pool), path.data_ptr(), path.stride(0), path.shape[1], s["path_length"].data_ptr(), s["length_out"].data_ptr())
    return _caller((cache, pool), (s["length_out"], s["k"], s["v"]), (lib.b200q_kv_compact_dev, args))


def _bind_admit(s):
    C, L, lib = _library()
    pool = _pool(s)
    free = (C.byref(pool), s["which"].data_ptr())
    reserve = (C.byref(pool), s["extra"].data_ptr(), s["status"].data_ptr())
    return _caller((pool,), (s["table"], s["length"], s["held"], s["refcount"], s["status"]), (lib.b200q_kv_free_dev, free),
                   (lib.b200q_kv_reserve_dev, reserve))


_BIND = dict(rope=_bind_rope, append=_bind_append, attention=_bind_attention, fork=_bind_fork, compact=_bind_compact, admit=_bind_admit)


# ------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """What run returns, from the definitions: 64-bit numbers, one sequence, head or page after another."""
    return _EXACT[case["kind"]](case, prepare(case, seed))


def _turned(case, x, positions):
    """Pair by pair, as a product of complex numbers."""
    r, base, kind, factor, span = case["rotary"], case["base"], case["scaling"], 8.0, 8192.0
    if kind == "stretched" and r > 2:
        base = base * math.pow(factor, r / (r - 2))
    if kind == "yarn":
        first = max(0, math.floor(r / 2 * math.log(span / 32.0 / (2 * math.pi), base)))
        last = min(r - 1, math.ceil(r / 2 * math.log(span / (2 * math.pi), base)))
    y = x.double().clone()
    for i in range(r // 2):
        w = math.exp(-2 * i / r * math.log(base))
        size = 1.0
        if kind == "linear":
            w /= factor
        elif kind == "yarn":
            mix = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            w = mix * w / factor + (1 - mix) * w
            size = 1 + math.log(factor) / 10
        elif kind == "banded":
            length = 2 * math.pi / w
            if length > span / 1.0:
                w /= factor
            elif length >= span / 4.0:
                mix = (span / length - 1.0) / 3.0
                w = (1 - mix) * w / factor + mix * w
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        z = torch.complex(x[..., a].double(), x[..., b].double()) * torch.polar(torch.full_like(positions, size, dtype=torch.float64),
                                                                              positions.double() * w)[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_rope(case, s):
    return _turned(case, s["x"], s["positions"])


def _exact_append(case, s):
    k, v = s["k"].double(), s["v"].double()
    lens, table, ps, at, row = _lengths(case), s["table"].tolist(), case["page"], [], 0
    where = []
    for n, count in enumerate(_drafts(case)):
        for i in range(count):
            p = lens[n] + i
            at.append(p)
            where.append(table[n][p // ps] * ps + p % ps)
    at = torch.tensor(at, device=DEV) if s["positions"] is None else s["positions"]
    where = torch.tensor(where, device=DEV)
    k[0, where // ps, where % ps] = _turned(case, s["key"], at)
    v[0, where // ps, where % ps] = s["value"].double()
    return _turned(case, s["q"], at), k, v


def _exact_attention(case, s):
    ps, d, per = case["page"], case["dim"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for n, (length, count) in enumerate(zip(_lengths(case), _drafts(case))):
        total = length + count
        pages = s["table"][n, :_up(total, ps)].long()
        k = s["k"][0].index_select(0, pages).flatten(0, 1)[:total]
        v = s["v"][0].index_select(0, pages).flatten(0, 1)[:total]
        seen = torch.ones((count, total), dtype=torch.bool, device=DEV)
        if s["mask"] is None:
            seen[:, length:] = torch.ones((count, count), dtype=torch.bool, device=DEV).tril()
        else:
            for j in range(count):
                seen[:, length + j] = s["mask"][row:row + count, j // 32].long().bitwise_and(1 << (j % 32)).ne(0)
        for h in range(case["kv_heads"]):
            q = s["q"][row:row + count, h * per:(h + 1) * per].double().transpose(0, 1)
            w = (q @ k[:, h].double().t() / math.sqrt(d)).masked_fill(~seen, -math.inf).softmax(-1)
            out[row:row + count, h * per:(h + 1) * per] = (w @ v[:, h].double()).transpose(0, 1)
        row += count
    return out


def _lowest(count, busy):
    """The `count` lowest pages that nobody holds."""
    found, page = [], 0
    while len(found) < count:
        if not busy[page]:
            found.append(page)
        page += 1
    return found


def _exact_fork(case, s):
    ps, parents = case["page"], _parents(case)
    table, lens, held, refs = s["table"].tolist(), s["length"].tolist(), s["held"].tolist(), s["refcount"].tolist()
    before, old_lens, old_held = [list(r) for r in table], list(lens), list(held)
    k, v = s["k"].double(), s["v"].double()
    ragged = [i for i, p in enumerate(parents) if p != i and old_lens[p] % ps]
    new = dict(zip(ragged, _lowest(len(ragged), refs)))
    for i, p in enumerate(parents):
        if p == i:
            continue
        full = old_lens[p] // ps
        table[i] = before[p][:full] + [-1] * (len(before[p]) - full)
        for page in before[p][:full]:
            refs[page] += 1
        for page in before[i][:old_held[i]]:
            refs[page] -= 1
        if i in new:
            table[i][full] = new[i]
            refs[new[i]] += 1
            part = old_lens[p] % ps
            k[:, new[i], :part], v[:, new[i], :part] = k[:, before[p][full], :part], v[:, before[p][full], :part]
        held[i], lens[i] = full + (i in new), old_lens[p]
    whole = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, lens, held, refs, [0])]
    return (*whole, k, v)


def _exact_compact(case, s):
    ps, table, lens, path = case["page"], s["table"].tolist(), s["length"].tolist(), s["path"].tolist()
    k, v = s["k"].double(), s["v"].double()
    after = []
    for n, count in enumerate(_accepted(case)):
        for i in range(count):
            a, b = lens[n] + path[n][i], lens[n] + i
            for t in (k, v):
                t[:, table[n][b // ps], b % ps] = t[:, table[n][a // ps], a % ps]
        after.append(lens[n] + count)
    return torch.tensor(after, dtype=torch.int32, device=DEV), k, v


def _exact_admit(case, s):
    ps, table, lens, held, refs = case["page"], s["table"].tolist(), s["length"].tolist(), s["held"].tolist(), s["refcount"].tolist()
    prompts = _prompts(case)
    for n in range(0, case["seqs"], 3):
        for j in range(held[n]):
            refs[table[n][j]] -= 1
            table[n][j] = -1
        lens[n] = held[n] = 0
    want = [_up(lens[n] + (prompts[n] if n % 3 == 0 else case["drafts"]), ps) for n in range(case["seqs"])]
    free = [p for p, c in enumerate(refs) if c == 0]
    for n in range(case["seqs"]):
        while held[n] < want[n]:
            page = free.pop(0)
            table[n][held[n]] = page
            refs[page] = 1
            held[n] += 1
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, lens, held, refs, [0]))


_EXACT = dict(rope=_exact_rope, append=_exact_append, attention=_exact_attention, fork=_exact_fork, compact=_exact_compact, admit=_exact_admit)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["rows"] * case["heads"] * case["dim"]
        return dict(bytes=4.0 * n + 4 * case["rows"], flops=3.0 * case["rows"] * case["heads"] * case["rotary"])
    lens = _lengths(case)
    if kind == "admit":
        ps = case["page"]
        given = [_up(p, ps) for i, p in enumerate(_prompts(case)) if i % 3 == 0]
        # a page given back: its entry read and cleared, its count read and written; a page handed out: entry and count written
        return dict(bytes=4.0 * case["pages"] + 24.0 * sum(given) + 24.0 * case["seqs"], flops=0)
    hk, d = case["kv_heads"], case["dim"]
    if kind == "fork":
        ps, parents = case["page"], _parents(case)
        moved = sum(lens[p] % ps for i, p in enumerate(parents) if p != i)
        entries = sum(_up(lens[p], ps) + _up(lens[i], ps) for i, p in enumerate(parents) if p != i)
        return dict(bytes=8.0 * moved * case["layers"] * hk * d + 16.0 * entries, flops=0)
    if kind == "compact":
        return dict(bytes=8.0 * sum(_accepted(case)) * case["layers"] * hk * d + 12.0 * case["seqs"], flops=0)
    counts, hq = _drafts(case), case["q_heads"]
    rows = sum(counts)
    if kind == "append":
        return dict(bytes=4.0 * rows * (hq + 2 * hk) * d + 8.0 * rows, flops=3.0 * rows * (hq + hk) * case["rotary"])
    pairs = sum(t * (l + t) for l, t in zip(lens, counts))
    return dict(bytes=4.0 * hk * d * sum(l + t for l, t in zip(lens, counts)) + 4.0 * rows * hq * d, flops=4.0 * pairs * hq * d)
