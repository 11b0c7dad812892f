"""The decoding operators' host side: what is refused before anything reaches a device, and the rotary frequencies."""
import ctypes as C
import math

import pytest

import tpu_mlir_b200._lib as L
from decode_model import frequencies

FAKE = 0x10000          # an aligned address that no refused call looks at


@pytest.fixture(scope="module")
def lib():
    L.build()
    return L.lib()


def pool(**kw):
    d = dict(table=FAKE, length=FAKE, held=FAKE, refcount=FAKE, scratch=FAKE, table_stride=8, sequences=4, table_width=8, pages=32, page_size=16, scratch_words=1000)
    d.update(kw)
    return L.KvPool(**d)


def cache(**kw):
    d = dict(k=FAKE, v=FAKE, layer_stride=32 * 16 * 2 * 64, page_stride=16 * 2 * 64, slot_stride=2 * 64, head_stride=64, layers=3, heads=2, head_dim=64, dtype=L.DT_BF16)
    d.update(kw)
    return L.KvCache(**d)


def attention(**kw):
    d = dict(q=FAKE, out=FAKE, row_start=FAKE, mask=FAKE, workspace=FAKE, workspace_bytes=1 << 30, q_row_stride=256, q_head_stride=64, out_row_stride=256,
             out_head_stride=64, mask_stride=1, rows=4, q_heads=4, layer=0, scale=0.125)
    d.update(kw)
    return L.TreeAttention(**d)


def append(**kw):
    d = dict(q=FAKE, q_out=FAKE + 4096, k=FAKE, v=FAKE, row_start=FAKE, positions=None, q_row_stride=256, q_head_stride=64, q_out_row_stride=256,
             q_out_head_stride=64, k_row_stride=128, k_head_stride=64, v_row_stride=128, v_head_stride=64, rows=4, q_heads=4, layer=0)
    d.update(kw)
    return L.RopeAppend(**d)


def plan(**kw):
    p = L.RopePlan(head_dim=64, rotary_dim=64, interleaved=0, magnitude=1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def refused(lib, rc, code, word):
    assert rc == code, lib.b200q_last_error()
    assert word in lib.b200q_last_error(), lib.b200q_last_error()


BAD_POOLS = [(dict(table=None), L.ERR_INVALID, b"null"), (dict(length=None), L.ERR_INVALID, b"null"), (dict(held=None), L.ERR_INVALID, b"null"),
             (dict(refcount=None), L.ERR_INVALID, b"null"), (dict(refcount=FAKE + 2), L.ERR_INVALID, b"aligned"), (dict(sequences=-1), L.ERR_INVALID, b"shape"),
             (dict(table_width=0), L.ERR_INVALID, b"shape"), (dict(table_stride=7), L.ERR_INVALID, b"shape"), (dict(pages=0), L.ERR_INVALID, b"shape"),
             (dict(page_size=0), L.ERR_INVALID, b"shape"), (dict(sequences=1025), L.ERR_UNSUPPORTED, b"1024"), (dict(pages=(1 << 20) + 1), L.ERR_UNSUPPORTED, b"pages"),
             (dict(page_size=1 << 28), L.ERR_UNSUPPORTED, b"positions")]
BAD_CACHES = [(dict(k=None), L.ERR_INVALID, b"null"), (dict(v=None), L.ERR_INVALID, b"null"), (dict(v=FAKE + 8), L.ERR_INVALID, b"aligned"),
              (dict(dtype=L.DT_F32), L.ERR_UNSUPPORTED, b"bf16"), (dict(layers=0), L.ERR_INVALID, b"shape"), (dict(heads=0), L.ERR_INVALID, b"shape"),
              (dict(head_dim=0), L.ERR_INVALID, b"shape"), (dict(head_dim=60), L.ERR_UNSUPPORTED, b"head_dim"), (dict(head_dim=264), L.ERR_UNSUPPORTED, b"head_dim"),
              (dict(slot_stride=132), L.ERR_INVALID, b"strides"), (dict(page_stride=1), L.ERR_INVALID, b"strides"),
              (dict(head_stride=0), L.ERR_INVALID, b"positive"), (dict(slot_stride=-128), L.ERR_INVALID, b"positive"), (dict(layer_stride=-8), L.ERR_INVALID, b"positive"),
              (dict(page_stride=1 << 38), L.ERR_INVALID, b"positive")]


def calls(lib, c, p, a=None, r=None, pl=None):
    """Every entry point with these blocks: those that take the cache, then those that do not."""
    c, p, a, r, pl = C.byref(c), C.byref(p), C.byref(a or attention()), C.byref(r or append()), C.byref(pl or plan())
    yield True, lambda: lib.b200q_kv_fork_dev(c, p, FAKE, None, None)
    yield True, lambda: lib.b200q_kv_compact_dev(c, p, FAKE, 4, 4, FAKE, FAKE + 4096, None)
    yield True, lambda: lib.b200q_rope_append_dev(pl, c, p, r, None)
    yield True, lambda: lib.b200q_tree_attention_dev(c, p, a, None)
    yield False, lambda: lib.b200q_kv_reserve_dev(p, FAKE, None, None)
    yield False, lambda: lib.b200q_kv_free_dev(p, FAKE, None)


@pytest.mark.parametrize("kw,code,word", BAD_POOLS)
def test_bad_pools(lib, kw, code, word):
    for _, call in calls(lib, cache(), pool(**kw)):
        refused(lib, call(), code, word)


@pytest.mark.parametrize("kw,code,word", BAD_CACHES)
def test_bad_caches(lib, kw, code, word):
    for takes, call in calls(lib, cache(**kw), pool()):
        if takes:
            refused(lib, call(), code, word)
    n = C.c_int64()
    refused(lib, lib.b200q_tree_attention_workspace(C.byref(cache(**kw)), 4, C.byref(n)), code, word)


def test_null_blocks(lib):
    c, p, pl = C.byref(cache()), C.byref(pool()), C.byref(plan())
    for rc in (lib.b200q_kv_reserve_dev(None, FAKE, None, None), lib.b200q_kv_reserve_dev(p, None, None, None), lib.b200q_kv_free_dev(None, FAKE, None),
               lib.b200q_kv_free_dev(p, None, None), lib.b200q_kv_fork_dev(None, p, FAKE, None, None), lib.b200q_kv_fork_dev(c, None, FAKE, None, None),
               lib.b200q_kv_fork_dev(c, p, None, None, None), lib.b200q_kv_compact_dev(None, p, FAKE, 4, 4, FAKE, FAKE, None),
               lib.b200q_kv_compact_dev(c, None, FAKE, 4, 4, FAKE, FAKE, None), lib.b200q_kv_compact_dev(c, p, None, 4, 4, FAKE, FAKE, None),
               lib.b200q_kv_compact_dev(c, p, FAKE, 4, 4, None, FAKE, None), lib.b200q_kv_compact_dev(c, p, FAKE, 4, 4, FAKE, None, None),
               lib.b200q_rope_append_dev(None, c, p, C.byref(append()), None), lib.b200q_rope_append_dev(pl, None, p, C.byref(append()), None),
               lib.b200q_rope_append_dev(pl, c, None, C.byref(append()), None), lib.b200q_rope_append_dev(pl, c, p, None, None),
               lib.b200q_tree_attention_dev(None, p, C.byref(attention()), None), lib.b200q_tree_attention_dev(c, None, C.byref(attention()), None),
               lib.b200q_tree_attention_dev(c, p, None, None), lib.b200q_tree_attention_workspace(c, 4, None),
               lib.b200q_rope_dev(None, FAKE, FAKE, FAKE, 1, 1, 64, 64, 64, 64, L.DT_BF16, None), lib.b200q_rope_plan_init(None, 64, 64, 0, 10000.0, None)):
        refused(lib, rc, L.ERR_INVALID, b"")


@pytest.mark.parametrize("kw,code,word", [(dict(q=None), L.ERR_INVALID, b"null"), (dict(out=None), L.ERR_INVALID, b"null"), (dict(row_start=None), L.ERR_INVALID, b"null"),
                                          (dict(workspace=None), L.ERR_INVALID, b"null"), (dict(q=FAKE + 8), L.ERR_INVALID, b"aligned"),
                                          (dict(workspace=FAKE + 4), L.ERR_INVALID, b"aligned"), (dict(mask=FAKE + 1), L.ERR_INVALID, b"aligned"),
                                          (dict(q_row_stride=260), L.ERR_INVALID, b"strides"), (dict(out_head_stride=68), L.ERR_INVALID, b"strides"),
                                          (dict(q_heads=3), L.ERR_INVALID, b"q_heads"), (dict(q_heads=0), L.ERR_INVALID, b"q_heads"), (dict(rows=-1), L.ERR_INVALID, b"rows"),
                                          (dict(rows=1 << 31), L.ERR_INVALID, b"rows"), (dict(rows=(1 << 31) - 1), L.ERR_UNSUPPORTED, b"rows"),
                                          (dict(layer=3), L.ERR_INVALID, b"layer"), (dict(layer=-1), L.ERR_INVALID, b"layer"), (dict(scale=0.0), L.ERR_INVALID, b"scale"),
                                          (dict(scale=-1.0), L.ERR_INVALID, b"scale"), (dict(scale=float("nan")), L.ERR_INVALID, b"scale"),
                                          (dict(scale=float("inf")), L.ERR_INVALID, b"scale"), (dict(mask_stride=-1), L.ERR_INVALID, b"mask_stride")])
def test_bad_attention(lib, kw, code, word):
    refused(lib, lib.b200q_tree_attention_dev(C.byref(cache()), C.byref(pool()), C.byref(attention(**kw)), None), code, word)


@pytest.mark.parametrize("kw,code,word", [(dict(q=None), L.ERR_INVALID, b"null"), (dict(q_out=None), L.ERR_INVALID, b"null"), (dict(k=None), L.ERR_INVALID, b"null"),
                                          (dict(v=None), L.ERR_INVALID, b"null"), (dict(row_start=None), L.ERR_INVALID, b"null"), (dict(v=FAKE + 1), L.ERR_INVALID, b"aligned"),
                                          (dict(positions=FAKE + 2), L.ERR_INVALID, b"aligned"), (dict(layer=3), L.ERR_INVALID, b"layer"), (dict(rows=-1), L.ERR_INVALID, b"shape"),
                                          (dict(q_heads=-1), L.ERR_INVALID, b"shape"), (dict(q_heads=70000), L.ERR_UNSUPPORTED, b"heads"),
                                          (dict(q_out=FAKE, q_out_row_stride=512), L.ERR_INVALID, b"in place")])
def test_bad_append(lib, kw, code, word):
    refused(lib, lib.b200q_rope_append_dev(C.byref(plan()), C.byref(cache()), C.byref(pool()), C.byref(append(**kw)), None), code, word)


def test_append_wants_the_caches_head(lib):
    refused(lib, lib.b200q_rope_append_dev(C.byref(plan(head_dim=128)), C.byref(cache()), C.byref(pool()), C.byref(append()), None), L.ERR_INVALID, b"head_dim")


@pytest.mark.parametrize("kw,code,word", [(dict(rotary_dim=66), L.ERR_INVALID, b"rotary_dim"), (dict(rotary_dim=7), L.ERR_INVALID, b"even"), (dict(rotary_dim=-2), L.ERR_INVALID, b"rotary"),
                                          (dict(head_dim=258), L.ERR_INVALID, b"256"), (dict(head_dim=0, rotary_dim=0), L.ERR_INVALID, b"head_dim")])
def test_bad_plans(lib, kw, code, word):
    refused(lib, lib.b200q_rope_dev(C.byref(plan(**kw)), FAKE, FAKE, FAKE, 1, 1, 64, 64, 64, 64, L.DT_BF16, None), code, word)
    p = L.RopePlan()
    p.head_dim = 77
    refused(lib, lib.b200q_rope_plan_init(C.byref(p), kw.get("head_dim", 64), kw.get("rotary_dim", 64), 0, 10000.0, None), code, word)
    assert p.head_dim == 77, "a refused plan was written"


def test_bad_rope(lib):
    def rope(x=FAKE, y=FAKE, pos=FAKE, rows=1, heads=1, strides=(64, 64, 64, 64), dtype=L.DT_BF16):
        return lib.b200q_rope_dev(C.byref(plan()), x, y, pos, rows, heads, *strides, dtype, None)
    refused(lib, rope(x=None), L.ERR_INVALID, b"null")
    refused(lib, rope(y=None), L.ERR_INVALID, b"null")
    refused(lib, rope(pos=None), L.ERR_INVALID, b"null")
    refused(lib, rope(rows=-1), L.ERR_INVALID, b"shape")
    refused(lib, rope(heads=-1), L.ERR_INVALID, b"shape")
    refused(lib, rope(heads=65536), L.ERR_UNSUPPORTED, b"heads")
    refused(lib, rope(dtype=L.DT_F32), L.ERR_UNSUPPORTED, b"dtype")
    refused(lib, rope(x=FAKE + 1), L.ERR_INVALID, b"aligned")
    refused(lib, rope(pos=FAKE + 1), L.ERR_INVALID, b"aligned")
    refused(lib, rope(strides=(64, 64, 128, 64)), L.ERR_INVALID, b"in place")


def test_bad_scaling(lib):
    p = L.RopePlan()

    def init(base=10000.0, **kw):
        d = dict(kind=L.ROPE_SCALING_YARN, factor=4.0, original_positions=4096.0, low_turns=1.0, high_turns=32.0)
        d.update(kw)
        return lib.b200q_rope_plan_init(C.byref(p), 64, 64, 0, base, C.byref(L.RopeScaling(**d)))
    assert init() == L.OK
    nan = float("nan")
    for kw in (dict(kind=5), dict(kind=-1), dict(factor=0.5), dict(factor=nan), dict(factor=float("inf")), dict(original_positions=0.0), dict(original_positions=nan),
               dict(low_turns=0.0), dict(low_turns=32.0), dict(high_turns=nan), dict(base=1.0), dict(base=nan), dict(base=float("inf"))):
        refused(lib, init(**kw), L.ERR_INVALID, b"rope_plan_init")


def test_bad_paths_and_scratch(lib):
    c, p = C.byref(cache()), C.byref(pool())
    refused(lib, lib.b200q_kv_compact_dev(c, p, FAKE, 3, 4, FAKE, FAKE + 4096, None), L.ERR_INVALID, b"paths")
    refused(lib, lib.b200q_kv_compact_dev(c, p, FAKE, 4, -1, FAKE, FAKE + 4096, None), L.ERR_INVALID, b"paths")
    refused(lib, lib.b200q_kv_compact_dev(c, p, FAKE, 2000, 1025, FAKE, FAKE + 4096, None), L.ERR_UNSUPPORTED, b"1024")
    words = lib.b200q_kv_scratch_words(4)
    assert 0 < lib.b200q_kv_scratch_words(0) <= words < lib.b200q_kv_scratch_words(5)
    for few in (dict(scratch=None), dict(scratch_words=words - 1)):
        refused(lib, lib.b200q_kv_fork_dev(c, C.byref(pool(**few)), FAKE, None, None), L.ERR_INVALID, b"scratch")
        refused(lib, lib.b200q_kv_compact_dev(c, C.byref(pool(**few)), FAKE, 4, 4, FAKE, FAKE, None), L.ERR_INVALID, b"scratch")   # in place: length_out is the pool's
    refused(lib, lib.b200q_kv_fork_dev(C.byref(cache(heads=65535, head_dim=256)), C.byref(pool(page_size=1 << 20)), FAKE, None, None), L.ERR_UNSUPPORTED, b"page")


def test_nothing_to_do_needs_no_device(lib):
    for _, call in calls(lib, cache(), pool(sequences=0)):
        assert call() == L.OK
    assert lib.b200q_tree_attention_dev(C.byref(cache()), C.byref(pool()), C.byref(attention(rows=0)), None) == L.OK
    assert lib.b200q_rope_append_dev(C.byref(plan()), C.byref(cache()), C.byref(pool()), C.byref(append(rows=0)), None) == L.OK
    assert lib.b200q_rope_dev(C.byref(plan()), FAKE, FAKE, FAKE, 0, 1, 64, 64, 64, 64, L.DT_BF16, None) == L.OK


def test_a_host_pointer_is_an_error_and_not_a_fault(lib):
    """With a device: not device memory.  Without one: no device.  Either way a status."""
    import numpy as np
    host = np.zeros(4096, np.int32)
    at = (host.ctypes.data + 15) // 16 * 16
    p = pool(table=at, length=at, held=at, refcount=at, scratch=at)
    for _, call in calls(lib, cache(k=at, v=at), p):
        assert call() < 0 and lib.b200q_last_error()


@pytest.mark.parametrize("rotary", [2, 4, 22, 64, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("kind,factor,span,low,high", [("none", 1.0, 0, 0, 0), ("linear", 4.0, 0, 0, 0), ("stretched", 8.0, 0, 0, 0), ("yarn", 16.0, 4096.0, 1.0, 32.0),
                                                       ("yarn", 1.0, 131072.0, 2.0, 3.0), ("banded", 8.0, 8192.0, 1.0, 4.0)])
def test_frequencies(lib, rotary, base, kind, factor, span, low, high):
    p = L.RopePlan()
    code = ["none", "linear", "stretched", "yarn", "banded"].index(kind)
    sc = L.RopeScaling(kind=code, factor=factor, original_positions=span, low_turns=low, high_turns=high)
    assert lib.b200q_rope_plan_init(C.byref(p), 256, rotary, 1, base, C.byref(sc)) == L.OK
    f, m = frequencies(rotary, base, kind, factor, span, low, high)
    assert (p.head_dim, p.rotary_dim, p.interleaved) == (256, rotary, 1)
    assert math.isclose(p.magnitude, m, rel_tol=2.0**-24)
    # powers and logarithms of the host's library on both sides: a few units in the last place each
    assert all(math.isclose(a, b, rel_tol=2.0**-48) for a, b in zip(p.frequency[:rotary // 2], f))
    assert all(x == 0 for x in p.frequency[rotary // 2:])
    if kind in ("yarn", "banded"):
        assert max(f) <= 1.0 and min(f) >= base ** (-1 + 2 / rotary) / factor * (1 - 1e-12)


def test_arrays_of_words_are_aligned(lib):
    c, p, odd = C.byref(cache()), C.byref(pool()), FAKE + 2
    for rc in (lib.b200q_kv_reserve_dev(p, odd, None, None), lib.b200q_kv_reserve_dev(p, FAKE, odd, None), lib.b200q_kv_free_dev(p, odd, None),
               lib.b200q_kv_fork_dev(c, p, odd, None, None), lib.b200q_kv_fork_dev(c, p, FAKE, odd, None),
               lib.b200q_kv_compact_dev(c, p, odd, 4, 4, FAKE, FAKE + 4096, None), lib.b200q_kv_compact_dev(c, p, FAKE, 4, 4, odd, FAKE + 4096, None),
               lib.b200q_kv_compact_dev(c, p, FAKE, 4, 4, FAKE, odd, None),
               lib.b200q_tree_attention_dev(c, p, C.byref(attention(row_start=odd)), None), lib.b200q_tree_attention_dev(c, p, C.byref(attention(status=odd)), None)):
        refused(lib, rc, L.ERR_INVALID, b"4-byte aligned")


def test_limits_of_32_bit_counts(lib):
    """What would be counted past 32 bits: a tile's rows behind the last one, pieces of a page behind the last one."""
    for rows in ((1 << 31) - 1, (1 << 31) - 200):
        refused(lib, lib.b200q_tree_attention_dev(C.byref(cache()), C.byref(pool()), C.byref(attention(rows=rows, q_heads=2)), None), L.ERR_UNSUPPORTED, b"rows")
    big = cache(heads=65535, head_dim=256)      # 2097120 pieces a slot
    refused(lib, lib.b200q_kv_fork_dev(C.byref(big), C.byref(pool(page_size=600)), FAKE, None, None), L.ERR_UNSUPPORTED, b"page")


def test_attention_in_place_wants_the_same_strides(lib):
    refused(lib, lib.b200q_tree_attention_dev(C.byref(cache()), C.byref(pool()), C.byref(attention(out_row_stride=512)), None), L.ERR_INVALID, b"in place")
