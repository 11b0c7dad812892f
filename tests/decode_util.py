"""Device tensors and argument blocks for the tests of the decoding operators."""
import ctypes as C

import numpy as np
import torch

import tpu_mlir_b200._lib as L
from decode_model import TORCH, Pool

DT = {"bf16": L.DT_BF16, "f16": L.DT_F16}
I32 = torch.int32


def i32(values):
    return torch.tensor(values, dtype=I32, device="cuda")


class Cache:
    """Keys, values and a pool on the device, and the same pool in Python."""

    def __init__(self, *, sequences, width, pages, page_size, heads=2, dim=64, layers=1, dtype="bf16", layout="nhd", seed=0, pad=0):
        self.model = Pool(sequences, width, pages, page_size)
        self.dtype, self.heads, self.dim, self.layers = dtype, heads, dim, layers
        g = torch.Generator().manual_seed(seed)
        shape = (layers, pages, page_size, heads, dim + pad) if layout == "nhd" else (layers, pages, heads, page_size, dim + pad)
        self.k, self.v = (torch.randn(shape, generator=g).to(TORCH[dtype]).cuda() for _ in range(2))
        if layout != "nhd":
            self.k, self.v = self.k.permute(0, 1, 3, 2, 4), self.v.permute(0, 1, 3, 2, 4)
        self.k, self.v = self.k[..., :dim], self.v[..., :dim]
        self.scratch = torch.full((int(L.lib().b200q_kv_scratch_words(sequences)) + 8,), -7, dtype=I32, device="cuda")
        self.status = torch.zeros(1, dtype=I32, device="cuda")
        self.up()

    def up(self):
        """The Python pool's state to the device."""
        m = self.model
        self.table, self.length, self.held, self.refcount = i32(m.table), i32(m.length), i32(m.held), i32(m.refcount)

    def pool(self):
        return L.KvPool(table=self.table.data_ptr(), length=self.length.data_ptr(), held=self.held.data_ptr(), refcount=self.refcount.data_ptr(),
                        scratch=self.scratch.data_ptr(), table_stride=self.table.stride(0), sequences=self.table.shape[0],
                        table_width=self.table.shape[1], pages=self.refcount.numel(), page_size=self.model.page_size,
                        scratch_words=self.scratch.numel() - 8)

    def cache(self):
        k = self.k
        return L.KvCache(k=k.data_ptr(), v=self.v.data_ptr(), layer_stride=k.stride(0), page_stride=k.stride(1), slot_stride=k.stride(2),
                         head_stride=k.stride(3), layers=self.layers, heads=self.heads, head_dim=self.dim, dtype=DT[self.dtype])

    def same_state(self):
        torch.cuda.synchronize()
        m = self.model
        assert self.length.tolist() == m.length and self.held.tolist() == m.held
        assert self.refcount.tolist() == m.refcount
        assert self.table.tolist() == m.table
        assert (self.scratch[-8:] == -7).all(), "words behind the scratch were written"

    # ---- calls
    def reserve(self, extra, stream=None):
        e = i32(extra)
        L.check(L.lib().b200q_kv_reserve_dev(C.byref(self.pool()), e.data_ptr(), self.status.data_ptr(), stream))

    def free(self, which, stream=None):
        w = i32(which)
        L.check(L.lib().b200q_kv_free_dev(C.byref(self.pool()), w.data_ptr(), stream))

    def fork(self, parent, stream=None):
        p = i32(parent)
        L.check(L.lib().b200q_kv_fork_dev(C.byref(self.cache()), C.byref(self.pool()), p.data_ptr(), self.status.data_ptr(), stream))

    def compact(self, path, counts, out=None, stream=None):
        p, c = i32(path), i32(counts)
        out = self.length if out is None else out
        L.check(L.lib().b200q_kv_compact_dev(C.byref(self.cache()), C.byref(self.pool()), p.data_ptr(), p.stride(0), p.shape[1], c.data_ptr(),
                                             out.data_ptr(), stream))

    def workspace(self, q_heads):
        need = C.c_int64()
        L.check(L.lib().b200q_tree_attention_workspace(C.byref(self.cache()), q_heads, C.byref(need)))
        return torch.full((need.value + 64,), 0xA5, dtype=torch.uint8, device="cuda")

    def attend(self, q, out, row_start, mask=None, scale=0.125, layer=0, stream=None, space=None):
        space = self.workspace(q.shape[1]) if space is None else space
        a = L.TreeAttention(q=q.data_ptr(), out=out.data_ptr(), row_start=row_start.data_ptr(), mask=None if mask is None else mask.data_ptr(),
                            workspace=space.data_ptr(), workspace_bytes=space.numel() - 64, q_row_stride=q.stride(0), q_head_stride=q.stride(1),
                            out_row_stride=out.stride(0), out_head_stride=out.stride(1), mask_stride=0 if mask is None else mask.stride(0),
                            rows=q.shape[0], q_heads=q.shape[1], layer=layer, scale=scale)
        L.check(L.lib().b200q_tree_attention_dev(C.byref(self.cache()), C.byref(self.pool()), C.byref(a), stream))
        return space

    def append(self, plan, q, q_out, k, v, row_start, positions=None, layer=0, stream=None):
        a = L.RopeAppend(q=q.data_ptr(), q_out=q_out.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), row_start=row_start.data_ptr(),
                         positions=None if positions is None else positions.data_ptr(), q_row_stride=q.stride(0), q_head_stride=q.stride(1),
                         q_out_row_stride=q_out.stride(0), q_out_head_stride=q_out.stride(1), k_row_stride=k.stride(0), k_head_stride=k.stride(1),
                         v_row_stride=v.stride(0), v_head_stride=v.stride(1), rows=q.shape[0], q_heads=q.shape[1], layer=layer)
        L.check(L.lib().b200q_rope_append_dev(C.byref(plan), C.byref(self.cache()), C.byref(self.pool()), C.byref(a), stream))


def rope_plan(dim, rotary, interleaved, base=10000.0, kind="none", factor=1.0, span=0.0, low=0.0, high=0.0):
    plan = L.RopePlan()
    code = ["none", "linear", "stretched", "yarn", "banded"].index(kind)
    sc = L.RopeScaling(kind=code, factor=factor, original_positions=span, low_turns=low, high_turns=high)
    L.check(L.lib().b200q_rope_plan_init(C.byref(plan), dim, rotary, int(interleaved), base, C.byref(sc)))
    return plan


def words(bits):
    """[rows][nodes] bool -> packed mask words on the device."""
    rows, nodes = bits.shape
    w = -(-nodes // 32)
    full = np.zeros((rows, 32 * w), np.uint64)
    full[:, :nodes] = bits
    packed = (full.reshape(rows, w, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
    return torch.from_numpy(packed.view(np.int32).copy()).cuda()


def random_tree(rng, nodes):
    """Ancestors (and itself) of every node."""
    sees = np.zeros((nodes, nodes), bool)
    for i in range(nodes):
        if i:
            sees[i] = sees[rng.integers(0, i)]
        sees[i, i] = True
    return sees


def f64(t):
    return t.double().cpu().numpy()
