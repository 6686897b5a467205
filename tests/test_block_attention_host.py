"""Attention over chosen blocks and the cache without a GPU: what the C entry points refuse before anything is launched, sizes of workspaces, what the Python
operators refuse, and the tests' own plain forms against differences and against each other."""
import ctypes as C

import numpy as np
import pytest
import torch

import block_util as plain
from vectorsparse_b200 import VsError, _lib, ops, torch_ops

F16, F32, BF16 = _lib.VS_F16, _lib.VS_F32, _lib.VS_BF16
BUF = np.zeros(4096, np.uint8)
P = (BUF.ctypes.data + 15) & ~15
STRIDES = (C.c_int64 * 3)(512, 64, 64)


def attention(dtype=F16, batch=1, queries=8, keys=8, heads=1, kv_heads=1, d=64, count=1, causal=1, q=P, qs=STRIDES, k=P, ks=STRIDES, lengths=None, lists=P, out=P, lse=P,
              scale=1.0, ws=P, nbytes=1 << 40):
    return _lib.lib().vs_selected_attention(dtype, batch, queries, keys, heads, kv_heads, d, count, causal, q, qs, k, ks, k, ks, lengths, lists, out, None, lse,
                                            C.c_float(scale), ws, nbytes, None)


@pytest.mark.parametrize("code,change", [
    (-2, dict(dtype=F32)), (-2, dict(dtype=7)), (-3, dict(queries=-1)), (-3, dict(heads=3, kv_heads=2)), (-3, dict(heads=0)), (-3, dict(kv_heads=0)), (-3, dict(d=4)),
    (-3, dict(d=60)), (-3, dict(d=136)), (-3, dict(count=0)), (-3, dict(queries=9)), (-3, dict(keys=(1 << 20) + 1)), (-3, dict(heads=129)), (-8, dict(causal=2)),
    (-3, dict(queries=4, lengths=P)), (-5, dict(lengths=P + 2)), (-8, dict(scale=0.0)), (-8, dict(scale=-1.0)), (-8, dict(scale=float("inf"))), (-8, dict(scale=float("nan"))),
    (-4, dict(q=None)), (-4, dict(qs=None)), (-4, dict(k=None)), (-4, dict(lists=None)), (-4, dict(out=None)), (-4, dict(lse=None)), (-4, dict(ws=None)),
    (-5, dict(q=P + 8)), (-5, dict(k=P + 2)), (-5, dict(out=P + 8)), (-5, dict(ws=P + 8)), (-5, dict(lists=P + 1)), (-5, dict(qs=(C.c_int64 * 3)(512, 68, 64))),
    (-3, dict(qs=(C.c_int64 * 3)(512, 0, 64))), (-3, dict(qs=(C.c_int64 * 3)(512, -64, 64))), (-3, dict(nbytes=0)), (-3, dict(batch=1 << 20, queries=1 << 20, keys=1 << 20)),
])
def test_refusals_of_attention(code, change):
    assert attention(**change) == code


def test_nothing_to_do():
    assert attention(batch=0, q=None, k=None, lists=None) == 0
    assert attention(queries=0, q=None) == 0
    L = _lib.lib()
    assert L.vs_cache_append(F16, 1, 1, 1, 64, P, P, P, P, P, P, P, 0, 1, P, STRIDES, P, STRIDES, P, 1, P, P, None, None) == 0
    assert L.vs_cache_append(F16, 1, 1, 1, 64, P, P, P, P, P, P, P, 1, 0, P, STRIDES, P, STRIDES, P, 1, P, P, None, None) == 0


def test_refusals_of_the_cache():
    L = _lib.lib()
    def append(dtype=F16, pages=1, kv=1, d=64, n=1, tokens=1, k=P, table=P, blocks=1, codes=P, lengths=P):
        return L.vs_cache_append(dtype, pages, 1, kv, d, codes, P, P, P, P, P, P, n, tokens, k, STRIDES, P, STRIDES, table, blocks, P, lengths, None, None)
    for code, change in ((-2, dict(dtype=F32)), (-3, dict(d=24)), (-3, dict(d=144)), (-3, dict(kv=0)), (-3, dict(n=-1)), (-3, dict(tokens=-1)), (-3, dict(blocks=-1)),
                         (-4, dict(k=None)), (-4, dict(table=None)), (-4, dict(codes=None)), (-4, dict(lengths=None)), (-5, dict(k=P + 2)), (-5, dict(codes=P + 4)), (-5, dict(lengths=P + 2))):
        assert append(**change) == code, change
    def select(heads=2, kv=1, count=1, blocks=1, q=P, lists=P, sums=P):
        return L.vs_cache_select(BF16, 1, heads, kv, 64, P, sums, 1, q, STRIDES, P, blocks, P, count, lists, None)
    for code, change in ((-3, dict(heads=3, kv=2)), (-3, dict(count=0)), (-3, dict(blocks=16385)), (-4, dict(q=None)), (-4, dict(lists=None)), (-5, dict(sums=P + 2)), (-5, dict(q=P + 8))):
        assert select(**change) == code, change
    def token(heads=2, kv=1, lists=None, count=0, scale=1.0, out=P, blocks=1000, ws=P, nbytes=1 << 40):
        return L.vs_cache_attention(F16, 1, 1, heads, kv, 64, P, P, P, P, P, P, 1, P, STRIDES, P, blocks, P, P, lists, count, out, C.c_float(scale), ws, nbytes, None)
    for code, change in ((-3, dict(heads=3, kv=2)), (-3, dict(lists=P, count=0)), (-8, dict(scale=0.0)), (-4, dict(out=None)), (-5, dict(out=P + 8)), (-3, dict(nbytes=0)), (-4, dict(ws=None))):
        assert token(**change) == code, change


def test_workspaces():
    L = _lib.lib()
    assert L.vs_select_blocks_workspace_bytes(0, 8, 8, 1, 64) == 0
    small, large = (L.vs_select_blocks_workspace_bytes(1, n, n, 4, 128) for n in (4096, 65536))
    assert 0 < small < large < (1 << 30)
    assert L.vs_selected_attention_workspace_bytes(1, 8192, 8192, 32, 4, 128, 1) > L.vs_selected_attention_workspace_bytes(1, 8192, 8192, 32, 4, 128, 0) > 0
    assert L.vs_cache_attention_workspace_bytes(1, 8, 8, 128, 8) == 0                    # few blocks: one piece
    assert L.vs_cache_attention_workspace_bytes(1, 8, 8, 128, 2048) > 0
    assert L.vs_cache_attention_workspace_bytes(512, 8, 8, 128, 2048) == 0               # enough sequences to fill the GPU


def test_host_tensors_are_refused():
    q, k = torch.zeros((1, 8, 4, 64), dtype=torch.float16), torch.zeros((1, 8, 2, 64), dtype=torch.float16)
    blocks = torch.zeros((1, 2, 8, 1), dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.select_blocks(q, k, blocks, None)
    with pytest.raises(TypeError):
        ops.selected_attention(q, k, k, blocks, q, None, None, 1.0)
    cache = torch_ops.BlockCache.empty(2, 2, 2, 64, torch.float16, "cpu")
    index = torch.zeros(1, dtype=torch.int32)
    with pytest.raises((TypeError, NotImplementedError)):   # the dispatcher has no kernel for the CPU, as with the other operators
        torch_ops.cache_append(cache, k[:, :1], k[:, :1], index[None], index, index)
    with pytest.raises((TypeError, NotImplementedError)):
        torch_ops.cache_attention(q[0, :1], cache, index[None], index, index, 1.0)
    with pytest.raises(VsError):
        torch_ops.BlockCache.empty(2, 2, 2, 64, torch.float32, "cpu")


def test_the_plain_gradients_against_differences():
    rng = np.random.default_rng(0)
    q, k, v, w = (rng.standard_normal(s) for s in ((2, 5, 4, 8), (2, 70, 2, 8), (2, 70, 2, 8), (2, 5, 4, 8)))
    blocks = np.array(rng.integers(-1, 3, (2, 2, 5, 2)), np.int32)
    _, *grads = plain.attention(q, k, v, blocks, 0.3, True, None, w)
    for i, g in enumerate(grads):
        d = rng.standard_normal(g.shape)
        values = []
        for e in (1e-6, -1e-6):
            x = [q, k, v]
            x[i] = x[i] + e * d
            values.append((plain.attention(*x, blocks, 0.3, True, None) * w).sum())
        assert abs((values[0] - values[1]) / 2e-6 - (g * d).sum()) <= 1e-6 * max(1.0, np.abs(g * d).sum())


def test_the_plain_attention_over_all_blocks_is_dense_attention():
    rng = np.random.default_rng(1)
    q, k, v = (torch.from_numpy(rng.standard_normal(s)) for s in ((1, 90, 4, 8), (1, 90, 2, 8), (1, 90, 2, 8)))
    blocks = np.tile(np.array([1, 0, 1], np.int32), (1, 2, 90, 1))
    s = torch.einsum("bqhd,bkhd->bhqk", q, k.repeat_interleave(2, 2)) * 0.4
    s = s.masked_fill(torch.ones(90, 90).triu(1).bool(), -torch.inf)
    want = torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v.repeat_interleave(2, 2))
    assert np.abs(plain.attention(q.numpy(), k.numpy(), v.numpy(), blocks, 0.4, True, None) - want.numpy()).max() <= 1e-12


def test_the_plain_choice():
    q = np.zeros((1, 130, 1, 1))
    q[:, :, 0, 0] = 1.0
    k = np.zeros((1, 200, 1, 1))
    k[0, :64], k[0, 64:128], k[0, 128:192] = 1.0, 3.0, 2.0
    got = plain.select(q, k, 2, True, None)                 # queries at positions 70 .. 199
    assert got[0, 0, 0].tolist() == [0, 1] and got[0, 0, 58].tolist() == [1, 2] and got[0, 0, 129].tolist() == [1, 3]
    assert plain.top(np.array([1.0, np.nan, 1.0, np.inf]), None, 3) == [0, 2, 3] and plain.top(np.array([]), 0, 2) == [0, -1]


def test_sizes_whose_indices_leave_32_bits_are_refused():
    """Queries are counted in words of 32 and tiles of 128 that reach past the last one, the entries of 32 lists by one number, and the places behind a list's end in steps of 32."""
    L, most, many = _lib.lib(), 0x7fff0000, (2 ** 31 - 1) // 32
    assert attention(queries=most + 1, keys=64, causal=0) == -3
    assert attention(queries=2 ** 31 - 1, keys=64, causal=0) == -3
    assert L.vs_selected_attention_workspace_bytes(1, most, 64, 1, 1, 8, 1) > L.vs_selected_attention_workspace_bytes(1, most - 64, 64, 1, 1, 8, 1) > 0
    assert L.vs_selected_attention_workspace_bytes(1, most + 1, 64, 1, 1, 8, 1) == 0
    assert attention(count=many + 1) == -3
    assert L.vs_select_blocks(F16, 1, 8, 8, 1, 1, 64, many + 1, 1, P, STRIDES, P, STRIDES, None, P, P, 1 << 40, None) == -3
    assert L.vs_cache_select(BF16, 1, 2, 1, 64, P, P, 1, P, STRIDES, P, 1, P, many + 1, P, None) == -3
    assert L.vs_cache_attention(F16, 1, 1, 2, 1, 64, P, P, P, P, P, P, 1, P, STRIDES, P, 1000, P, P, P, many + 1, P, C.c_float(1.0), P, 1 << 40, None) == -3
