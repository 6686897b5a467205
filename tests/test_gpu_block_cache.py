"""The cache of 8-bit blocks: appending, choosing and attention of single tokens against plain forms in 64 bits, and a run of them together.

Codes, scales and sums are compared bit for bit.  Attention: u = finfo.eps / 2 of the type for the result's rounding and the probabilities' (fp16 for codes, 2^-11;
the type's for the ring), on sums of |probability * value|."""
import numpy as np
import pytest
import torch

import block_util as plain
from vectorsparse_b200 import VsError, ops, torch_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Model:
    """What the cache should hold: every token of every sequence, and its pages and rings."""

    def __init__(self, n, blocks, Hkv, D, dtype, seed=0, spare=2):
        rng = np.random.default_rng(seed)
        self.n, self.Hkv, self.D, self.dtype = n, Hkv, D, dtype
        self.cache = torch_ops.BlockCache.empty(n * blocks + spare, n + spare, Hkv, D, dtype, DEV)
        self.table = rng.permutation(n * blocks + spare)[:n * blocks].reshape(n, blocks).astype(np.int32)
        self.tails = rng.permutation(n + spare)[:n].astype(np.int32)
        self.tokens = [[np.zeros((0, Hkv, D)), np.zeros((0, Hkv, D))] for _ in range(n)]
        self.blocks = [{}, {}]   # (sequence, block) -> codes [Hkv, 64, D], scales [Hkv]
        self.dev = [torch.from_numpy(x).to(DEV) for x in (self.table, self.tails)]

    def lengths(self):
        return torch.tensor([len(t[0]) for t in self.tokens], dtype=torch.int32, device=DEV)

    def append(self, k, v, counts=None):
        torch_ops.cache_append(self.cache, k, v, *self.dev, self.lengths(), None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
        for r in range(self.n):
            m = k.shape[1] if counts is None else counts[r]
            old = len(self.tokens[r][0])
            for i, x in enumerate((k, v)):
                self.tokens[r][i] = np.concatenate([self.tokens[r][i], plain.f64(x[r, :m])])
                for j in range(old // 64, (old + m) // 64):
                    pairs = [plain.rounded(self.tokens[r][i][j * 64:(j + 1) * 64, h]) for h in range(self.Hkv)]
                    self.blocks[i][r, j] = np.stack([p[0] for p in pairs]), np.array([p[1] for p in pairs])

    def check(self):
        c = self.cache
        for i, (codes, scales, ring) in enumerate(((c.k_codes, c.k_scales, c.k_ring), (c.v_codes, c.v_scales, c.v_ring))):
            codes, scales, ring = codes.cpu().numpy(), scales.cpu().numpy(), plain.f64(ring)
            used = set()
            for (r, j), (want, scale) in self.blocks[i].items():
                page = self.table[r, j]
                used.add(page)
                assert np.array_equal(codes[page], want) and np.array_equal(scales[page], scale), (r, j)
                if i == 0:
                    assert np.array_equal(c.k_sums[page].cpu().numpy(), want.sum(1, dtype=np.int16))
            for page in set(range(c.pages)) - used:
                assert not codes[page].any() and not scales[page].any()
            for r in range(self.n):
                have = self.tokens[r][i]
                for t in range(max(0, (len(have) // 64 - 1) * 64), len(have)):
                    assert np.array_equal(ring[self.tails[r], :, t % 128], have[t])
            for tail in set(range(c.tails)) - set(self.tails.tolist()):
                assert not ring[tail].any()

    def content(self, r, i):
        """[tokens, Hkv, D] as attention has them: complete blocks as codes times scales."""
        have = self.tokens[r][i].copy()
        for (s, j), (codes, scale) in self.blocks[i].items():
            if s == r:
                have[j * 64:(j + 1) * 64] = (codes.astype(np.float64) * scale.astype(np.float64)[:, None, None]).transpose(1, 0, 2)
        return have

    def select(self, q, count):
        out = np.full((self.n, self.Hkv, count), -1, np.int32)
        q, G = plain.f64(q), q.shape[1] // self.Hkv
        for r in range(self.n):
            full = len(self.tokens[r][0]) // 64
            for h in range(self.Hkv):
                s = q[r, h * G:(h + 1) * G].sum(0)
                scores = np.array([(self.blocks[0][r, j][0][h].astype(np.float64).sum(0) @ s) * np.float64(self.blocks[0][r, j][1][h]) for j in range(full)])
                if full:
                    out[r, h] = plain.top(scores, full - 1, count)
        return out

    def attention(self, q, scale, blocks=None):
        q, G = plain.f64(q), q.shape[1] // self.Hkv
        out, size = np.zeros_like(q), np.zeros_like(q)
        for r in range(self.n):
            k, v = self.content(r, 0), self.content(r, 1)
            full = len(k) // 64
            for h in range(self.Hkv):
                ids = range(full) if blocks is None else sorted({int(j) for j in blocks[r, h] if 0 <= j < full})
                t = np.concatenate([np.arange(j * 64, j * 64 + 64) for j in ids] + [np.arange(full * 64, len(k))]).astype(np.int64)
                if not len(t):
                    continue
                s = q[r, h * G:(h + 1) * G] @ k[t, h].T * scale
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[r, h * G:(h + 1) * G] = p @ v[t, h]
                size[r, h * G:(h + 1) * G] = p @ np.abs(v[t, h])
        return out, size

    def close(self, got, q, scale, blocks=None):
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        want, size = self.attention(q, scale, blocks)
        u = torch.finfo(self.dtype).eps / 2
        error, bound = np.abs(plain.f64(got) - want), (u + 2.0 ** -11 + 2.0 ** -16) * size + u * np.abs(want) + 2.0 ** -24
        assert (error <= bound).all(), float((error - bound).max())


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def filled(n, lens, Hkv, D, dtype, seed=0, room=0):
    m = Model(n, max(1, max(lens) // 64 + room), Hkv, D, dtype, seed)
    if max(lens):
        m.append(randn(n, max(lens), Hkv, D, dtype=dtype, seed=seed), randn(n, max(lens), Hkv, D, dtype=dtype, seed=seed + 1), list(lens))
    return m


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hkv,D", [(1, 64), (2, 128), (3, 80), (2, 16), (1, 112)])
def test_append(dtype, Hkv, D):
    m = Model(3, 8, Hkv, D, dtype)
    for step, (T, counts) in enumerate([(1, None), (62, None), (1, None), (3, [0, 3, 1]), (100, [100, 1, 64]), (64, None), (130, [5, 130, 129]), (1, None)]):
        m.append(randn(3, T, Hkv, D, dtype=dtype, seed=step), randn(3, T, Hkv, D, dtype=dtype, seed=100 + step), counts)
        m.check()


def test_append_of_what_is_no_number_and_of_nothing():
    m = Model(2, 4, 1, 64, torch.float16)
    k = randn(2, 128, 1, 64, dtype=torch.float16, seed=1)
    k[0, 3, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 65504.0])
    k[0, 64:128] = 0                                   # a block of zeros: scale 0
    k[1, :64] = 2.0 ** -24                             # the smallest numbers
    m.append(k, k.flip(1).contiguous())
    c, page = m.cache, m.table[0, 0]
    assert c.k_codes[page, 0, 3, :4].tolist() == [0, 127, -127, 127]
    assert c.k_scales[page, 0].item() == np.float32(65504) * (np.float32(1) / np.float32(127))
    m.tokens[0][0][3, 0, :3] = 0
    m.tokens[0][1][124, 0, :3] = 0
    c.k_ring[m.tails[0], 0, 3, :3], c.v_ring[m.tails[0], 0, 124, :3] = 0, 0
    m.check()


def test_a_sequence_may_go_back_and_take_other_tokens():
    m = filled(2, [100, 70], 2, 64, torch.float16, room=1)
    kept = [[x.copy() for x in t] for t in m.tokens]
    m.append(randn(2, 5, 2, 64, dtype=torch.float16, seed=50), randn(2, 5, 2, 64, dtype=torch.float16, seed=51))
    m.tokens = kept
    m.append(randn(2, 60, 2, 64, dtype=torch.float16, seed=52), randn(2, 60, 2, 64, dtype=torch.float16, seed=53))
    m.check()


def test_pages_and_rings_that_are_not_there():
    """A table too short, pages and rings out of range: nothing is written there, nothing read, the others are served."""
    m = filled(3, [200, 200, 200], 1, 64, torch.float16)
    before = [x.clone() for x in m.cache._tensors().values()]
    table = m.dev[0].clone()
    table[0], table[1, 1] = m.cache.pages, -1
    tails = m.dev[1].clone()
    tails[2] = m.cache.tails
    q = randn(3, 4, 64, dtype=torch.float16, seed=9)
    got = torch_ops.cache_attention(q, m.cache, table, tails, m.lengths(), 0.125)
    lists = torch_ops.cache_select(q, m.cache, table, m.lengths(), 3)
    assert lists[0, 0].tolist() == [2, -1, -1] and lists[1, 0].tolist() == [0, 2, -1]
    keep = [np.arange(192, 200), np.r_[0:64, 128:200], np.arange(192)]
    for r in range(3):
        k, v = m.content(r, 0)[keep[r], 0], m.content(r, 1)[keep[r], 0]
        s = plain.f64(q)[r] @ k.T * 0.125
        p = np.exp(s - s.max(1, keepdims=True))
        assert np.abs(plain.f64(got)[r] - p @ v / p.sum(1, keepdims=True)).max() <= 2.0 ** -9 * np.abs(v).max()
    new = randn(3, 60, 1, 64, dtype=torch.float16, seed=3)
    short = table[:, :3].contiguous()
    short[1, 1] = 0
    torch_ops.cache_append(m.cache, new, new, short, torch.full_like(tails, -1), m.lengths())
    assert all(torch.equal(a, b) for a, b in zip(before, m.cache._tensors().values()))
    torch_ops.cache_append(m.cache, new, new, short, m.dev[1], m.lengths())      # block 3 has no place in the table
    assert torch.equal(before[0], m.cache.k_codes) and not torch.equal(before[5], m.cache.k_ring)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,lens", [(1, 1, 64, [1]), (8, 2, 128, [0, 63, 64, 65]), (4, 4, 80, [300, 129]), (32, 1, 96, [190, 2]), (7, 1, 128, [1000, 64, 1]),
                                           (40, 2, 48, [256, 257]), (16, 1, 16, [777]), (6, 3, 112, [130, 640]), (4, 2, 32, [64 * 40 + 3, 5])])
def test_attention(dtype, Hq, Hkv, D, lens):
    m = filled(len(lens), lens, Hkv, D, dtype, 3)
    q = randn(len(lens), Hq, D, dtype=dtype, seed=77)
    m.close(torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), D ** -0.5), q, D ** -0.5)
    for count in (1, 3, 20):
        lists = torch_ops.cache_select(q, m.cache, m.dev[0], m.lengths(), count)
        assert np.array_equal(lists.cpu().numpy(), m.select(q, count))
        m.close(torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), D ** -0.5, lists), q, D ** -0.5, lists.cpu().numpy())
    any_list = torch.from_numpy(np.random.default_rng(1).integers(-3, max(lens) // 64 + 3, (len(lens), Hkv, 12)).astype(np.int32)).to(DEV)
    m.close(torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), D ** -0.5, any_list), q, D ** -0.5, any_list.cpu().numpy())


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e-30), (torch.bfloat16, 1e30), (torch.bfloat16, 0.0), (torch.float16, 6e-8), (torch.float16, 300.0)])
def test_queries_of_any_size(dtype, size):
    """bf16 queries beyond fp16's range; the scale of the softmax brings the scores back where the size would make them all alike."""
    m = filled(2, [200, 64], 1, 64, dtype, 4)
    q = (randn(2, 3, 64, dtype=torch.float32, seed=5) * size).to(dtype)
    scale = 0.125 / size if size else 1.0
    m.close(torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), scale), q, scale)


def test_long_sequences_in_pieces():
    m = filled(2, [64 * 130 + 9, 64 * 33], 1, 128, torch.bfloat16, 6)
    q = randn(2, 8, 128, dtype=torch.bfloat16, seed=2)
    assert ops.cache_attention_workspace(q, m.cache, m.dev[0]) > 0
    first = torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), 0.09)
    m.close(first, q, 0.09)
    for _ in range(3):
        assert torch.equal(first, torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), 0.09))


def test_pages_beyond_two_to_the_31():
    """Codes of one tensor past 2^31 bytes from its start."""
    pages = (1 << 31) // (64 * 128) + 8
    cache = torch_ops.BlockCache.empty(pages, 2, 1, 128, torch.float16, DEV)
    table = torch.tensor([[pages - 1, 0], [pages - 2, 1]], dtype=torch.int32, device=DEV)
    small = torch_ops.BlockCache.empty(4, 2, 1, 128, torch.float16, DEV)
    near = torch.tensor([[2, 0], [3, 1]], dtype=torch.int32, device=DEV)
    tails, zero = torch.arange(2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    k, v, q = (randn(2, n, h, 128, dtype=torch.float16, seed=n) for n, h in ((130, 1), (130, 1), (1, 4)))
    for c, t in ((cache, table), (small, near)):
        torch_ops.cache_append(c, k, v, t, tails, zero)
    lengths = zero + 130
    a, b = (torch_ops.cache_attention(q[:, 0], c, t, tails, lengths, 0.1) for c, t in ((cache, table), (small, near)))
    assert torch.equal(a, b) and torch.isfinite(a).all()
    a, b = (torch_ops.cache_select(q[:, 0], c, t, lengths, 2) for c, t in ((cache, table), (small, near)))
    assert torch.equal(a, b)


def test_prompt_then_tokens():
    """As they are used: a prompt's attention over its own blocks, its cache, then token by token with a choice at each, captured once and replayed."""
    n, Hq, Hkv, D, count, dtype = 2, 8, 2, 64, 3, torch.float16
    L = 64 * 6 + 61
    q, k, v = (randn(n, L, h, D, dtype=dtype, seed=h + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    prompt = torch_ops.selected_attention(q, k, v, torch_ops.select_blocks(q, k, count), 0.125)
    assert torch.isfinite(prompt).all()
    m = Model(n, 8, Hkv, D, dtype)
    m.append(k, v)
    x = [randn(n, 1, h, D, dtype=dtype, seed=h) for h in (Hq, Hkv, Hkv)]
    lengths = m.lengths()
    def token():
        torch_ops.cache_append(m.cache, x[1], x[2], *m.dev, lengths)
        lengths.add_(1)
        lists = torch_ops.cache_select(x[0][:, 0], m.cache, m.dev[0], lengths, count)
        return torch_ops.cache_attention(x[0][:, 0], m.cache, *m.dev, lengths, 0.125, lists), lists
    token()                                    # warm, and undone: the same token comes again
    lengths.sub_(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lists = token()
    for step in range(6):                      # across the end of a block
        for i, h in enumerate((Hq, Hkv, Hkv)):
            x[i].copy_(randn(n, 1, h, D, dtype=dtype, seed=1000 * step + h + i))
        tokens = [plain.f64(x[i]) for i in (1, 2)]
        graph.replay()
        torch.cuda.synchronize()
        for r in range(n):
            for i in range(2):
                m.tokens[r][i] = np.concatenate([m.tokens[r][i], tokens[i][r]])
                length = len(m.tokens[r][i])
                if length % 64 == 0:
                    pairs = [plain.rounded(m.tokens[r][i][-64:, h]) for h in range(Hkv)]
                    m.blocks[i][r, length // 64 - 1] = np.stack([p[0] for p in pairs]), np.array([p[1] for p in pairs])
        m.check()
        assert np.array_equal(lists.cpu().numpy(), m.select(x[0][:, 0], count))
        m.close(out, x[0][:, 0], 0.125, lists.cpu().numpy())


def test_refusals():
    m = filled(2, [70, 70], 2, 64, torch.float16)
    q, c = randn(2, 4, 64, dtype=torch.float16, seed=0), m.cache
    n = m.lengths()
    def refused(error, f, *args, **kw):
        with pytest.raises(error):
            f(*args, **kw)
    refused(VsError, torch_ops.cache_attention, q, c, *m.dev, n, 0.0)
    refused(ValueError, torch_ops.cache_attention, q[:, :3], c, *m.dev, n, 1.0)
    refused(ValueError, torch_ops.cache_attention, q[:, :, :32], c, *m.dev, n, 1.0)
    refused(TypeError, torch_ops.cache_attention, q.bfloat16(), c, *m.dev, n, 1.0)
    refused(ValueError, torch_ops.cache_attention, q, c, m.dev[0][:1], m.dev[1], n, 1.0)
    refused(TypeError, torch_ops.cache_attention, q, c, *m.dev, n.long(), 1.0)
    refused(TypeError, torch_ops.cache_attention, q.cpu(), c, *m.dev, n, 1.0)
    refused(ValueError, torch_ops.cache_attention, q, c, *m.dev, n, 1.0, blocks=torch.zeros((2, 1, 3), dtype=torch.int32, device=DEV))
    refused(TypeError, torch_ops.cache_append, c, q[:, None, :2].float(), q[:, None, :2].float(), *m.dev, n)
    refused(ValueError, torch_ops.cache_append, c, q[:, None], q[:, None], *m.dev, n)
    refused((ValueError, VsError), torch_ops.cache_select, q, c, m.dev[0], n, 0)
    refused(ValueError, torch_ops.BlockCache, c.k_codes[:, :, :32], c.v_codes, c.k_scales, c.v_scales, c.k_sums, c.k_ring, c.v_ring)
    refused(TypeError, torch_ops.BlockCache, c.k_codes, c.v_codes, c.k_scales.half(), c.v_scales, c.k_sums, c.k_ring, c.v_ring)
    odd = torch_ops.BlockCache.empty(2, 2, 1, 24, torch.float16, DEV)
    with pytest.raises(VsError):
        torch_ops.cache_append(odd, *(torch.zeros((1, 1, 1, 24), dtype=torch.float16, device=DEV),) * 2, m.dev[0][:1], m.dev[1][:1], n[:1])


def test_a_dispatch_mode_sees_the_operators():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func.namespace == "vsparse":
                self.seen.append(func.overloadpacket.__name__)
            return func(*args, **(kwargs or {}))

    m = filled(2, [70, 130], 1, 64, torch.float16, room=1)
    q = randn(2, 4, 64, dtype=torch.float16, seed=0)
    lists = torch_ops.cache_select(q, m.cache, m.dev[0], m.lengths(), 2)
    out = torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), 0.125, lists)
    x = q[None]
    leaf = x.clone().requires_grad_()
    blocks = torch_ops.select_blocks(x, x[:, :, :2], 1)
    with Names() as mode:
        assert torch.equal(torch_ops.cache_select(q, m.cache, m.dev[0], m.lengths(), 2), lists)
        assert torch.equal(torch_ops.cache_attention(q, m.cache, *m.dev, m.lengths(), 0.125, lists), out)
        m.append(randn(2, 3, 1, 64, dtype=torch.float16, seed=1), randn(2, 3, 1, 64, dtype=torch.float16, seed=2))
        assert torch.equal(torch_ops.select_blocks(x, x[:, :, :2], 1), blocks)
        torch_ops.selected_attention(leaf, x[:, :, :2], x[:, :, :2], blocks, 0.125).sum().backward()
        torch_ops.selected_attention(x, x[:, :, :2], x[:, :, :2], blocks, 0.125)
    m.check()
    assert mode.seen == ["cache_select", "cache_attention", "cache_append", "select_blocks", "selected_attention", "selected_attention_backward", "selected_attention"]
    assert torch.isfinite(leaf.grad).all()


@pytest.mark.parametrize("blocks", [40, 300, 1300])
def test_selection_of_equal_scores_and_missing_pages(blocks):
    """Scores that are all alike, or alike in groups: the lowest blocks; blocks without a page cannot be had."""
    m = Model(2, blocks, 1, 16, torch.float16)
    length = torch.tensor([blocks * 64 + 3, blocks * 64], dtype=torch.int32, device=DEV)
    c, q = m.cache, torch.ones((2, 2, 16), dtype=torch.float16, device=DEV)
    c.k_sums.fill_(3)
    c.k_scales.fill_(0.5)
    table = m.dev[0].clone()
    for count in (1, 2, 7, 33, blocks, blocks + 4):
        got = torch_ops.cache_select(q, c, table, length, count).cpu().numpy()
        want = sorted({blocks - 1, *range(min(count, blocks) - 1)})
        assert (got[:, 0, :len(want)] == np.array(want)).all() and (got[:, 0, len(want):] == -1).all()
    c.k_sums[table[0, 5::9].long()] = 4             # a group above the rest
    c.k_sums[table[1, 11].long()] = 5
    table[0, 14], table[1, 3] = -1, c.pages
    for count in (2, 5, 20):
        got = torch_ops.cache_select(q, c, table, length, count).cpu().numpy()
        best = [[j for j in range(5, blocks, 9) if j != 14], [11]]
        for r, gone in ((0, 14), (1, 3)):
            order = [j for j in best[r] if j != blocks - 1] + [j for j in range(blocks - 1) if j not in best[r] and j != gone]
            want = sorted(order[:count - 1] + [blocks - 1])
            assert got[r, 0, :len(want)].tolist() == want and (got[r, 0, len(want):] == -1).all(), (count, r)


def test_per_sequence_tensors_of_another_shape_are_refused():
    """lengths, tails and counts have one dimension: of as many elements in two, the binding's quick path is no more permissive than the operators."""
    m = Model(2, 3, 1, 64, torch.float16)
    x = torch.randn(2, 70, 1, 64, device=DEV, dtype=torch.float16)
    q, lengths, (table, tails) = x[:, :2].reshape(2, 2, 64), m.lengths(), m.dev
    m.append(x, x)
    for call in (lambda **k: torch_ops.cache_append(m.cache, x, x, table, k.get("tails", tails), k.get("lengths", lengths), k.get("counts")),
                 lambda **k: torch_ops.cache_attention(q, m.cache, table, k.get("tails", tails), k.get("lengths", lengths), 0.125)):
        for name in ("tails", "lengths"):
            with pytest.raises(ValueError):
                call(**{name: lengths[:, None]})
    with pytest.raises(ValueError):
        torch_ops.cache_append(m.cache, x, x, table, tails, lengths, lengths[None])
    with pytest.raises(ValueError):
        torch_ops.cache_select(q, m.cache, table, lengths[:, None], 1)
    m.check()
    q4, blocks = x[:, :, :, None].reshape(2, 70, 1, 64), torch.zeros((2, 1, 70, 1), dtype=torch.int32, device=DEV)
    n = torch.tensor([70, 3], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        torch_ops.select_blocks(q4, q4, 1, lengths=n[:, None])
    with pytest.raises(ValueError):
        torch_ops.selected_attention(q4, q4, q4, blocks, 0.125, lengths=n[None])
