"""Attention over chosen blocks: the choice, the attention and its gradients against plain forms in 64 bits.

Tolerances.  u = finfo.eps / 2 is the largest relative error of one rounding to the type.  A result is a sum over keys of weights (rounded to
the type: u each) times values (exact), divided in fp32 and rounded (u): within u * (sum of |weight * value| + |result|) and fp32 noise of the
scores, 2^-20 of the same sums.  A gradient's terms carry the rounding of the weight or of the score's gradient (u), and that of `out` in
rowsum(out o grad_out) (u of sum |out * grad_out|, as large as |weight| * |grad_out| * |v| terms): 3 u of the sums of magnitudes bounds both, and its own rounding
adds u of the value."""
import numpy as np
import pytest
import torch

import block_util as plain
from vectorsparse_b200 import VsError, ops, torch_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def tensors(B, Lq, Lk, Hq, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(DEV) for s in ((B, Lq, Hq, D), (B, Lk, Hkv, D), (B, Lk, Hkv, D), (B, Lq, Hq, D))]


def lists(B, Hkv, Lq, Lk, count, seed):
    """Any lists: unordered, with repetitions, -1 and numbers that are no block."""
    return torch.from_numpy(np.random.default_rng(seed).integers(-2, -(-Lk // 64) + 2, (B, Hkv, Lq, count)).astype(np.int32)).to(DEV)


def magnitudes(q, k, v, blocks, scale, causal, lengths, grad):
    """Sums of the magnitudes of the terms of out, grad_q, grad_k, grad_v."""
    (B, Lq, Hq, D), (_, Lk, Hkv, _) = q.shape, k.shape
    group = Hq // Hkv
    o, gq, gk, gv = np.zeros_like(q), np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for b in range(B):
        for h in range(Hkv):
            for i in range(Lq):
                t = plain.named(blocks, b, h, i, Lq, Lk, causal, lengths)
                if not len(t):
                    continue
                rows = slice(h * group, (h + 1) * group)
                s = q[b, i, rows] @ k[b, t, h].T * scale
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                d = np.abs(grad[b, i, rows])
                av = np.abs(v[b, t, h])
                o[b, i, rows] = p @ av
                dp = d @ av.T
                ds = p * (dp + (p * dp).sum(1, keepdims=True)) * scale
                gq[b, i, rows] = ds @ np.abs(k[b, t, h])
                gk[b, t, h] += ds.T @ np.abs(q[b, i, rows])
                gv[b, t, h] += p.T @ d
    return o, gq, gk, gv


def check(dtype, q, k, v, blocks, scale, causal, lengths, grad):
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out = torch_ops.selected_attention(*leaves, blocks, scale, causal, n)
    got = (out, *torch.autograd.grad(out, leaves, grad))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    args = [plain.f64(x) for x in (q, k, v)] + [blocks.cpu().numpy(), scale, causal, lengths, plain.f64(grad)]
    u = torch.finfo(dtype).eps / 2
    for name, a, b, m in zip(("out", "grad_q", "grad_k", "grad_v"), got, plain.attention(*args), magnitudes(*args)):
        assert a.dtype == dtype and tuple(a.shape) == b.shape
        error = np.abs(plain.f64(a) - b)
        bound = (3 * u + 2.0 ** -18) * m + u * np.abs(b) + 2.0 ** -24   # the last: fp16 below its normal range
        assert (error <= bound).all(), (name, float((error - bound).max()), float(error.max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,count", [
    (1, 1, 1, 1, 1, 64, 1), (2, 1, 200, 4, 2, 128, 2), (1, 64, 64, 2, 1, 64, 1), (1, 65, 65, 8, 1, 128, 2), (2, 130, 257, 3, 3, 40, 3), (1, 191, 191, 7, 1, 96, 3),
    (1, 33, 300, 16, 1, 80, 4), (1, 100, 100, 10, 2, 8, 2), (1, 150, 400, 2, 2, 128, 5), (1, 40, 90, 32, 1, 64, 2), (1, 5, 70, 128, 1, 64, 2), (3, 97, 97, 6, 2, 32, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_and_gradients(dtype, B, Lq, Lk, Hq, Hkv, D, count, causal):
    q, k, v, grad = tensors(B, Lq, Lk, Hq, Hkv, D, dtype, 7 * Lq + D)
    check(dtype, q, k, v, lists(B, Hkv, Lq, Lk, count, Lq), D ** -0.5, causal, None, grad)


@pytest.mark.parametrize("group", [1, 2, 4])
def test_padded_batches(group):
    """Whatever stands behind a sequence's end, in every operand, reaches nothing; results there are zeros."""
    lengths = [150, 1, 64, 0, 129]
    q, k, v, grad = tensors(5, 150, 150, 2 * group, 2, 64, torch.float16, group)
    blocks = lists(5, 2, 150, 150, 3, group)
    for causal in (True, False):
        check(torch.float16, q, k, v, blocks, 0.125, causal, lengths, grad)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = torch_ops.selected_attention(q, k, v, blocks, 0.125, True, n)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 0.125, True, n), leaves, grad)
    dirty = [x.clone() for x in (q, k, v, grad)]
    for x in dirty:
        for b, m in enumerate(lengths):
            x[b, m::2], x[b, m + 1::2] = float("nan"), float("inf")
    leaves = [x.requires_grad_() for x in dirty[:3]]
    out = torch_ops.selected_attention(*leaves, blocks, 0.125, True, n)
    again = torch.autograd.grad(out, leaves, dirty[3])
    assert ops.device_status() == 0
    for name, a, b in (("out", out, want), *zip(("grad_q", "grad_k", "grad_v"), again, grads)):
        assert torch.isfinite(a).all(), name
        for r, m in enumerate(lengths):
            assert (a[r, m:] == 0).all(), name
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -9, atol=2.0 ** -9), name   # another order of sums where a tile was computed again


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 65504.0])
def test_masked_keys_reach_nothing(value):
    """A key or value that a query does not attend to - not listed, or behind it - may be anything."""
    q, k, v, grad = tensors(1, 192, 192, 4, 1, 64, torch.float16, 3)
    blocks = torch.zeros((1, 1, 192, 2), dtype=torch.int32, device=DEV)
    blocks[:, :, 64:, 1] = torch.arange(64, 192, device=DEV) // 64
    blocks[:, :, 100:, 0] = -1          # of block 1 the queries 64 .. 99 see block 0
    n, m = 70, 130                      # what a key at 70 reaches: queries 70 .. 127; at 130: 130 ..
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    want = torch_ops.selected_attention(*leaves, blocks, 0.125)
    grads = torch.autograd.grad(want, leaves, grad)
    k2, v2 = k.clone(), v.clone()
    k2[:, n], v2[:, m] = value, value
    reached = torch.zeros(192, dtype=torch.bool, device=DEV)
    reached[n:128] = True
    reached[m:] = True
    out = torch_ops.selected_attention(q, k2, v2, blocks, 0.125)
    assert torch.allclose(out[:, ~reached].float(), want[:, ~reached].float(), rtol=2.0 ** -9, atol=2.0 ** -9)
    leaves = [q.clone().requires_grad_(), k2.requires_grad_(), v2.requires_grad_()]
    gq, _, _ = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 0.125), leaves, grad)
    assert torch.allclose(gq[:, ~reached].float(), grads[0][:, ~reached].float(), rtol=2.0 ** -9, atol=2.0 ** -9)
    # a query and a row of grad_out reach the gradients of the keys that they attend to: here of block 1 alone
    q2, g2 = q.clone(), grad.clone()
    q2[:, 110], g2[:, 111] = value, value
    leaves = [q2.requires_grad_(), k.clone().requires_grad_(), v.clone().requires_grad_()]
    again = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 0.125), leaves, g2)
    for i in (1, 2):
        for block in (slice(0, 64), slice(128, 192)):
            assert torch.allclose(again[i][:, block].float(), grads[i][:, block].float(), rtol=2.0 ** -8, atol=2.0 ** -8)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale,size", [(0.125, 8.0), (1e-3, 1.0), (3.0, 4.0), (1e-30, 1.0)])
def test_scores_of_any_size(dtype, scale, size):
    """Scores that the running maximum has to follow by hundreds, or that are all alike."""
    q, k, v, _ = tensors(1, 160, 320, 4, 2, 64, dtype, 5)
    k = k * torch.linspace(0.1, size, 320, device=DEV)[None, :, None, None].to(dtype)
    blocks = lists(1, 2, 160, 320, 4, 5)
    got = plain.f64(torch_ops.selected_attention(q, k, v, blocks, scale))
    args = [plain.f64(x) for x in (q, k, v)] + [blocks.cpu().numpy(), scale, True, None]
    want = plain.attention(*args)
    u = torch.finfo(dtype).eps / 2
    # a score s is off by fp32 noise: its weight by |s| 2^-22, and no score is above |q| |k| scale
    top = float(np.abs(args[0]).sum(-1).max() * np.abs(args[1]).max() * scale)
    bound = (3 * u + 2.0 ** -18 + top * 2.0 ** -21) * np.abs(args[2]).max()
    assert np.abs(got - want).max() <= bound


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,count", [(1, 1, 1, 1, 1, 64, 1), (2, 300, 300, 4, 2, 64, 3), (1, 70, 700, 6, 1, 128, 4), (1, 40, 900, 2, 2, 24, 20),
                                                    (1, 9, 200, 16, 1, 128, 1), (1, 64, 3000, 2, 1, 8, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_selection(dtype, B, Lq, Lk, Hq, Hkv, D, count, causal):
    q, k, _, _ = tensors(B, Lq, Lk, Hq, Hkv, D, dtype, Lk)
    got = torch_ops.select_blocks(q, k, count, causal)
    assert np.array_equal(got.cpu().numpy(), plain.select(plain.f64(q), plain.f64(k), count, causal, None))


def test_selection_of_padded_batches_ties_and_what_is_no_number():
    lengths = [400, 1, 0, 130]
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q, k, _, _ = tensors(4, 400, 400, 4, 2, 32, torch.bfloat16, 1)
    for b, m in enumerate(lengths):
        q[b, m:], k[b, m:] = float("nan"), float("nan")
    k[0, 64:128] = k[0, 0:64]                # equal scores: the lower block
    k[0, 200, 0, 3], k[0, 300, 1, 5] = float("nan"), float("inf")
    q[0, 399, 0] = 0
    with np.errstate(all="ignore"):
        for causal in (True, False):
            for count in (1, 2, 3, 9):
                got = torch_ops.select_blocks(q, k, count, causal, n).cpu().numpy()
                assert np.array_equal(got, plain.select(plain.f64(q), plain.f64(k), count, causal, lengths)), (causal, count)


@pytest.mark.parametrize("count", [2, 5, 40, 127, 129, 200])
def test_selection_of_scores_that_32_bits_cannot_tell_apart(count):
    """Blocks whose scores differ in the last places of 64 bits, or not at all; queries of zeros; more candidates than are ranked again at once."""
    q, k, _, _ = tensors(1, 70, 64 * 300, 2, 1, 64, torch.float16, 11)
    base = k[:, :64].clone()
    k[:, :64 * 290] = base.repeat(1, 290, 1, 1)                              # all alike
    k[:, 64 * 100 + 3, 0, 0] += 2.0 ** -9                                    # but for one element of some
    k[:, 64 * 150 + 3, 0, 1] -= 2.0 ** -9
    k[:, 64 * 200 + 7, 0, 0] += 2.0 ** -9
    q[:, 5], q[:, 60] = 0, 2.0 ** -24
    k[:, 64 * 250:64 * 251] *= 2
    for causal in (True, False):
        got = torch_ops.select_blocks(q, k, count, causal).cpu().numpy()
        assert np.array_equal(got, plain.select(plain.f64(q), plain.f64(k), count, causal, None)), causal


@pytest.mark.parametrize("scale", [1e-20, 1e-38, 1e15, 3e38])
def test_selection_beyond_the_range_of_32_bits(scale):
    q, k, _, _ = tensors(1, 40, 64 * 40, 4, 2, 64, torch.float32, 12)
    q, k = (q * min(scale, 1e37)).bfloat16(), (k.clamp(-1, 1) * scale).bfloat16()
    got = torch_ops.select_blocks(q, k, 6).cpu().numpy()
    assert np.array_equal(got, plain.select(plain.f64(q), plain.f64(k), 6, True, None))


def test_many_blocks():
    """Lists over more blocks than one CTA keeps scores for 32, and for 8, queries of."""
    for keys in (64 * 700 + 5, 64 * 1024, 64 * 1025, 64 * 4000):
        q, k, v, _ = tensors(1, 3, keys, 2, 1, 64, torch.float16, 2)
        got = torch_ops.select_blocks(q, k, 6)
        assert np.array_equal(got.cpu().numpy(), plain.select(plain.f64(q), plain.f64(k), 6, True, None))
        out = torch_ops.selected_attention(q, k, v, got, 0.125)
        want = plain.attention(plain.f64(q), plain.f64(k), plain.f64(v), got.cpu().numpy(), 0.125, True, None)
        assert np.abs(plain.f64(out) - want).max() <= 2.0 ** -9


def test_layouts():
    """[B, H, L, D] seen as [B, L, H, D], slices of a wider projection, expanded and misaligned operands: the results of contiguous ones."""
    q, k, v, grad = tensors(2, 100, 100, 4, 2, 64, torch.bfloat16, 9)
    blocks = torch_ops.select_blocks(q, k, 2)
    want = torch_ops.selected_attention(q, k, v, blocks, 0.125)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    packed = torch.cat([q, k, v], 2)
    sliced = packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x) for x in (q, k, v)]
    for x in (heads_first, sliced, odd):
        assert torch.equal(torch_ops.select_blocks(x[0], x[1], 2), blocks)
        assert torch.equal(torch_ops.selected_attention(*x, blocks, 0.125), want)
    one = k[:1].clone().requires_grad_()
    shared = one.expand(2, -1, -1, -1)
    out = torch_ops.selected_attention(q, shared, v, blocks, 0.125)
    assert torch.equal(out, torch_ops.selected_attention(q, shared.contiguous(), v, blocks, 0.125))
    g, = torch.autograd.grad(out, one, grad)
    both = shared.detach().contiguous().requires_grad_()
    whole, = torch.autograd.grad(torch_ops.selected_attention(q, both, v, blocks, 0.125), both, grad)
    assert torch.equal(g, whole.sum(0, keepdim=True))


def test_gradients_against_differences():
    """Directional derivatives of the operator itself, bf16 leaves: the loss moves as the gradients say."""
    q, k, v, w = tensors(1, 96, 96, 4, 2, 64, torch.float16, 21)
    blocks = torch_ops.select_blocks(q, k, 2)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 0.125), leaves, w)
    args = [plain.f64(x) for x in (q, k, v)]
    at = [blocks.cpu().numpy(), 0.125, True, None]
    rng = np.random.default_rng(0)
    for i in range(3):
        d = rng.standard_normal(args[i].shape)
        moved = []
        for e in (1e-4, -1e-4):
            x = list(args)
            x[i] = x[i] + e * d
            moved.append((plain.attention(*x, *at) * plain.f64(w)).sum())
        slope, said = (moved[0] - moved[1]) / 2e-4, (plain.f64(grads[i]) * d).sum()
        # each element is off by 4 u of its magnitude's terms at most, at random signs under d: the root of the sum of squares, times 4
        size = np.sqrt((plain.f64(grads[i]) ** 2).sum())
        assert abs(slope - said) <= 4 * 4 * 2.0 ** -11 * size * 4, i


def test_results_do_not_depend_on_the_run():
    q, k, v, grad = tensors(2, 500, 500, 8, 2, 128, torch.bfloat16, 4)
    def step():
        blocks = torch_ops.select_blocks(q, k, 3)
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = torch_ops.selected_attention(*leaves, blocks, 0.1)
        return (blocks, out, *torch.autograd.grad(out, leaves, grad))
    first = step()
    for _ in range(3):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)


def test_captured_and_on_another_stream():
    q, k, v, grad = tensors(1, 300, 300, 4, 2, 64, torch.float16, 8)
    def step(q, k, v):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = torch_ops.selected_attention(*leaves, torch_ops.select_blocks(q, k, 3), 0.125)
        return (out, *torch.autograd.grad(out, leaves, grad))
    want = step(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(q, k, v)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    x = [torch.zeros_like(t) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*x)
    for a, b in zip(x, (q, k, v)):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_empty_calls():
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 0, 0), (2, 3, 0)):
        q, k, v, _ = tensors(B, Lq, Lk, 2, 1, 64, torch.float16, 0)
        blocks = torch_ops.select_blocks(q, k, 2, causal=False)
        assert blocks.shape == (B, 1, Lq, 2) and (blocks == -1).all() or Lk > 0
        leaves = [x.requires_grad_() for x in (q, k, v)]
        out = torch_ops.selected_attention(*leaves, blocks, 1.0, causal=False)
        for g in (out, *torch.autograd.grad(out, leaves, torch.ones_like(out))):
            assert (g == 0).all()


def test_refusals():
    q, k, v, _ = tensors(1, 8, 8, 4, 2, 64, torch.float16, 0)
    blocks = torch_ops.select_blocks(q, k, 2)
    good = (q, k, v, blocks, 0.125)
    def refused(error, *args, **kw):
        with pytest.raises(error):
            torch_ops.selected_attention(*args, **kw)
    refused(VsError, q, k, v, blocks, 0.0)
    refused(VsError, q, k, v, blocks, -1.0)
    refused(VsError, q, k, v, blocks, float("nan"))
    refused(VsError, q.float(), k.float(), v.float(), blocks, 0.125)
    refused(TypeError, q, k.bfloat16(), v, blocks, 0.125)
    refused(TypeError, q, k, v, blocks.long(), 0.125)
    refused(ValueError, q, k, v[:, :4], blocks, 0.125)
    refused(ValueError, q, k, v, blocks[:, :1], 0.125)
    refused(ValueError, q[:, :, :3], k, v, blocks, 0.125)
    refused(VsError, q, k[:, :4], v[:, :4], blocks, 0.125)                       # causal with more queries than keys
    refused(VsError, q[:, 4:], k, v, blocks[:, :, 4:].contiguous(), 0.125, lengths=torch.ones(1, dtype=torch.int32, device=DEV))
    refused(ValueError, *good, lengths=torch.ones(2, dtype=torch.int32, device=DEV))
    refused(TypeError, *good, lengths=torch.ones(1, device=DEV))
    refused(TypeError, q, k.cpu(), v, blocks, 0.125)
    wide = torch.zeros((1, 8, 2, 136), dtype=torch.float16, device=DEV)
    with pytest.raises(VsError):
        torch_ops.select_blocks(wide, wide, 1)
    with pytest.raises(RuntimeError):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        g, = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 0.125).sum(), leaves[0], create_graph=True)
        g.sum().backward()


def test_a_workspace_of_exactly_the_size_and_too_small_ones():
    """The C entry points take the sizes that they name and refuse a byte less, before anything runs."""
    import ctypes as C

    from vectorsparse_b200 import _lib
    q, k, v, _ = tensors(1, 130, 130, 4, 2, 64, torch.float16, 6)
    blocks = torch_ops.select_blocks(q, k, 2)
    want = torch_ops.selected_attention(q, k, v, blocks, 0.125)
    n = ops.selected_attention_workspace(q, k)
    buffer = torch.full((n + 64,), 0x5a, dtype=torch.uint8, device=DEV)
    out, lse = torch.empty_like(q), torch.empty((1, 4, 130), dtype=torch.float32, device=DEV)
    strides = [(C.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, v)]
    def call(nbytes):
        return _lib.lib().vs_selected_attention(0, 1, 130, 130, 4, 2, 64, 2, 1, q.data_ptr(), strides[0], k.data_ptr(), strides[1], v.data_ptr(), strides[2], None,
                                                blocks.data_ptr(), out.data_ptr(), None, lse.data_ptr(), C.c_float(0.125), buffer.data_ptr(), nbytes,
                                                torch.cuda.current_stream().cuda_stream)
    assert call(n - 1) == -3
    assert call(n) == 0
    assert torch.equal(out, want) and (buffer[n:] == 0x5a).all()


def test_backward_in_a_graph_beside_an_eager_one_and_two_calls_at_once():
    """A captured step beside an eager graph of other leaves; the same operator on two streams at once."""
    q, k, v, grad = tensors(1, 260, 260, 4, 1, 128, torch.bfloat16, 13)
    blocks = torch_ops.select_blocks(q, k, 3)
    eager = [x.clone().requires_grad_() for x in (q, k, v)]
    held = torch_ops.selected_attention(*eager, blocks, 0.1)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch_ops.selected_attention(*leaves, blocks, 0.1)
        grads = torch.autograd.grad(out, leaves, grad)
    graph.replay()
    want = torch.autograd.grad(held, eager, grad)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, grads))
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                x = [t.detach().requires_grad_() for t in (q, k, v)]
                y = torch_ops.selected_attention(*x, torch_ops.select_blocks(q, k, 3), 0.1)
                results.append((y, *torch.autograd.grad(y, x, grad)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(r, (held, *want)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,count", [(1, 1, 4, 5, 1, 80, 2), (2, 2, 2, 8, 4, 32, 20), (1, 3, 7, 2, 2, 128, 1), (1, 1, 1, 64, 1, 8, 1)])
def test_a_handful_of_rows(dtype, B, Lq, Lk, Hq, Hkv, D, count):
    """So few products are computed in fp32: every result within its own rounding and the fp32 sums, without the weights' 16-bit ones."""
    q, k, v, grad = tensors(B, Lq, Lk, Hq, Hkv, D, dtype, 31 * Lk + D)
    blocks = torch_ops.select_blocks(q, k, count)
    check(dtype, q, k, v, blocks, D ** -0.5, True, None, grad)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out = torch_ops.selected_attention(*leaves, blocks, D ** -0.5)
    got = (out, *torch.autograd.grad(out, leaves, grad))
    want = plain.attention(*(x.double().cpu().numpy() for x in (q, k, v)), blocks.cpu().numpy(), D ** -0.5, True, None, grad.double().cpu().numpy())
    for x, y in zip(got, want):
        y = np.asarray(y)
        # half a step of the type, and 2^-16 of the largest element for fp32 sums of some hundred products, for exp2 and for out's remainder in 16 bits
        allowed = np.abs(y) * torch.finfo(dtype).eps / 2 + (2.0 ** -16 + torch.finfo(dtype).tiny) * max(1.0, np.abs(y).max())
        assert (np.abs(x.detach().double().cpu().numpy() - y) <= allowed).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_key_gradients_of_blocks_that_any_number_of_tiles_has_listed(dtype, D):
    """Block j of the keys is listed by the queries of the first TILES[j] tiles: odd and even numbers, one and some hundred.  With 32 heads to a head of keys a tile
    is four queries.  The same bits in every run."""
    tiles = (1, 2, 3, 4, 5, 6, 7, 8, 150, 151)
    queries, keys = 4 * max(tiles), 64 * len(tiles)
    q, k, v, grad = tensors(1, queries, keys, 32, 1, D, dtype, D)
    blocks = torch.full((1, 1, queries, len(tiles)), -1, dtype=torch.int32, device=DEV)
    for j, n in enumerate(tiles):
        blocks[0, 0, :4 * n, j] = j
    check(dtype, q, k, v, blocks, D ** -0.5, False, None, grad)
    def gradients():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        return torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, D ** -0.5, False), leaves, grad)
    first = gradients()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, gradients()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(1, 0, -1, 0), (0, 1, -1), (1, 1, 0, 0, -1, -1, 0, 0)])
def test_selection_where_the_heads_of_a_group_cancel(dtype, heads):
    """Heads whose large parts cancel: what is left is far below the rounding of a 32-bit sum on its way."""
    q, k, _, _ = tensors(1, 150, 64 * 40, 2 * len(heads), 2, 64, dtype, 14)
    large = (tensors(1, 150, 1, 2, 2, 64, dtype, 15)[0].float().clamp(-4, 4) * 2.0 ** 12).to(dtype)
    for h, sign in enumerate(heads):
        for kv in range(2):
            x = q[:, :, kv * len(heads) + h]
            x.copy_(large[:, :, kv] * sign if sign else x * 2.0 ** -8)
    for causal in (True, False):
        got = torch_ops.select_blocks(q, k, 6, causal).cpu().numpy()
        assert np.array_equal(got, plain.select(plain.f64(q), plain.f64(k), 6, causal, None)), causal


@pytest.mark.parametrize("q_scale,k_scale", [(1.0, 1.0), (1.0, 2.0 ** -76), (2.0 ** -76, 1.0), (2.0 ** -50, 2.0 ** -66)])
@pytest.mark.parametrize("causal", [True, False])
def test_selection_of_near_ties_whose_squares_underflow(q_scale, k_scale, causal):
    """Scores that differ in the 28th bit, of operands whose squares are below 32 bits' range.  All blocks have the same keys but for the order of the two
    elements of some pairs, which a query with equal elements in a pair does not see but for the rounding of its sum, and an element of their own under a
    query element of 2^-20."""
    blocks, rng = 44, np.random.default_rng(7)
    k = np.tile(rng.standard_normal((64, 64)).astype(np.float32), (blocks, 1, 1))
    for j in range(blocks):
        for p in range(1, 32):
            if rng.random() < 0.5:
                k[j][:, [2 * p, 2 * p + 1]] = k[j][:, [2 * p + 1, 2 * p]]
    k[:, :, 0] = rng.permutation(blocks)[:, None] / 32
    q = np.repeat(rng.standard_normal((1, 20, 1, 32)), 2, 3).astype(np.float32)
    q[..., 0] = 2.0 ** -20
    k = torch.from_numpy(k.reshape(1, 64 * blocks, 1, 64)).bfloat16().mul(k_scale).to(DEV)
    q = torch.from_numpy(q).bfloat16().mul(q_scale).to(DEV)
    got = torch_ops.select_blocks(q, k, 6, causal).cpu().numpy()
    assert np.array_equal(got, plain.select(plain.f64(q), plain.f64(k), 6, causal, None))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_size,k_size", [(2.0 ** -4, 4.0), (4.0, 2.0 ** -4)])   # sums that show what their terms have lost: gradients of q, of k
@pytest.mark.parametrize("value", [float("inf"), float("nan"), 1000.0])
def test_small_gradients_beside_a_row_of_large_ones(D, q_size, k_size, value):
    """fp16, grad_out of 1e-4: the scores' gradients lie below the type's normal range unless they are lifted, whatever stands in one row of grad_out.

    Besides the tolerances above: with M the largest element of the rows that share a lift (the row for grad_q, the rows that have listed the block for grad_k), a
    score's gradient is multiplied by 32 / M or more before it is rounded, and below the normal range a rounding is off by 2^-25, so a term by 2^-25 M / 32 times its
    key or query."""
    q, k, v, grad = tensors(2, 200, 200, 4, 2, D, torch.float16, 17)
    q, k, v, grad = q * q_size, k * k_size, v * 2.0 ** -4, (grad.float() * 1e-4).half()
    blocks = lists(2, 2, 200, 200, 3, 17)
    b, i, h = 1, 150, 2
    blocks[b, h // 2, i] = torch.tensor([1, 3, -1], dtype=torch.int32)
    given = grad.clone()
    reached = [np.zeros(x.shape, bool) for x in (q, k, v)]
    if np.isfinite(value):
        given[b, i, h] = grad[b, i, h] = (grad[b, i, h].float() * 1e7).half()   # N(0, 1000^2)
    else:
        given[b, i, h, 5] = value
        grad[b, i, h] = 0
        reached[0][b, i, h] = True
        for x in reached[1:]:
            x[b, 64:128, h // 2] = x[b, 192:, h // 2] = True
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 1.0, False), leaves, given)
    assert ops.device_status() == 0
    args = [plain.f64(x) for x in (q, k, v)] + [blocks.cpu().numpy(), 1.0, False, None, plain.f64(grad)]
    below = [np.zeros(x.shape) for x in args[:3]]
    peak = np.zeros((2, 2, 4))
    rows = [(b, h, i, plain.named(args[3], b, h, i, 200, 200, False, None), slice(2 * h, 2 * h + 2)) for b in range(2) for h in range(2) for i in range(200)]
    for b, h, i, t, heads in rows:
        peak[b, h, np.unique(t // 64)] = np.maximum(peak[b, h, np.unique(t // 64)], np.abs(args[7][b, i, heads]).max())
    for b, h, i, t, heads in rows:
        if len(t):
            below[0][b, i, heads] = 2.0 ** -30 * np.abs(args[7][b, i, heads]).max(-1)[:, None] * np.abs(args[1][b, t, h]).sum(0)
            below[1][b, t, h] += 2.0 ** -30 * peak[b, h, t // 64][:, None] * np.abs(args[0][b, i, heads]).sum(0)
    u = torch.finfo(torch.float16).eps / 2
    for name, a, want, m, floor, not_here in zip(("grad_q", "grad_k", "grad_v"), got, plain.attention(*args)[1:], magnitudes(*args)[1:], below, reached):
        error = np.where(not_here, 0, np.abs(plain.f64(a) - want))
        assert (error <= (3 * u + 2.0 ** -18) * m + u * np.abs(want) + floor + 2.0 ** -24).all(), (name, float(error.max()))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("queries", [255, 256, 257, 512, 513, 1025, 3100, 60000])
def test_key_gradients_of_blocks_that_very_many_tiles_have_listed(D, queries):
    """Sums of one sign over as many tiles as there are queries: 128 heads, so a tile is one.

    A sum in tensor memory is cut off, by less than 2^-21 of itself, in each of 8 steps to a tile, 256 tiles at a stretch: 2^-10 besides the roundings of the
    terms, and 2^-18 for the stretches' own sum in fp32."""
    g = torch.Generator(DEV).manual_seed(queries + D)
    q, grad = (torch.randn((1, queries, 128, D), generator=g, device=DEV) for _ in range(2))
    k, v = ((0.25 * torch.randn((1, 100, 1, D), generator=g, device=DEV)).half() for _ in range(2))
    q, grad = q.half(), grad.abs().mul_(0.25).half()
    blocks = torch.tensor([0, 1], dtype=torch.int32, device=DEV).expand(1, 1, queries, 2).contiguous()
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    _, got_k, got_v = torch.autograd.grad(torch_ops.selected_attention(*leaves, blocks, 0.125, False), leaves, grad)
    assert ops.device_status() == 0
    want_k, want_v, size_k = (torch.zeros((100, D), dtype=torch.float64, device=DEV) for _ in range(3))
    k64, v64 = k[0, :, 0].double(), v[0, :, 0].double()
    for x, d in zip(q[0].view(-1, D).split(1 << 18), grad[0].view(-1, D).split(1 << 18)):
        x, d = x.double(), d.double()
        p = (x @ k64.T * 0.125).softmax(-1)
        dp = d @ v64.T
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * 0.125
        sizes = d @ v64.T.abs()
        sizes = p * (sizes + (p * sizes).sum(-1, keepdim=True)) * 0.125
        want_v += p.T @ d
        want_k += ds.T @ x
        size_k += sizes.T @ x.abs()
    u, steps = torch.finfo(torch.float16).eps / 2, 2.0 ** -10 + 2.0 ** -18
    assert ((got_v[0, :, 0].double() - want_v).abs() <= (2 * u + steps) * want_v).all()
    assert ((got_k[0, :, 0].double() - want_k).abs() <= (3 * u + steps) * size_k + u * want_k.abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("count", [255, 256, 257, 513, 1025, 4100])
def test_long_lists(D, count):
    """Sums of one sign over many blocks.  A sum in tensor memory is cut off, by less than 2^-21 of itself, in each of 4 steps to a block, 256 blocks at a stretch: 2^-11 besides
    the roundings of the weights and of the result, and 2^-18 for fp32."""
    g = torch.Generator(DEV).manual_seed(count + D)
    q, k, v = (torch.randn(s, generator=g, device=DEV) for s in ((1, 70, 2, D), (1, 64 * count, 1, D), (1, 64 * count, 1, D)))
    q, k, v = q.mul_(0.25).half(), k.half(), v.abs_().half()
    blocks = torch.arange(count, dtype=torch.int32, device=DEV).expand(1, 1, 70, count).contiguous()
    got = torch_ops.selected_attention(q, k, v, blocks, D ** -0.5, False)[0].double()
    assert ops.device_status() == 0
    want = torch.einsum("hqk,kd->qhd", (torch.einsum("qhd,kd->hqk", q[0].double(), k[0, :, 0].double()) * D ** -0.5).softmax(-1), v[0, :, 0].double())
    u = torch.finfo(torch.float16).eps / 2
    assert ((got - want).abs() <= (2 * u + 2.0 ** -11 + 2.0 ** -18) * want).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [40, 128])
def test_long_lists_of_unlike_rows(dtype, D):
    """Rows that begin after other rows' sums have been put aside, end before, miss blocks in between or have none; scores that grow along the sequence."""
    q, k, v, grad = tensors(1, 44, 64 * 700 + 9, 4, 2, D, dtype, 23)
    k = (k.float() * torch.linspace(0.1, 3, k.shape[1], device=DEV)[None, :, None, None]).to(dtype)
    rng = np.random.default_rng(23)
    blocks = np.full((1, 2, 44, 320), -1, np.int32)
    for h in range(2):
        for i in range(44):
            lo, hi = [(0, 701), (300, 701), (0, 200), (650, 660), (700, 701), (256, 257), (0, 0)][i % 7]
            some = rng.permutation(np.arange(lo, hi))[:320 if i % 3 else 300]
            blocks[0, h, i, :len(some)] = some
    check(dtype, q, k, v, torch.from_numpy(blocks).to(DEV), D ** -0.5, False, None, grad)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("count", [256, 257, 513, 1025, 16000])
def test_query_gradients_of_long_lists(D, count):
    """Values that are the keys: a gradient of q is grad_out times the keys' covariance, a sum whose terms agree in sign.  With M the largest sum on the way: cut off by
    less than 2^-21 M in each of 8 steps to a block, 256 blocks at a stretch: 2^-10 M.  A result of forward is off by up to 2^-11 of its terms' magnitudes (as above), and
    rowsum(out o grad_out) with it: scale times that times the sum of weight times key.  fp32 besides: 2^-18 of all magnitudes.  The scores' gradients go in as two words of fp16.

    The gradient's part along the exact one is a sum over all elements, in which fp32 noise and the result's rounding have no sign: there 2^-18 of the sum is left of the former,
    and u, all of its rounding if it had one, of the latter."""
    g = torch.Generator(DEV).manual_seed(count + D)
    q, k, grad = (torch.randn(s, generator=g, device=DEV) for s in ((1, 70, 2, D), (1, 64 * count, 1, D), (1, 70, 2, D)))
    q, k, grad = q.mul_(0.25).half(), k.half(), grad.half()
    blocks = torch.arange(count, dtype=torch.int32, device=DEV).expand(1, 1, 70, count).contiguous()
    x, scale = q.clone().requires_grad_(), D ** -0.5
    got, = torch.autograd.grad(torch_ops.selected_attention(x, k, k, blocks, scale, False), x, grad)
    assert ops.device_status() == 0
    u, k64 = torch.finfo(torch.float16).eps / 2, k[0, :, 0].double()
    along = allowed = square = 0.0
    for i in range(0, 70, 3):
        p = (q[0, i].double() @ k64.T * scale).softmax(-1)
        d = grad[0, i].double()
        dp = d @ k64.T
        delta = (p * dp).sum(-1, keepdim=True)
        ds = (p * (dp - delta) * scale).view(2, count, 64)
        parts = torch.einsum("hnt,ntd->hnd", ds, k64.view(count, 64, D))
        want, most = parts.sum(1), parts.cumsum(1).abs().amax(1)
        sizes = p * (d.abs() @ k64.abs().T + (p * (d.abs() @ k64.abs().T)).sum(-1, keepdim=True)) * scale
        wrong_delta = (d.abs() * (p @ k64.abs())).sum(-1, keepdim=True) * 2.0 ** -11
        bound = 2.0 ** -10 * most + scale * wrong_delta * (p @ k64).abs() + 2.0 ** -18 * (sizes @ k64.abs()) + u * want.abs() + 2.0 ** -24
        off = got[0, i].double() - want
        assert (off.abs() <= bound).all(), i
        along += (off * want).sum().item()
        square += (want ** 2).sum().item()
        allowed += (want.abs() * (2.0 ** -10 * most + scale * wrong_delta * (p @ k64).abs() + (u + 2.0 ** -18) * want.abs())).sum().item()
    assert abs(along) <= allowed, (along / square, allowed / square)
