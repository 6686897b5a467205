"""Attention over blocks that the data choose: the operators' cases and their plain forms.

    select         which blocks of 64 keys each query attends to, by a cheap score
    attend         attention over the chosen blocks, forward
    train          the same in a training step: forward and the gradients of q, k and v
    append         new tokens into a paged cache, complete blocks in 8 bits with a scale for each block and head
    cache_select   which blocks of the cache a single token attends to
    decode         attention of single tokens over the cache: all blocks, or the chosen ones

In a case: B the batch (cache operators: sequences), Lq and Lk the queries and keys, Hq and Hkv their heads, D the width of a head, count the
blocks chosen for a query (0: all), T the tokens appended to a sequence.  `own` says whether `run` computes the plain form or calls the library.
"""
import math
import types

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 64
RING = 2 * BLOCK


def _attn(op, B, Lq, Lk, Hq, Hkv, D, count, dtype, padded=False):
    return dict(op=op, B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, count=count, dtype=dtype, padded=padded)


def _cache(op, B, Lk, Hq, Hkv, D, dtype, count=0, T=0):
    return dict(op=op, B=B, Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, count=count, T=T)


def listed():
    return [
        # the layer of the fixed-mask benchmark (16 heads, sequence 4096, 64 wide) choosing its blocks itself, every head alone
        dict(_attn("select", 1, 4096, 4096, 16, 16, 64, 8, "f16"), name="select_4096"),
        # a long prompt with grouped heads
        dict(_attn("select", 1, 16384, 16384, 32, 4, 128, 16, "bf16"), name="select_16384"),
        # a short ragged prompt: what a call costs
        dict(_attn("attend", 1, 333, 333, 16, 4, 64, 4, "bf16"), name="attend_short_ragged"),
        # the last chunk of a long prompt, its earlier keys already there
        dict(_attn("attend", 1, 1024, 16384, 32, 4, 128, 16, "f16"), name="attend_chunk"),
        # the whole of a long prompt
        dict(_attn("attend", 1, 16384, 16384, 32, 4, 128, 16, "bf16"), name="attend_16384"),
        # a training step of the fixed-mask benchmark's layer, a batch of sequences padded to 2048, no shared heads
        dict(_attn("train", 4, 2048, 2048, 16, 16, 64, 6, "f16", True), name="train_2048_padded"),
        # a training step at length 8192, grouped heads
        dict(_attn("train", 1, 8192, 8192, 32, 4, 128, 16, "bf16"), name="train_8192"),
        # one token for each of 64 sequences
        dict(_cache("append", 64, 2048, 32, 8, 128, "bf16", T=1), name="append_token"),
        # prompts of up to 4096 tokens into an empty cache
        dict(_cache("append", 4, 0, 32, 8, 128, "bf16", T=4096), name="append_prompt"),
        # the blocks of one token for each of 64 sequences
        dict(_cache("cache_select", 64, 16384, 32, 8, 128, "bf16", count=16), name="cache_select_64"),
        # the chosen blocks of few sequences: latency
        dict(_cache("decode", 4, 16384, 32, 8, 128, "f16", count=16), name="decode_chosen"),
        # the whole cache of many sequences: bandwidth
        dict(_cache("decode", 32, 8192, 32, 8, 128, "bf16"), name="decode_whole"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: lengths 1 to 16384, 1 to 16 query heads for a head of keys, heads 16 to 128 wide, both types."""
    largest = {c["op"]: work(c)["flops"] + work(c)["bytes"] for c in listed()}   # each operator's last listed case is its largest
    while True:
        op = rng.choice(["select", "attend", "train", "append", "cache_select", "decode"])
        hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        dtype = rng.choice(["f16", "bf16"])
        if op in ("select", "attend", "train"):
            lq = _log_int(rng, 1, 16384 if op != "train" else 8192)
            padded = rng.random() < 0.3
            lk = lq if padded or rng.random() < 0.6 else min(16384, lq + _log_int(rng, 1, 8192))
            D = rng.choice([64, 128, 128, 64, 32, 80, 96])
            case = _attn(op, _log_int(rng, 1, 6), lq, lk, hkv * group, hkv, D, rng.randint(1, 20), dtype, padded)
            rows = lq * hkv * group
        else:
            T = 0
            if op == "append":
                T = rng.choice([1, 1, rng.randint(2, 64), _log_int(rng, 65, 4096)])
            lk = _log_int(rng, 1, 16384) if op != "append" else _log_int(rng, 1, 2048) if T <= BLOCK else rng.randint(0, 8) * BLOCK
            D = rng.choice([64, 128, 128, 64, 32, 80, 96])
            count = rng.randint(1, 24) if op == "cache_select" or (op == "decode" and rng.random() < 0.5) else 0
            case = _cache(op, _log_int(rng, 1, 64), lk, hkv * group, hkv, D, dtype, count, T)
            rows = 0
        if op in ("select", "cache_select") and not 2 <= case["count"] <= lk // BLOCK - 8:
            continue   # nothing to choose
        if work(case)["flops"] + work(case)["bytes"] <= largest[op] and rows * case["B"] * case["Lk"] <= 32 * 16384 * 16384:
            return case


def _lengths(case):
    """The tokens of each sequence of a padded batch, or in the cache: spread from the whole length downwards, one of them a single token."""
    B, L = case["B"], case["Lk"]
    if case["op"] == "append":   # beyond two blocks a prompt starts at a block's border
        return [L if case["T"] > BLOCK else max(0, L - 37 * b) for b in range(B)]
    return [1 if b == 3 and B > 3 else max(1, L - (b * L) // (2 * B)) for b in range(B)]


def _counts(case):
    return [max(1, case["T"] - (b * case["T"]) // (2 * case["B"])) for b in range(case["B"])]


def _ranges(case):
    """(first position, positions) of the queries of each sequence that are there."""
    if case["padded"]:
        return [(0, n) for n in _lengths(case)]
    return [(case["Lk"] - case["Lq"], case["Lq"])] * case["B"]


def work(case):
    Hq, Hkv, D, count = case["Hq"], case["Hkv"], case["D"], case["count"]
    if case["op"] in ("select", "attend", "train"):
        B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
        q, kv, lists = B * Lq * Hq * D * 2, B * Lk * Hkv * D * 2, B * Hkv * Lq * count * 4
        candidates = named = 0
        for first, n in _ranges(case):
            for block in range(first // BLOCK, (first + n - 1) // BLOCK + 1):
                lo, hi = max(first, block * BLOCK), min(first + n, (block + 1) * BLOCK)   # positions of queries in this block
                candidates += (hi - lo) * block
                named += (hi - lo) * min(count - 1, block) * BLOCK
                named += (hi * (hi + 1) - lo * (lo + 1)) // 2 - (hi - lo) * block * BLOCK
        if case["op"] == "select":
            return {"bytes": q + kv + lists, "flops": 2 * D * Hkv * candidates}
        if case["op"] == "attend":
            return {"bytes": 2 * q + 2 * kv + lists, "flops": 4 * D * Hq * named}
        return {"bytes": 2 * q + 2 * kv + lists + 3 * q + 4 * kv, "flops": 14 * D * Hq * named}
    lengths = _lengths(case)
    if case["op"] == "append":
        tokens = codes = 0
        for n, c in zip(lengths, _counts(case)):
            tokens += c
            codes += ((n + c) // BLOCK - n // BLOCK) * BLOCK
        return {"bytes": Hkv * D * (tokens * 4 + codes * 2 + min(tokens, RING * len(lengths)) * 4), "flops": 4 * Hkv * D * (tokens + codes)}
    if case["op"] == "cache_select":
        blocks = sum(n // BLOCK for n in lengths)
        return {"bytes": len(lengths) * Hq * D * 2 + blocks * Hkv * (2 * D + 4) + len(lengths) * Hkv * count * 4, "flops": 2 * D * Hkv * blocks}
    blocks = sum(min(count, n // BLOCK) if count else n // BLOCK for n in lengths)
    tail = sum(n % BLOCK for n in lengths)
    return {"bytes": 2 * len(lengths) * Hq * D * 2 + Hkv * (blocks * (BLOCK * D * 2 + 8) + tail * D * 4),
            "flops": 4 * D * Hq * (blocks * BLOCK + tail)}


# ---- inputs -------------------------------------------------------------------------------------------------------

def _tokens(g, B, L, Hkv, group, D, run, topics, dtype):
    """[B, L, Hkv * group, D]: text that stays with a subject for `run` tokens and then takes up another of `topics`."""
    subject = torch.randint(0, topics.shape[1], (B, Hkv, L // run + 1), generator=g, device=DEVICE)
    subject = subject.repeat_interleave(run, dim=2)[:, :, :L]
    base = torch.gather(topics, 1, subject.permute(1, 0, 2).reshape(Hkv, B * L, 1).expand(-1, -1, D)).view(Hkv, B, L, D).permute(1, 2, 0, 3)
    x = torch.randn((B, L, Hkv, group, D), generator=g, device=DEVICE, dtype=torch.float32)
    x += 0.5 * base[:, :, :, None]
    return x.view(B, L, Hkv * group, D).to(dtype)


def _qkv(case, g):
    B, Hkv, D, dtype = case["B"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    topics = torch.randn((Hkv, 32, D), generator=g, device=DEVICE)
    q = _tokens(g, B, case["Lq"], Hkv, case["Hq"] // Hkv, D, 48, topics, dtype)
    k = _tokens(g, B, case["Lk"], Hkv, 1, D, 96, topics, dtype)
    v = _tokens(g, B, case["Lk"], Hkv, 1, D, 96, topics, dtype)
    return q, k, v


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _make_cache(case, g):
    """A cache of 8-bit pages in the order in which they came free, its newest tokens in rings of two blocks."""
    B, Hkv, D, dtype = case["B"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    lengths = _lengths(case)
    most = max(n + c for n, c in zip(lengths, _counts(case) if case["T"] else [0] * B)) // BLOCK
    most = max(1, most)
    pages = B * most + 3
    table = torch.randperm(pages, generator=g, device=DEVICE)[:B * most].to(torch.int32).view(B, most)
    codes = [torch.randint(-127, 128, (pages, Hkv, BLOCK, D), generator=g, device=DEVICE, dtype=torch.int8) for _ in range(2)]
    topics = torch.randint(-40, 41, (Hkv, 32, D), generator=g, device=DEVICE, dtype=torch.int16)
    subject = torch.randint(0, 32, (pages,), generator=g, device=DEVICE)
    codes[0] = (codes[0] // 3 + topics[:, subject].permute(1, 0, 2)[:, :, None]).to(torch.int8)
    scales = [(torch.rand((pages, Hkv), generator=g, device=DEVICE) + 0.5) * 0.03 for _ in range(2)]
    rings = [torch.randn((B + 2, Hkv, RING, D), generator=g, device=DEVICE).to(dtype) for _ in range(2)]
    sums = codes[0].sum(2, dtype=torch.int16)
    tails = torch.randperm(B + 2, generator=g, device=DEVICE)[:B].to(torch.int32)
    parts = dict(k_codes=codes[0], v_codes=codes[1], k_scales=scales[0], v_scales=scales[1], k_sums=sums, k_ring=rings[0], v_ring=rings[1])
    if own:
        from vectorsparse_b200 import torch_ops
        cache = torch_ops.BlockCache(**parts)
    else:
        cache = types.SimpleNamespace(**parts)
    return cache, table, tails, _int32(lengths), topics


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = types.SimpleNamespace(case=case, scale=case["D"] ** -0.5)
    if case["op"] in ("select", "attend", "train"):
        s.q, s.k, s.v = _qkv(case, g)
        s.lengths = _int32(_lengths(case)) if case["padded"] else None
        if case["op"] != "select":
            s.blocks = _plain_select(s.q, s.k, case["count"], s.lengths)
        if case["op"] == "train":
            s.grad = torch.randn(s.q.shape, generator=g, device=DEVICE).to(s.q.dtype)
        return s
    s.cache, s.table, s.tails, s.lengths, topics = _make_cache(case, g)
    B, Hq, Hkv, D, dtype = case["B"], case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        s.counts = _int32(_counts(case))
        s.k, s.v = (torch.randn((B, case["T"], Hkv, D), generator=g, device=DEVICE).to(dtype) for _ in range(2))
        return s
    subject = torch.randint(0, 32, (B,), generator=g, device=DEVICE)
    q = torch.randn((B, Hkv, Hq // Hkv, D), generator=g, device=DEVICE)
    q += topics[:, subject].permute(1, 0, 2)[:, :, None].float() / 60
    s.q = q.view(B, Hq, D).to(dtype)
    s.blocks = None
    if case["op"] == "decode" and case["count"]:
        s.blocks = _plain_cache_select(s.q, s.cache, s.table, s.lengths, case["count"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "train":
        s.q, s.k, s.v = (x.requires_grad_() for x in (s.q, s.k, s.v))
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _chosen(scores, candidate, always, count):
    """Ascending indices of `always` (-1: none) and of the best candidates of the last axis, -1 behind them; a score that is no number is the lowest."""
    n = scores.shape[-1]
    index = torch.arange(n, device=scores.device)
    scores = torch.nan_to_num(scores, nan=-torch.finfo(scores.dtype).max).masked_fill(~candidate, -math.inf)
    scores = scores.masked_fill(index == always[..., None], math.inf)
    order = torch.sort(scores, dim=-1, descending=True, stable=True)
    taken = order.indices[..., :count]
    taken = torch.where(order.values[..., :count] == -math.inf, n, taken)
    taken = torch.sort(taken, dim=-1).values
    taken = torch.where(taken == n, -1, taken).to(torch.int32)
    return torch.nn.functional.pad(taken, (0, count - taken.shape[-1]), value=-1)


def _plain_select(q, k, count, lengths):
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    blocks = -(-Lk // BLOCK)
    means = torch.nn.functional.pad(k.double(), (0, 0, 0, 0, 0, blocks * BLOCK - Lk)).view(B, blocks, BLOCK, Hkv, D).sum(2) / BLOCK
    sums = q.double().view(B, Lq, Hkv, Hq // Hkv, D).sum(3)
    position = torch.arange(Lq, device=q.device) + (Lk - Lq)
    index = torch.arange(blocks, device=q.device)
    out = torch.empty((B, Hkv, Lq, count), dtype=torch.int32, device=q.device)
    for b in range(B):
        for h in range(Hkv):
            scores = sums[b, :, h] @ means[b, :, h].T
            out[b, h] = _chosen(scores, index < (position // BLOCK)[:, None], position // BLOCK, count)
        if lengths is not None:
            out[b, :, position >= lengths[b]] = -1
    return out


def _mask(blocks, b, h, lo, hi, Lq, Lk, lengths):
    """Which keys queries lo .. hi of a head of keys attend to: [hi - lo, Lk]."""
    n = -(-Lk // BLOCK)
    listed = blocks[b, h, lo:hi].long()
    named = torch.zeros((hi - lo, n + 1), dtype=torch.bool, device=blocks.device)
    named.scatter_(1, torch.where(listed < 0, n, listed), True)
    named = named[:, :n].repeat_interleave(BLOCK, dim=1)[:, :Lk]
    key = torch.arange(Lk, device=blocks.device)
    named &= key <= (torch.arange(lo, hi, device=blocks.device) + (Lk - Lq))[:, None]
    if lengths is not None:
        named &= key < lengths[b]
    return named


def _plain_attention(s, grad=None):
    B, Lq, Hq, D = s.q.shape
    Lk, Hkv = s.k.shape[1:3]
    group = Hq // Hkv
    out = torch.zeros_like(s.q)
    if grad is not None:
        gq, gk, gv = torch.zeros_like(s.q), torch.zeros(s.k.shape, device=DEVICE), torch.zeros(s.v.shape, device=DEVICE)
    step = max(1, (1 << 28) // (group * Lk))
    for b in range(B):
        for h in range(Hkv):
            k, v = s.k[b, :, h].float(), s.v[b, :, h].float()
            for lo in range(0, Lq, step):
                hi = min(Lq, lo + step)
                rows = slice(h * group, (h + 1) * group)
                mask = _mask(s.blocks, b, h, lo, hi, Lq, Lk, s.lengths)
                q = s.q[b, lo:hi, rows].transpose(0, 1).float()
                p = (q @ k.T).mul_(s.scale).masked_fill_(~mask, -math.inf)
                top = p.amax(-1, keepdim=True)
                p = p.sub_(torch.where(top == -math.inf, 0, top)).exp_()
                p = p.div_(p.sum(-1, keepdim=True).clamp_min_(torch.finfo(torch.float32).tiny))
                o = p @ v
                out[b, lo:hi, rows] = o.transpose(0, 1).to(out.dtype)
                if grad is None:
                    continue
                d = grad[b, lo:hi, rows].transpose(0, 1).float()
                ds = p * (d @ v.T - (d * o).sum(-1, keepdim=True)) * s.scale
                gq[b, lo:hi, rows] = (ds @ k).transpose(0, 1).to(gq.dtype)
                gk[b, :, h] += torch.einsum("gqk,gqd->kd", ds, q)
                gv[b, :, h] += torch.einsum("gqk,gqd->kd", p, d)
    return out if grad is None else (out, gq, gk.to(s.k.dtype), gv.to(s.v.dtype))


def _plain_append(s):
    c = s.cache
    lengths, counts = s.lengths.tolist(), s.counts.tolist()
    for r, (n, m) in enumerate(zip(lengths, counts)):
        for new, codes, scales, ring, sums in ((s.k, c.k_codes, c.k_scales, c.k_ring, c.k_sums), (s.v, c.v_codes, c.v_scales, c.v_ring, None)):
            ring = ring[s.tails[r]]
            new = new[r, :m].transpose(0, 1)
            first, last = n // BLOCK, (n + m) // BLOCK
            at = first % 2 * BLOCK
            x = torch.cat([ring[:, at:at + n % BLOCK], new], 1)
            full = x[:, :(last - first) * BLOCK].float().reshape(x.shape[0], last - first, BLOCK, x.shape[2])
            if last > first:
                pages = s.table[r, first:last].long()
                scale = full.abs().amax((2, 3)) / 127
                code = torch.round(full / scale[:, :, None, None]).to(torch.int8)
                codes[pages], scales[pages] = code.transpose(0, 1), scale.T
                if sums is not None:
                    sums[pages] = code.sum(2, dtype=torch.int16).transpose(0, 1)
            kept = torch.arange(max(n, (last - 1) * BLOCK), n + m, device=DEVICE)
            ring[:, kept % RING] = new[:, kept - n]
    return c.k_codes, c.v_codes, c.k_scales, c.v_scales, c.k_sums, c.k_ring, c.v_ring


def _plain_cache_select(q, cache, table, lengths, count):
    B, Hq, D = q.shape
    Hkv = cache.k_codes.shape[1]
    sums = q.double().view(B, Hkv, Hq // Hkv, D).sum(2)
    scores = torch.einsum("bnhd,bhd->bhn", cache.k_sums[table.long()].double(), sums)
    scores = scores * cache.k_scales[table.long()].double().transpose(1, 2)
    complete = (lengths // BLOCK)[:, None]
    candidate = (torch.arange(table.shape[1], device=q.device) < complete)[:, None]
    return _chosen(scores, candidate, (complete - 1).expand(-1, Hkv), count)


def _plain_decode(s):
    c, dtype = s.cache, torch.float32
    B, Hq, D = s.q.shape
    Hkv = c.k_codes.shape[1]
    out = torch.zeros_like(s.q)
    for r, n in enumerate(s.lengths.tolist()):
        full, rest, at = n // BLOCK, n % BLOCK, n // BLOCK % 2 * BLOCK
        pages = s.table[r, :full].long()
        k, v = ((x[pages].to(dtype) * y[pages].to(dtype)[:, :, None, None]).transpose(0, 1).reshape(Hkv, full * BLOCK, D)
                for x, y in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)))
        k, v = (torch.cat([x, y[s.tails[r], :, at:at + rest].to(dtype)], 1) for x, y in ((k, c.k_ring), (v, c.v_ring)))
        scores = s.q[r].to(dtype).view(Hkv, Hq // Hkv, D) @ k.transpose(1, 2) * s.scale
        if s.blocks is not None:
            listed = s.blocks[r].long()
            named = torch.zeros((Hkv, full + 1), dtype=torch.bool, device=DEVICE).scatter_(1, torch.where(listed < 0, full, listed), True)
            named = torch.cat([named[:, :full].repeat_interleave(BLOCK, dim=1), torch.ones((Hkv, rest), dtype=torch.bool, device=DEVICE)], 1)
            scores = scores.masked_fill(~named[:, None], -math.inf)
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        out[r] = (p @ v / p.sum(-1, keepdim=True)).view(Hq, D).to(out.dtype)
    return out


# ---- one pass ---------------------------------------------------------------------------------------------------------

def _own(s):
    from vectorsparse_b200 import torch_ops
    op = s.case["op"]
    if op == "select":
        return torch_ops.select_blocks(s.q, s.k, s.case["count"], lengths=s.lengths)
    if op == "attend":
        return torch_ops.selected_attention(s.q, s.k, s.v, s.blocks, s.scale, lengths=s.lengths)
    if op == "train":
        out = torch_ops.selected_attention(s.q, s.k, s.v, s.blocks, s.scale, lengths=s.lengths)
        return (out.detach(), *torch.autograd.grad(out, (s.q, s.k, s.v), s.grad))
    if op == "append":
        c = s.cache
        torch_ops.cache_append(c, s.k, s.v, s.table, s.tails, s.lengths, s.counts)
        return c.k_codes, c.v_codes, c.k_scales, c.v_scales, c.k_sums, c.k_ring, c.v_ring
    if op == "cache_select":
        return torch_ops.cache_select(s.q, s.cache, s.table, s.lengths, s.case["count"])
    return torch_ops.cache_attention(s.q, s.cache, s.table, s.tails, s.lengths, s.scale, blocks=s.blocks)


def run(state):
    if own:
        return _own(state)
    op = state.case["op"]
    with torch.no_grad():
        if op == "select":
            return _plain_select(state.q, state.k, state.case["count"], state.lengths)
        if op == "attend":
            return _plain_attention(state)
        if op == "train":
            return _plain_attention(state, state.grad)
        if op == "append":
            return _plain_append(state)
        if op == "cache_select":
            return _plain_cache_select(state.q, state.cache, state.table, state.lengths, state.case["count"])
        return _plain_decode(state)


# ---- the definitions in 64 bits, query by query ------------------------------------------------------------------------

def _exact_attention(s, grad):
    """Every query gathers the keys of its own blocks."""
    B, Lq, Hq, D = s.q.shape
    Lk, Hkv = s.k.shape[1:3]
    group, count = Hq // Hkv, s.blocks.shape[-1]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    gq, gk, gv = (torch.zeros(x.shape, dtype=torch.float64, device=DEVICE) for x in (s.q, s.k, s.v))
    step = max(1, (1 << 26) // (count * BLOCK * D))
    for b in range(B):
        n = Lk if s.lengths is None else int(s.lengths[b])
        for h in range(Hkv):
            heads = slice(h * group, (h + 1) * group)
            for lo in range(0, Lq, step):
                hi = min(Lq, lo + step)
                t = (s.blocks[b, h, lo:hi, :, None].long() * BLOCK + torch.arange(BLOCK, device=DEVICE)).flatten(1)
                here = torch.arange(lo, hi, device=DEVICE)[:, None] + (Lk - Lq)
                valid = (t >= 0) & (t <= here) & (t < n)
                t = t.clamp(0, Lk - 1)
                k, v, q = s.k[b, :, h][t].double(), s.v[b, :, h][t].double(), s.q[b, lo:hi, heads].double()
                w = torch.einsum("qgd,qtd->qgt", q, k) * s.scale
                w = torch.where(valid[:, None], w, -math.inf)
                top = w.amax(-1, keepdim=True)
                w = torch.exp(w - torch.where(torch.isinf(top), 0.0, top))
                total = w.sum(-1, keepdim=True)
                w = w / torch.where(total > 0, total, 1.0)
                o = torch.einsum("qgt,qtd->qgd", w, v)
                out[b, lo:hi, heads] = o
                if grad is None:
                    continue
                d = grad[b, lo:hi, heads].double()
                dw = torch.einsum("qgd,qtd->qgt", d, v)
                ds = w * (dw - (w * dw).sum(-1, keepdim=True)) * s.scale
                gq[b, lo:hi, heads] = torch.einsum("qgt,qtd->qgd", ds, k)
                gk[b, :, h].index_add_(0, t.flatten(), torch.einsum("qgt,qgd->qtd", ds, q).flatten(0, 1))
                gv[b, :, h].index_add_(0, t.flatten(), torch.einsum("qgt,qgd->qtd", w, d).flatten(0, 1))
    return out if grad is None else (out, gq, gk, gv)


def _exact_select(case, s):
    """The blocks of one query after another, from a ranking of all of them."""
    B, Lq, Hq, D = s.q.shape
    Lk, Hkv = s.k.shape[1:3]
    count = case["count"]
    k = s.k.transpose(1, 2).double().cumsum(2)
    ends = torch.arange(BLOCK - 1, Lk - Lk % BLOCK, BLOCK, device=DEVICE)
    sums = k[:, :, ends].diff(dim=2, prepend=torch.zeros_like(k[:, :, :1]))
    out = torch.full((B, Hkv, Lq, count), -1, dtype=torch.int32, device=DEVICE)
    first = Lk - Lq
    for b, (start, n) in enumerate(_ranges(case)):
        for block in range(start // BLOCK, (start + n - 1) // BLOCK + 1):
            lo, hi = max(start, block * BLOCK) - first, min(start + n, (block + 1) * BLOCK) - first
            q = s.q[b, lo:hi].double().view(hi - lo, Hkv, Hq // Hkv, D).sum(2)
            scores = torch.einsum("qhd,hjd->hqj", q, sums[b, :, :block])
            best = torch.topk(scores, min(count - 1, block), dim=-1).indices
            best = torch.cat([best, torch.full_like(best[..., :1], block) if best.shape[-1] else best.new_full((Hkv, hi - lo, 1), block)], -1)
            out[b, :, lo:hi, :best.shape[-1]] = torch.sort(best, dim=-1).values.to(torch.int32)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "select":
        return _exact_select(case, s)
    if op in ("attend", "train"):
        return _exact_attention(s, s.grad if op == "train" else None)
    if op == "append":
        return _exact_append(s)
    if op == "cache_select":
        return _exact_cache_select(case, s)
    return _exact_decode(s)


def _exact_append(s):
    """Scales and rings token by token; a code next to a half is what 32 bits make of it, so codes and their sums have no other value."""
    scales, rings = [], []
    for new, scale, ring in ((s.k, s.cache.k_scales, s.cache.k_ring), (s.v, s.cache.v_scales, s.cache.v_ring)):
        before, scale, ring = ring.double(), scale.double(), ring.double()
        for r, (n, m) in enumerate(zip(s.lengths.tolist(), s.counts.tolist())):
            tail, top = s.tails[r], 0.0
            if n % BLOCK:
                top = before[tail, :, n // BLOCK * BLOCK % RING:][:, :n % BLOCK].abs().amax((1, 2))
            for lo in range(n, n + m):
                top = torch.maximum(new[r, lo - n].double().abs().amax(1), torch.as_tensor(top, device=DEVICE, dtype=torch.float64))
                if lo % BLOCK == BLOCK - 1:
                    scale[s.table[r, lo // BLOCK].long()] = top / 127
                    top = 0.0
                if lo >= ((n + m) // BLOCK - 1) * BLOCK:
                    ring[tail, :, lo % RING] = new[r, lo - n].double()
        scales.append(scale)
        rings.append(ring)
    return None, None, scales[0], scales[1], None, rings[0], rings[1]


def _exact_cache_select(case, s):
    """One sequence and one head after another, the sums taken from the codes."""
    c = s.cache
    B, Hq, D = s.q.shape
    Hkv = c.k_codes.shape[1]
    out = torch.full((B, Hkv, case["count"]), -1, dtype=torch.int32, device=DEVICE)
    for r, n in enumerate(s.lengths.tolist()):
        full = n // BLOCK
        if not full:
            continue
        pages = s.table[r, :full].long()
        for h in range(Hkv):
            q = s.q[r, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].double().sum(0)
            score = (c.k_codes[pages, h].double().sum(1) * q).sum(1) * c.k_scales[pages, h].double()
            score[full - 1] = math.inf
            best = torch.sort(torch.topk(score, min(full, case["count"])).indices).values
            out[r, h, :best.numel()] = best.to(torch.int32)
    return out


def _exact_decode(s):
    """One head and one block after another, weights not yet divided by their sum."""
    c = s.cache
    B, Hq, D = s.q.shape
    Hkv = c.k_codes.shape[1]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    for r, n in enumerate(s.lengths.tolist()):
        full, at = n // BLOCK, n // BLOCK % 2 * BLOCK
        for h in range(Hkv):
            q = s.q[r, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].double()
            ids = torch.arange(full, device=DEVICE) if s.blocks is None else s.blocks[r, h][s.blocks[r, h] >= 0].long()
            pages = s.table[r].long()[ids]
            k = (c.k_codes[pages, h].double() * c.k_scales[pages, h].double()[:, None, None]).flatten(0, 1)
            v = (c.v_codes[pages, h].double() * c.v_scales[pages, h].double()[:, None, None]).flatten(0, 1)
            k = torch.cat([k, c.k_ring[s.tails[r], h, at:at + n % BLOCK].double()])
            v = torch.cat([v, c.v_ring[s.tails[r], h, at:at + n % BLOCK].double()])
            out[r, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)] = torch.softmax(q @ k.T * s.scale, -1) @ v
    return out
