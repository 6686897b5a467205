"""Plain forms in 64 bits of attention over chosen blocks and of the 8-bit cache, one query after another, for the tests."""
import numpy as np

BLOCK, RING = 64, 128


def f64(t):
    return t.detach().double().cpu().numpy()


def top(scores, always, count):
    """Ascending list of `always` and the best others, ties to the lowest index, -1 behind."""
    big = np.finfo(np.float64).max
    scores = np.nan_to_num(scores, nan=-big, posinf=big, neginf=-big)
    order = [j for j in np.argsort(-scores, kind="stable") if j != always]
    taken = sorted(([always] if always is not None else []) + order[:max(0, count - (always is not None))])
    return taken + [-1] * (count - len(taken))


def select(q, k, count, causal, lengths):
    (B, Lq, Hq, D), (_, Lk, Hkv, _) = q.shape, k.shape
    out = np.full((B, Hkv, Lq, count), -1, np.int32)
    for b in range(B):
        n = Lk if lengths is None else lengths[b]
        for h in range(Hkv):
            means = [k[b, j:min(j + BLOCK, n), h].mean(0) for j in range(0, n, BLOCK)]
            for i in range(Lq if lengths is None else n):
                own = (i + Lk - Lq) // BLOCK if causal else None
                c = means[:own] if causal else means
                s = q[b, i, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].sum(0)
                out[b, h, i] = top(np.array([s @ m for m in c]), own, count)
    return out


def named(blocks, b, h, i, Lq, Lk, causal, lengths):
    """Keys that query i attends to."""
    n = Lk if lengths is None else lengths[b]
    if lengths is not None and i >= n:
        return np.zeros(0, np.int64)
    end = min(n, i + Lk - Lq + 1) if causal else n
    t = [np.arange(j * BLOCK, min((j + 1) * BLOCK, end)) for j in sorted({int(j) for j in blocks[b, h, i] if 0 <= j < -(-Lk // BLOCK)})]
    return np.concatenate(t) if t else np.zeros(0, np.int64)


def attention(q, k, v, blocks, scale, causal, lengths, grad=None):
    (B, Lq, Hq, D), (_, Lk, Hkv, _) = q.shape, k.shape
    group = Hq // Hkv
    out, gq, gk, gv = np.zeros_like(q), np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for b in range(B):
        for h in range(Hkv):
            for i in range(Lq):
                t = named(blocks, b, h, i, Lq, Lk, causal, lengths)
                if not len(t):
                    continue
                rows = slice(h * group, (h + 1) * group)
                s = q[b, i, rows] @ k[b, t, h].T * scale
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[b, i, rows] = p @ v[b, t, h]
                if grad is not None:
                    d = grad[b, i, rows]
                    dp = d @ v[b, t, h].T
                    ds = p * (dp - (p * dp).sum(1, keepdims=True)) * scale
                    gq[b, i, rows] = ds @ k[b, t, h]
                    gk[b, t, h] += ds.T @ q[b, i, rows]
                    gv[b, t, h] += p.T @ d
    return out if grad is None else (out, gq, gk, gv)


def rounded(x):
    """(codes, scale) of one block and head, [64, D], as 32-bit arithmetic has them."""
    x = x.astype(np.float32)
    finite = np.where(np.isfinite(x), x, np.float32(0))
    scale = np.float32(np.abs(finite).max()) * (np.float32(1) / np.float32(127))
    with np.errstate(all="ignore"):
        q = np.rint(x / scale) if scale > 0 else np.zeros_like(x)
    return np.nan_to_num(np.clip(q, -127, 127), nan=0.0).astype(np.int8), scale
