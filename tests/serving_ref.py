"""Plain numpy forms, in 64 bits, of the operators of a serving step of many sequences (include/ps_hip.h ps_hip_cache_*, ps_hip_sample, ps_hip_adapters_*), and their types on the host."""
import numpy as np

F32, F16, BF16 = 0, 1, 30
HALF_STEP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}  # the largest relative error of a rounding to the type (numbers of ordinary size)
TINY = {F32: 2.0**-149, F16: 2.0**-24, BF16: 2.0**-133}  # the spacing of its smallest numbers


def pack(x, dtype):
    """float64 -> the type's bits, to nearest even (NaN and infinities stay)."""
    x = np.asarray(x, dtype=np.float32)
    if dtype == F32:
        return x
    if dtype == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = np.ascontiguousarray(x).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def unpack(x, dtype):
    if dtype == BF16:
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def lengths(n_kv, count, n_ctx, n_new):
    n0 = np.clip(np.asarray(n_kv), 0, n_ctx)
    c = np.full(len(n0), n_new) if count is None else np.asarray(count)
    return n0, np.clip(c, 0, np.minimum(n_new, n_ctx - n0))


def attend(q, k, v, n0, cnt, scale, tree=None):
    """q [T, H, D], k / v [slots, G, D] with the new rows in place, one sequence -> out [cnt, H, D], weights [G, n0 + cnt], sum of p |v| [cnt, H, D], largest sum of |q| |k| of a visible score"""
    G, R = k.shape[1], q.shape[1] // k.shape[1]
    n = n0 + cnt
    see = np.ones((cnt, n), dtype=bool)
    see[:, n0:] = np.tril(np.ones((cnt, cnt), dtype=bool)) if tree is None else tree[:cnt, :cnt] != 0
    out, size, w = np.zeros((cnt, q.shape[1], q.shape[2])), np.zeros((cnt, q.shape[1], q.shape[2])), np.zeros((G, n))
    far = 0.0
    for h in range(q.shape[1]):
        g = h // R
        some = see.any(1)
        kk, vv = k[:n, g], v[:n, g]
        with np.errstate(invalid="ignore"):
            z = scale * (q[:cnt, h] @ np.where(see.any(0)[:, None], kk, 0).T)
        z = np.where(see, z, -np.inf)
        far = max(far, float((abs(scale) * np.abs(q[:cnt, h]) @ np.abs(np.where(np.isfinite(kk), kk, 0)).T).max(initial=0)))
        top = np.where(some, z.max(1, initial=-np.inf), 0)
        p = np.exp(z - top[:, None])
        p = np.where(some[:, None], p / np.where(some, p.sum(1), 1)[:, None], 0)
        for t in range(cnt):  # what a token does not see is not multiplied by zero
            out[t, h] = p[t, see[t]] @ vv[see[t]]
            size[t, h] = p[t, see[t]] @ np.abs(vv[see[t]])
        w[g] += p.sum(0)
    return out, w, size, far


def evict(n, keep, recent, first, weight, pos):
    """One head of one sequence that holds n > keep slots -> the slot that each of the first `keep` slots takes its row from."""
    top = pos[:n].max()
    protect = (pos[:n] < first) | (pos[:n].astype(np.int64) > int(top) - recent)
    w = np.where(np.isnan(weight[:n]), -np.inf, weight[:n])
    nan = np.isnan(weight[:n])
    order = sorted(range(n), key=lambda j: (0 if protect[j] else 1, 0 if protect[j] else (1 if nan[j] else 0), 0.0 if protect[j] else -w[j], j))
    kept = np.zeros(n, dtype=bool)
    kept[order[:keep]] = True
    take = np.arange(keep)
    take[~kept[:keep]] = [j for j in range(keep, n) if kept[j]]
    return take


def sample(logits, temperature, top_k, top_p, min_p, u):
    """One row -> (id, probability, how near the draw and the cuts came to another answer)."""
    z = np.asarray(logits, dtype=np.float64)
    cand = np.flatnonzero(~np.isnan(z) & (z > -np.inf))
    if len(cand) == 0:
        return -1, 0.0, 1.0
    order = cand[np.lexsort((cand, -z[cand]))]
    if not temperature > 0:
        order, temperature = order[:1], 1.0
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        d = np.where(z[order] == z[order[0]], 0.0, z[order] - z[order[0]])
    w = np.exp(d / temperature)
    w[w < np.exp(-40.0)] = 0
    near = 1.0
    if top_p < 1:
        c = np.cumsum(w)
        goal = max(top_p, 0.0) * c[-1]
        near = min(near, np.abs(c - goal).min() / c[-1]) if top_p > 0 else near
        order = order[:int((c < goal).sum()) + 1]
        w = w[:len(order)]
    if min_p > 0:
        near = min(near, np.abs(w[1:] - min(min_p, 1.0)).min(initial=1.0))
        order = order[w >= min(min_p, 1.0)]
        w = w[:len(order)]
    c = np.cumsum(w)
    u = u if u > 0 else 0.0
    if u >= 1:
        i = int((w > 0).sum()) - 1
    else:
        i = min(int((c <= u * c[-1]).sum()), int((w > 0).sum()) - 1)
        near = min(near, np.abs(c - u * c[-1]).min() / c[-1]) if u > 0 else near
    return int(order[i]), w[i] / c[-1], near
