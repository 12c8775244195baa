"""Plain 64-bit statements of the paged 4-bit cache, its planner and its attention (numpy; tests only)."""
import numpy as np


def quantise(x):
    """Rows (last axis) of fp16 / fp32 values -> codes uint8 and (step, low) fp16, in the fp32 arithmetic that defines
    them: low = fp16(min), step = fp16((max - min) / 15), code = clamp(rint((x - low) / step), 0, 15)."""
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        low = lo.astype(np.float16)
        step = ((hi - lo) / np.float32(15)).astype(np.float16)
        c = np.rint((x - low.astype(np.float32)) / step.astype(np.float32))
        code = np.where(step > 0, np.clip(np.nan_to_num(c), 0, 15), 0).astype(np.uint8)
        bad = ~(np.abs(x) < 65520).all(-1, keepdims=True)
    code = np.where(bad, 0, code).astype(np.uint8)
    par = np.concatenate([step, low], -1)
    return code, np.where(bad, np.float16(np.nan), par).astype(np.float16)


def values(code, par):
    par = par.astype(np.float64)
    return par[..., :1] * code + par[..., 1:]


def page_bytes(page, heads, hd):
    return heads * page * (hd + 8)


class Pages:
    """The cache on the host, in the documented layout."""

    def __init__(self, n_pages, page, heads, hd, fill=255):
        self.page, self.heads, self.hd = page, heads, hd
        self.bytes = np.full((n_pages, page_bytes(page, heads, hd)), fill, np.uint8)

    def _parts(self, page_id, h):
        b = self.bytes[page_id].reshape(self.heads, -1)[h]
        n = self.page * self.hd // 2
        k, v = b[:n].reshape(self.page, -1), b[n:2 * n].reshape(self.page, -1)
        par = b[2 * n:].reshape(2, self.page, 4)
        return (k, v), par

    def put(self, slot, k, v):
        """k, v [heads, hd] of one token."""
        p, at = divmod(int(slot), self.page)
        for h in range(self.heads):
            codes, par = self._parts(p, h)
            for i, x in enumerate((k, v)):
                c, q = quantise(x[h])
                codes[i][at] = c[0::2] | (c[1::2] << 4)
                par[i, at] = q.view(np.uint8)

    def get(self, slot):
        p, at = divmod(int(slot), self.page)
        out = np.empty((2, self.heads, self.hd))
        for h in range(self.heads):
            codes, par = self._parts(p, h)
            for i in range(2):
                c = np.empty(self.hd, np.uint8)
                c[0::2], c[1::2] = codes[i][at] & 15, codes[i][at] >> 4
                out[i, h] = values(c, par[i, at].copy().view(np.float16))
        return out

    def steps(self, slot):
        p, at = divmod(int(slot), self.page)
        return np.array([self._parts(p, h)[1][1, at].copy().view(np.float16)[0] for h in range(self.heads)], np.float64)


def plan(ctx, new, table, free, count, page, max_blocks, max_tokens):
    """One request after the other; (q_start, kv_len, table, slots, free_left, refused)."""
    table = table.copy()
    q_start, kv_len, slots = [0], [], np.full(max_tokens, -1, np.int64)
    need_sum, taken, refused = 0, 0, 0
    for i, (c, n) in enumerate(zip(ctx.tolist(), new.tolist())):
        r0 = q_start[-1]
        r1 = r0 + max(n, 0)
        q_start.append(r1)
        ok = c >= 0 and n >= 0 and c + n <= max_blocks * page and r1 <= max_tokens
        if ok:
            have, end = -(-c // page), -(-(c + n) // page)
            need_sum += end - have
            ok = end == have or need_sum <= count
        if not ok:
            refused += 1
            kv_len.append(max(c, 0))
            continue
        for b in range(have, end):
            table[i, b] = free[count - 1 - taken]
            taken += 1
        kv_len.append(c + n)
        for t in range(n):
            slots[r0 + t] = int(table[i, (c + t) // page]) * page + (c + t) % page
    return (np.minimum(q_start, max_tokens + 1).astype(np.int32), np.array(kv_len, np.int32), table, slots,
            count - taken, refused)


def attention(pages, q, q_start, kv_len, table, scale, prefix=None):
    """fp64 result and a bound on the error of a 32-bit evaluation rounded to fp16 (rows outside requests: NaN).

    The bound: the output's rounding (2^-11 of it); weights that may be rounded to fp16 against codes centred within 8
    steps (2^-11 of 8 sum p step); 32-bit scores: terms of up to 4 S (step * code and low before they cancel, S the sum of
    the magnitudes |q k|) in 128 roundings that add like a random walk, 4 * 11 * 2^-24 S < 2^-18 S, which moves the result
    by that part of the greatest value; and 32-bit sums, statistics and exponentials, within 2^-18 of it."""
    n_tokens, heads, hd = q.shape
    group = heads // pages.heads
    out = np.full(q.shape, np.nan)
    tol = np.zeros(q.shape)
    for i in range(len(kv_len)):
        a, b, length = int(q_start[i]), int(q_start[i + 1]), int(kv_len[i])
        cap = table.shape[1] * pages.page
        length_c = min(max(length, 0), cap)
        ids = [int(table[i, j // pages.page]) for j in range(length_c)]
        live = np.array([0 <= p < len(pages.bytes) for p in ids], bool)
        kv = np.zeros((length_c, 2, pages.heads, hd))
        step = np.zeros((length_c, pages.heads))
        for j in range(length_c):
            if live[j]:
                kv[j] = pages.get(ids[j] * pages.page + j % pages.page)
                step[j] = pages.steps(ids[j] * pages.page + j % pages.page)
        for r in range(a, b):
            limit = length - (b - a) + (r - a) + 1
            if prefix is not None:
                limit = max(limit, int(prefix[i]))
            limit = max(0, min(limit, length_c))
            see = live[:limit]
            for h in range(heads):
                if not see.any():
                    out[r, h] = 0
                    continue
                k, v = kv[:limit, 0, h // group][see], kv[:limit, 1, h // group][see]
                z = k @ q[r, h].astype(np.float64) * scale
                size = float((np.abs(k) @ np.abs(q[r, h].astype(np.float64))).max() * abs(scale))
                p = np.exp(z - z.max())
                p /= p.sum()
                out[r, h] = p @ v
                tol[r, h] = (2 ** -11 * (np.abs(out[r, h]) + 8 * (p @ step[:limit, h // group][see])) +
                             2 ** -18 * (1 + size) * np.abs(v).max() + 2 ** -24)
    return out, tol
