"""A plain paged 8-bit cache on the CPU, one position after the other, and the bound that an attention over it keeps.

Codes and scales follow the header's definition in fp32; attention is in 64 bits over the values they stand for.

bound() is derived for kernels that hold q as a sum of two fp16 numbers (relative 2^-22) and codes exactly, form
scores, the softmax and its sums in fp32, and for 16-bit rows hold q as given and the probabilities in
fp16 (relative 2^-11).  With S = max_j scale * sum_d |q_d K_jd| the absolute error of a score is at most
  ds = S * ((head_dim + 8) 2^-24 + 2^-22)      rounding of the sum of head_dim products, scale factors, q's split
so a probability is off by the factor exp(2 ds) at most (its own score and the maximum's), plus the exponential's
and the factors' own few roundings.  The sums over n positions add at most (n / 32 + 48) 2^-23 relative: a
matrix product or wave adds 32 positions at a time.  All of this is relative to A = sum_j p_j |V_j|, and a running
rescale of earlier pages adds one rounding per page, counted in n / 32.

A kernel of 16-bit rows may multiply code + 128 and subtract the 128 from the finished sums.  The summands of a score are
then q_d s_j (code + 128), those of an output p_j v_j (code + 128), and the roundings above are relative to these:
S and, for the sums over positions, A are formed of |K_jd| + 128 s_j and |V_j| + 128 v_j.

Two absolute terms.  A kernel that holds p_j times the V scale v_j in fp16, as one number or as the sum of two,
relative to 2^-14 of the largest such product of the row, rounds the smallest ones to multiples of 2^-24: an
error of 2^-39 max_i(p_i v_i) for each position, times a code of at most 127.  And a product below 2^-126 of the largest
one is lost in fp32, which takes as much as 2^-126 max(v) / v_j from the sum of the p for each position.
"""
import numpy as np

BLOCK = 32


class Pool:
    """Pages of sequences, by the order that the header states."""

    def __init__(self, seqs, max_len, pages):
        self.W, self.max_len = -(-max_len // BLOCK), max_len
        self.tables = [[] for _ in range(seqs)]
        self.stack = list(range(pages - 1, -1, -1))

    def plan(self, have, add, rows):
        """(starts, positions, slots, tables, row's sequence) or None, when nothing changes."""
        need = [-(-(h + a) // BLOCK) for h, a in zip(have, add)]
        held = sum(map(len, self.tables))
        if (min(have) < 0 or min(add) < 0 or max(h + a for h, a in zip(have, add)) > self.max_len or sum(add) > rows
                or sum(need) > held + len(self.stack)):
            return None
        for t, n in zip(self.tables, need):
            self.stack += t[n:]
            del t[n:]
        for t, n in zip(self.tables, need):
            while len(t) < n:
                t.append(self.stack.pop())
        starts = np.concatenate([[0], np.cumsum(add)])
        seq = [b for b, a in enumerate(add) for _ in range(a)]
        pos = [h + i for h, a in zip(have, add) for i in range(a)]
        slots = [self.tables[b][p // BLOCK] * BLOCK + p % BLOCK for b, p in zip(seq, pos)]
        tables = np.full((len(have), self.W), -1)
        for b, t in enumerate(self.tables):
            tables[b, :len(t)] = t
        return starts, np.array(pos, int), np.array(slots, int), tables, np.array(seq, int)


class Cache:
    """Codes and scales of one layer's K (or V): dicts by (page, head)."""

    def __init__(self, pages, heads, hd):
        self.codes = np.zeros((pages, heads, BLOCK, hd), np.int32)
        self.scales = np.zeros((pages, heads), np.float32)

    def append(self, x, slots):
        x = np.asarray(x, np.float32)
        t = 0
        while t < len(slots):
            page, f = slots[t] // BLOCK, slots[t] % BLOCK
            m = 1
            while f + m < BLOCK and t + m < len(slots) and slots[t + m] == slots[t] + m:
                m += 1
            for g in range(x.shape[1]):
                self._run(page, g, f, x[t:t + m, g])
            t += m

    def _run(self, page, g, f, x):
        a = np.abs(x)
        finite = a[np.isfinite(a)]
        t = np.float32((finite.max() if finite.size else np.float32(0)) / np.float32(127))
        if t < 2.0 ** -100:
            t = np.float32(0)
        s = self.scales[page, g] if f else np.float32(0)
        if s > 0:
            k = 0
            while np.float64(s) * 2.0 ** k < t:
                k += 1
            if k:
                self.codes[page, g, :f] = np.rint(self.codes[page, g, :f] * 2.0 ** -k).astype(np.int32)
            s = np.float32(np.float64(s) * 2.0 ** k)
        else:
            s = t
        with np.errstate(all="ignore"):
            q = np.clip(np.rint(x / s), -127, 127) if s > 0 else np.zeros_like(x)
        self.codes[page, g, f:f + len(x)] = np.where(np.isnan(q), 0, q).astype(np.int32)
        self.scales[page, g] = s

    def values(self, table, n):
        """[n][heads][hd] in fp32: positions 0..n-1 of a sequence."""
        idx = np.asarray(table[:-(-n // BLOCK)], int)
        v = self.codes[idx].astype(np.float32) * self.scales[idx][:, :, None, None]
        return v.transpose(0, 2, 1, 3).reshape(-1, v.shape[1], v.shape[3])[:n]

    def scale_of(self, table, n):
        """[n][heads]: the scale of each position's page."""
        idx = np.asarray(table[:-(-n // BLOCK)], int)
        return np.repeat(self.scales[idx].astype(np.float64), BLOCK, axis=0)[:n]


def attend(q, K, V, ks, vs, have, scale, half_eps):
    """(out, bound) in 64 bits of rows q [n][H][hd] over K, V [have + n][KVH][hd] with scales ks, vs [have + n][KVH]; half_eps:
    half a step of out's type."""
    add = 128 if half_eps > 2.0 ** -20 else 0
    n, H, hd = q.shape
    G = H // K.shape[1]
    out, bound = np.zeros((n, H, hd)), np.zeros((n, H, hd))
    K, V = K.astype(np.float64), V.astype(np.float64)
    L = have + 1 + np.arange(n)                        # positions that a row looks at
    seen = np.arange(have + n)[None, :] < L[:, None]
    for h in range(H):
        kk, vv, k_s, v_s = K[:have + n, h // G], V[:have + n, h // G], ks[:have + n, h // G], vs[:have + n, h // G]
        y = q[:, h].astype(np.float64)
        with np.errstate(invalid="ignore"):
            s = np.where(seen, scale * (y @ kk.T), -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
        l = p.sum(1, keepdims=True)
        out[:, h] = p @ vv / l
        A = p @ np.abs(vv) / l
        S = np.where(seen, scale * (np.abs(y) @ np.abs(kk).T + add * k_s[None, :] * np.abs(y).sum(1, keepdims=True)), 0)
        ds = S.max(1, keepdims=True) * ((hd + 8) * 2.0 ** -24 + 2.0 ** -22)
        w = np.where(seen, np.maximum(v_s, 2.0 ** -100)[None, :], np.nan)
        rel, sums = np.expm1(2 * ds), (L[:, None] / 32 + 48) * 2.0 ** -23
        if half_eps > 2.0 ** -20:
            rel = rel + 2.0 ** -11
        rel = rel + L[:, None] * 2.0 ** -126 * np.nanmax(w, 1, keepdims=True) / np.nanmin(w, 1, keepdims=True)
        err = A * rel + (A + add * (p @ v_s)[:, None] / l) * sums
        err = err + L[:, None] * 2.0 ** -39 * 127 * np.nanmax(p * w, 1, keepdims=True) / l
        bound[:, h] = err + (np.abs(out[:, h]) + err) * half_eps
    return out, bound
