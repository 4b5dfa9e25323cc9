"""Plain 64-bit forms of the serving operators of a ragged batch (cache append with rotation, chunk attention, sampling),
written from their definitions with loops over sequences, and the inputs the tests share."""
import numpy as np

from oracle import oracle as O

SENTINEL = 0xFFFFFFFF


def bf16(x):
    """f32 -> the f32 value of its nearest bf16."""
    return O.bf16_to_f32(O.f32_to_bf16(np.ascontiguousarray(x, np.float32)))


class Batch:
    """A ragged batch over a paged cache: `new` and `total` tokens per sequence, shuffled blocks, unused table entries
    SENTINEL.  The pools hold values of their type; `poison` fills everything that no visible key occupies with NaN."""

    def __init__(self, new, total, heads=8, kv_heads=2, dh=128, block=16, pool_bf16=True, pad_rows=0, seed=0, spare_blocks=2,
                 q_scale=1.0, poison=False):
        rng = np.random.default_rng(seed)
        self.new, self.total, self.heads, self.kv_heads, self.dh, self.block = list(new), list(total), heads, kv_heads, dh, block
        self.pool_bf16 = pool_bf16
        self.batch, self.rows = len(new), int(sum(new)) + pad_rows
        used = [-(-t // block) for t in total]
        self.width = max(1, max(used) + 1)
        self.blocks = sum(used) + spare_blocks
        order = rng.permutation(self.blocks).astype(np.uint32)
        self.tables = np.full((self.batch, self.width), SENTINEL, np.uint32)
        at = 0
        for b, u in enumerate(used):
            self.tables[b, :u] = order[at:at + u]
            at += u
        self.q_starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.seq_lens = np.array(total, np.uint32)
        ekv = kv_heads * dh
        self.k = rng.standard_normal((self.blocks, block, ekv)).astype(np.float32)
        self.v = rng.standard_normal((self.blocks, block, ekv)).astype(np.float32)
        if pool_bf16:
            self.k, self.v = bf16(self.k), bf16(self.v)
        if poison:
            live = np.zeros((self.blocks, block), bool)
            for b, t in enumerate(total):
                pos = np.arange(t)
                live[self.tables[b, pos // block], pos % block] = True
            self.k[~live] = np.nan
            self.v[~live] = np.inf
            self.v[~live, ::2] = np.nan
        self.q = (rng.standard_normal((self.rows, heads * dh)) * q_scale).astype(np.float32)

    def places(self, b):
        pos = np.arange(self.total[b])
        return self.tables[b, pos // self.block], pos % self.block

    def pool_array(self, x):
        return O.f32_to_bf16(x.ravel()).reshape(x.shape) if self.pool_bf16 else x


def attention_ref(bt, q, scale, split_terms=True):
    """(out, bound): f64 results [rows, heads * dh] (NaN behind the last sequence) and, per element, how far an evaluation in
    32 bits may be off.

    The bound: a score is a sum of dh products; whatever the order of the f32 sum, its error is at most
    ds = (dh + 8) 2^-23 scale sum_d |q_d k_d| (2^-23: the tensor cores may cut instead of rounding; three bf16 terms hold an f32
    q to 2^-24, which the 8 covers).  A weight then is off by a factor e^(2 ds) (its own score and the maximum's) times
    1 + 2^-21 (exponential and its argument, 2 ulp of an argument below 16) and, for its two bf16 terms, 1 + 2^-16.  The sums
    of n weights and of n weighted values add n 2^-23 each.  With one bf16 term (`split_terms` false) a weight is off by
    2^-8 instead of 2^-16.  All factors act on sum_j p_j |v_j|."""
    out = np.full((bt.rows, bt.heads * bt.dh), np.nan)
    bound = np.zeros_like(out)
    g = bt.heads // bt.kv_heads
    for b in range(bt.batch):
        n, t = bt.new[b], bt.total[b]
        blk, off = bt.places(b)
        kk = bt.k[blk, off].astype(np.float64).reshape(t, bt.kv_heads, bt.dh)
        vv = bt.v[blk, off].astype(np.float64).reshape(t, bt.kv_heads, bt.dh)
        for i in range(n):
            row = int(bt.q_starts[b]) + i
            see = t - n + i + 1
            qq = q[row].astype(np.float64).reshape(bt.heads, bt.dh)
            for h in range(bt.heads):
                ks, vs = kk[:see, h // g], vv[:see, h // g]
                s = ks @ qq[h] * scale
                ds = (bt.dh + 8) * 2.0 ** -23 * abs(scale) * (np.abs(ks) @ np.abs(qq[h])).max()
                p = np.exp(s - s.max())
                p /= p.sum()
                sl = slice(h * bt.dh, (h + 1) * bt.dh)
                out[row, sl] = p @ vs
                rel = np.expm1(2 * ds + 2.0 ** -21) + (2.0 ** -16 if split_terms else 2.0 ** -8) + 2 * see * 2.0 ** -23
                bound[row, sl] = 2 * rel * (p @ np.abs(vs))
    return out, bound


def append_ref(bt, qkv, cos, sin, rotary, adjacent, positions=None):
    """(q [rows, heads * dh], k pool, v pool) in f64 before the rounding to their types, and the same shapes of
    |a cos| + |b sin|, which bounds the f32 error of a rotated element by 2^-23 of it."""
    h, kv, dh = bt.heads, bt.kv_heads, bt.dh
    q = np.full((bt.rows, h * dh), np.nan)
    qm = np.zeros_like(q)
    k, v = bt.k.astype(np.float64), bt.v.astype(np.float64)
    km, vm = np.zeros_like(k), np.zeros_like(v)
    for b in range(bt.batch):
        for i in range(bt.new[b]):
            row = int(bt.q_starts[b]) + i
            pos = bt.total[b] - bt.new[b] + i
            ang = pos if positions is None else int(positions[row])
            x = qkv[row].astype(np.float64).reshape(h + 2 * kv, dh)
            c, s = cos[ang].astype(np.float64), sin[ang].astype(np.float64)
            y, m = x.copy(), np.abs(x)
            for p in range(rotary // 2):
                ia, ib = (2 * p, 2 * p + 1) if adjacent else (p, p + rotary // 2)
                a, bb = x[:h + kv, ia], x[:h + kv, ib]
                y[:h + kv, ia], y[:h + kv, ib] = a * c[p] - bb * s[p], bb * c[p] + a * s[p]
                m[:h + kv, ia], m[:h + kv, ib] = abs(a * c[p]) + abs(bb * s[p]), abs(bb * c[p]) + abs(a * s[p])
            q[row], qm[row] = y[:h].ravel(), m[:h].ravel()
            blk, off = int(bt.tables[b, pos // bt.block]), pos % bt.block
            k[blk, off], km[blk, off] = y[h:h + kv].ravel(), m[h:h + kv].ravel()
            v[blk, off], vm[blk, off] = y[h + kv:].ravel(), 0.0
    return (q, k, v), (qm, km, vm)


def sample_ref(x, t, k, p, m, u):
    """(id, prob, kept, gap) of one row in f64; `gap` is the smallest relative distance of a border (top-p, the draw) to the running
    sums it is compared with: a decision is only well defined where that is well above 1e-13."""
    x = np.asarray(x, np.float64)
    bad = np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any()
    if bad or not (0 <= t < np.inf) or np.isnan(p) or np.isnan(m) or not (0 <= u < 1):
        return -1, 0.0, 0, 1.0
    if t == 0:
        return int(np.argmax(x)), 1.0, 1, 1.0
    live = [i for i in sorted(range(len(x)), key=lambda i: (-x[i], i)) if x[i] > -np.inf]
    if k > 0:
        live = live[:k]
    w = np.exp((x[live] - x[live[0]]) / t)
    gap = 1.0
    if p < 1:
        c = np.cumsum(w)
        n = int(np.searchsorted(c, p * c[-1])) + 1 if p > 0 else 1
        if p > 0:
            gap = min(gap, np.abs(c[:-1] / c[-1] - p).min() if len(c) > 1 else 1.0)
        live, w = live[:n], w[:n]
    n = max(1, int((w >= m).sum()))
    live, w = np.array(live[:n]), w[:n]
    o = np.argsort(live)
    live, w = live[o], w[o]
    c = np.cumsum(w)
    i = min(int(np.searchsorted(c, u * c[-1], side="right")), len(c) - 1) if u > 0 else 0
    if len(c) > 1 and u > 0:          # u = 0 draws the first kept token whatever its weight: every weight is positive
        gap = min(gap, np.abs(c[:-1] / c[-1] - u).min())
    return int(live[i]), w[i] / c[-1], len(live), gap
