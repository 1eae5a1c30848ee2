"""Plain 64-bit forms of attention over a cache of rows, of the weight that rows receive and of their removal, for small inputs, and the
bounds that follow from the roundings the kernels make."""
import numpy as np

from tests import helpers as H

F = np.float32
NONE = 0xFFFFFFFF
EPS_F32 = 2.0 ** -24


def as_type(x, bf16):
    """float32 values that the type holds, and what goes to the device."""
    x = np.ascontiguousarray(x, F)
    if not bf16:
        return x, x
    v = H.to_bf16_f32(x).reshape(x.shape)
    return v, (v.view(np.uint32) >> 16).astype(np.uint16)


def from_bf16(u):
    return (np.ascontiguousarray(u).astype(np.uint32) << 16).view(F)


def family(parents):
    """[token][token]: whether the second is the first or an ancestor of it; depths."""
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while True:
            m[i, j] = True
            p = int(parents[j])
            if not p < j:
                break
            j = p
    return m, m.sum(1) - 1


class Call:
    """One call's inputs as arrays: keys, values [total][kv_head][d], q [token][head][d] (float32 values), the segments (begin, rows, query_begin, queries,
    base) and what attention is told."""

    def __init__(self, keys, values, q, segs, scale, softcap=0.0, slopes=None, window=0, causal=True, prefix=None, row_pos=None, row_doc=None, q_pos=None,
                 q_doc=None, parents=None, rows=None):
        self.__dict__.update(locals())
        self.kv, self.d = keys.shape[1:]
        self.heads = q.shape[1]
        self.group = self.heads // self.kv

    def seen(self, i, h):
        """[token][row] for KV head h of segment i, and the distances."""
        b, n, q0, t, base = self.segs[i]
        if self.rows is not None:
            n = min(n, int(self.rows[i]))
        ctx = n - min(n, t)
        rp = base + np.arange(n, dtype=np.int64) if self.row_pos is None else self.row_pos[h][b:b + n].astype(np.int64)
        qp = base + ctx + np.arange(t, dtype=np.int64) if self.q_pos is None else self.q_pos[q0:q0 + t].astype(np.int64)
        fam = None
        if self.parents is not None:
            fam, depth = family(self.parents[q0:q0 + t])
            if self.row_pos is None:
                rp[ctx:] = base + ctx + depth[:n - ctx]
            if self.q_pos is None:
                qp = base + ctx + depth
        away = qp[:, None] - rp[None]
        ok = np.ones_like(away, bool) if not self.causal else away >= 0
        if self.window:
            ok &= np.abs(away) < self.window
        if self.prefix is not None:
            ok |= (rp < int(self.prefix[i]))[None]
        if self.row_doc is not None:
            ok &= self.row_doc[h][b:b + n][None] == self.q_doc[q0:q0 + t][:, None]
        if fam is not None:
            ok[:, ctx:] &= fam[:, :n - ctx]
        return n, ok, np.abs(away)

    def scores(self, i, h, n, ok, away):
        """[group][token][row] scores (-inf where not seen) and a bound on what a float32 computation of them is off by."""
        b, _, q0, t, _ = self.segs[i]
        hs = slice(h * self.group, (h + 1) * self.group)
        q, k = self.q[q0:q0 + t, hs].astype(np.float64), self.keys[b:b + n, h].astype(np.float64)
        k = np.where(ok.any(0)[:, None], k, 0.0)
        s = np.einsum("tgd,rd->gtr", q, k) * float(F(self.scale))
        # d products and sums in float32 (float32 factors as two tf32 numbers: 2^-21 of a term more); the scaling; cap and bias: a few roundings of their size
        off = np.einsum("tgd,rd->gtr", np.abs(q), np.abs(k)) * abs(self.scale) * ((self.d + 8) * EPS_F32 + 2.0 ** -21)
        if self.softcap:
            s = self.softcap * np.tanh(s / self.softcap)
            off = off + 4 * 2.0 ** -23 * self.softcap
        if self.slopes is not None:
            s = s - self.slopes[hs].astype(np.float64)[:, None, None] * away
        off = off + 2.0 ** -22 * (np.abs(s) + 1.0)
        return np.where(ok, s, -np.inf), np.where(ok, off, 0.0)

    def attend(self, bf16):
        """out, lse and how far each may be off; NaN where no segment has the token."""
        out = np.full(self.q.shape, np.nan)
        lse, out_tol, lse_tol = np.full(self.q.shape[:2], np.nan), np.zeros(self.q.shape), np.zeros(self.q.shape[:2])
        for i, (b, _, q0, t, _) in enumerate(self.segs):
            for h in range(self.kv if t else 0):
                n, ok, away = self.seen(i, h)
                s, off = self.scores(i, h, n, ok, away)
                v = np.where(ok.any(0)[:, None], self.values[b:b + n, h].astype(np.float64), 0.0)
                top = s.max(-1, keepdims=True, initial=-np.inf)
                p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
                total = p.sum(-1)
                w = p / np.where(total > 0, total, 1.0)[..., None]
                hs = slice(h * self.group, (h + 1) * self.group)
                o = np.stack([np.stack([w[g, r][ok[r]] @ v[ok[r]] if ok[r].any() else np.zeros(self.d) for r in range(t)]) for g in range(self.group)])
                mag = np.einsum("gtr,rd->gtd", w, np.abs(np.where(np.isfinite(v), v, 0.0)))
                worst = off.max(-1, initial=0.0)
                # weights off by e^(2 worst) - 1 and sums of n terms in float32; bfloat16: each weight and the result rounded by half a step
                rel = 2 * worst + (n / 8 + 48) * EPS_F32 + 2.0 ** -20
                tol = rel[..., None] * mag + 1e-30
                if bf16:
                    tol = tol + 2.0 ** -8 * mag + 2.0 ** -8 * (np.abs(o) + tol + 2.0 ** -8 * mag)
                out[q0:q0 + t, hs] = o.transpose(1, 0, 2)
                out_tol[q0:q0 + t, hs] = tol.transpose(1, 0, 2)
                with np.errstate(divide="ignore"):
                    z = np.log(total) + np.where(np.isfinite(top), top, 0.0)[..., 0]
                lse[q0:q0 + t, hs] = z.T
                lse_tol[q0:q0 + t, hs] = (worst + (n / 8 + 48) * EPS_F32 + 2.0 ** -21 * (1 + np.abs(np.where(np.isfinite(z), z, 0.0)))).T
        return out, lse, out_tol, lse_tol

    def received(self, lse, before, decay):
        """weights [kv_head][row] for the lse that is handed in, and how far they may be off."""
        w, tol = before.astype(np.float64).copy(), np.zeros(before.shape)
        for i, (b, _, q0, t, _) in enumerate(self.segs):
            for h in range(self.kv):
                n, ok, away = self.seen(i, h)
                s, off = self.scores(i, h, n, ok, away)
                hs = slice(h * self.group, (h + 1) * self.group)
                z = lse[q0:q0 + t, hs].astype(np.float64).T[:, :, None]
                with np.errstate(invalid="ignore"):
                    p = np.where(np.isfinite(z) & ok[None], np.exp(s - z), 0.0)
                add = p.sum((0, 1))
                w[h, b:b + n] = decay * before[h, b:b + n].astype(np.float64) + add
                # e^off - 1, the exponent's own rounding, the exponential's 2^-22, the sum's terms
                tol[h, b:b + n] = (p * (off + 2.0 ** -20 + 2.0 ** -22 * np.abs(np.where(np.isfinite(s - np.where(np.isfinite(z), z, 0.0)), s - np.where(np.isfinite(z), z, 0.0), 0.0)))).sum((0, 1)) + \
                    (self.group * t + 8) * EPS_F32 * add + 4 * EPS_F32 * np.abs(w[h, b:b + n]) + 1e-37
        return w, tol


def evict(weights, positions, budget, sink, recent):
    """The row that comes to each place: one KV head of one segment, row by row."""
    n = len(weights)
    if n <= budget:
        return np.arange(n)
    newest = int(positions.max())
    pinned = [int(p) < sink or (recent > 0 and newest - int(p) < recent) for p in positions]
    key = [0.0 if pinned[r] else (np.inf if np.isnan(weights[r]) else -float(weights[r])) for r in range(n)]
    rank = sorted(range(n), key=lambda r: (not pinned[r], np.isnan(weights[r]) and not pinned[r], key[r], r))
    keep = set(rank[:budget])
    late = iter(r for r in range(budget, n) if r in keep)
    return np.array([r if r in keep else next(late) for r in range(budget)])
