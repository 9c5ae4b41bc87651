"""Plain implementation in 64 bits of the paged 8-bit key/value cache and of beam selection.

Host code on numpy / CPU tensors, written from the definitions in include/cats_b200.h; independent
of the kernels."""
import numpy as np
import torch

EXP_MIN, EXP_MAX = -24, 60


def e4m3(x):
    """float64 array -> the nearest e4m3 values (ties to even, saturating at 448, NaN for what is not
    finite), by the format's definition: 3 bits behind the leading one, exponents -6 .. 8."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x)
    a = np.where(bad, 0.0, np.abs(x))
    _, e = np.frexp(a)                                  # a = m * 2^e, 0.5 <= m < 1
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    q = np.minimum(np.rint(a / step) * step, 448.0)     # rint: ties to even
    return np.where(bad, np.nan, np.copysign(q, x))


def exponent(amax):
    """Least e in EXP_MIN .. EXP_MAX with amax <= 448 * 2^e."""
    e = EXP_MIN
    while e < EXP_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """values [layers, pages, 2, heads, page, hd] (code values), exps [layers, pages, 2, heads],
    table, lens, refs: as in the struct, as numpy arrays."""

    def __init__(self, values, exps, table, lens, refs):
        self.values, self.exps = np.array(values, np.float64), np.array(exps, np.int64)
        self.table, self.lens, self.refs = (np.array(t, np.int64) for t in (table, lens, refs))
        self.page = self.values.shape[4]

    @classmethod
    def of(cls, cache):
        f = lambda t: t.cpu().numpy()  # noqa: E731
        vals = cache.codes.view(torch.uint8).cpu().view(torch.float8_e4m3fn).float().numpy()
        return cls(vals, np.round(np.log2(np.maximum(f(cache.scales), 2.0 ** -24))), f(cache.table), f(cache.lens),
                   f(cache.refs))

    def _pages(self, n):
        return -(-n // self.page)

    def _free(self):
        ids = np.nonzero(self.refs == 0)[0]
        return int(ids[0]) if len(ids) else -1

    def grow(self, counts):
        """Returns which sequences grew."""
        out, stuck = [], False
        free = list(np.nonzero(self.refs == 0)[0])
        for b, n in enumerate(counts):
            have, need = self._pages(self.lens[b]), self._pages(self.lens[b] + n)
            if need > self.table.shape[1]:
                out.append(False)
                continue
            if need > have:
                stuck = stuck or need - have > len(free)
                if stuck:
                    out.append(False)
                    continue
                for j in range(have, need):
                    self.table[b, j] = free.pop(0)
                    self.refs[self.table[b, j]] = 1
            self.lens[b] += n
            out.append(n > 0)
        return out

    def append(self, layer, qkv, counts, nh, cos=None, sin=None):
        """qkv [tokens, heads, hd] float64.  Returns the rotated queries."""
        qkv = np.array(qkv, np.float64)
        hd, nkv = self.values.shape[5], self.values.shape[3]
        q, t = np.zeros((len(qkv), nh, hd)), 0
        for b, n in enumerate(counts):
            for i in range(n):
                pos = self.lens[b] - n + i
                x = qkv[t]
                if cos is not None:
                    turned = np.concatenate((-x[:, hd // 2:], x[:, :hd // 2]), -1)
                    rot = x * cos[pos] + turned * sin[pos]
                else:
                    rot = x
                q[t] = rot[:nh]
                qkv[t, nh:nh + nkv] = rot[nh:nh + nkv]
                t += 1
            # page by page, all its new rows at once
            start, t0 = self.lens[b] - n, t - n
            for j in range(start // self.page, self._pages(self.lens[b])):
                a, z = max(start, j * self.page), min(self.lens[b], (j + 1) * self.page)
                if z <= a:
                    continue
                pid = self.table[b, j]
                rows = qkv[t0 + a - start:t0 + z - start, nh:].reshape(z - a, 2, nkv, hd)
                for kv in range(2):
                    for h in range(nkv):
                        r = rows[:, kv, h]
                        fin = np.abs(r[np.isfinite(r)])
                        e = exponent(fin.max() if fin.size else 0.0)
                        old = a - j * self.page
                        blk = self.values[layer, pid, kv, h]
                        if old:
                            e0 = self.exps[layer, pid, kv, h]
                            e = max(e, e0)
                            blk[:old] = e4m3(blk[:old] * 2.0 ** (e0 - e))
                        blk[old:z - j * self.page] = e4m3(r * 2.0 ** -e)
                        self.exps[layer, pid, kv, h] = e
        return q

    def rows(self, layer, b, n):
        """(keys, values) [heads, n, hd] of the first n positions of sequence b."""
        ids = self.table[b, :self._pages(n)]
        x = self.values[layer][ids] * np.exp2(self.exps[layer][ids].astype(np.float64))[..., None, None]
        x = x.transpose(1, 2, 0, 3, 4).reshape(2, x.shape[2], -1, x.shape[4])[:, :, :n]
        return x[0], x[1]

    def attend(self, layer, q, counts, scale=None):
        """q [tokens, nh, hd] float64.  Returns (out, bounds): bounds is a dict of what tolerances are
        made of, per output: pv = sum p |v|, s = max over keys of scale * sum |q k|, v = max |v|, n = keys."""
        q = np.asarray(q, np.float64)
        out = np.zeros_like(q)
        pv, smax, vmax, cnt = np.zeros_like(q), np.zeros(q.shape[:2]), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
        scale = q.shape[2] ** -0.5 if scale is None else scale
        group, t = q.shape[1] // self.values.shape[3], 0
        for b, n in enumerate(counts):
            for i in range(n):
                keys = self.lens[b] - n + i + 1
                if keys > 0:
                    k, v = self.rows(layer, b, keys)
                    for h in range(q.shape[1]):
                        kk, vv = k[h // group], v[h // group]
                        x = kk @ q[t, h] * scale
                        p = np.exp(x - x.max())
                        p /= p.sum()
                        out[t, h] = p @ vv
                        pv[t, h] = p @ np.abs(vv)
                        smax[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
                        vmax[t, h] = np.abs(vv).max()
                        cnt[t, h] = keys
                t += 1
        return out, {"pv": pv, "s": smax[..., None], "v": vmax[..., None], "n": cnt[..., None]}

    def reorder(self, parents):
        table, lens = self.table.copy(), self.lens.copy()
        n = len(parents)
        ok = [p if 0 <= p < n else -1 for p in parents]
        eldest = {}
        for i, p in enumerate(ok):
            if p >= 0:
                eldest.setdefault(p, i)
        copies = []
        for i in range(n):                              # what every old row held is let go ...
            for j in range(self._pages(lens[i])):
                if table[i, j] >= 0:
                    self.refs[table[i, j]] -= 1
        for i, p in enumerate(ok):                      # ... and taken up by its children
            self.table[i] = -1 if p < 0 else table[p]
            self.lens[i] = 0 if p < 0 else lens[p]
            if p < 0:
                continue
            full, part = lens[p] // self.page, lens[p] % self.page
            for j in range(full + (1 if part and eldest[p] == i else 0)):
                if table[p, j] >= 0:
                    self.refs[table[p, j]] += 1
            if part and eldest[p] != i:
                copies.append((i, full, table[p, full], part))
        for i, full, src, part in copies:
            dst = self._free() if src >= 0 else -1          # (a page that the parent lacks, the child lacks too)
            self.table[i, full] = dst
            if dst >= 0:
                self.refs[dst] = 1
                self.values[:, dst, :, :, :part] = self.values[:, src, :, :, :part]
                self.exps[:, dst] = self.exps[:, src]

    def compact(self):
        n = int((self.refs > 0).sum())
        holes = [i for i in range(n) if self.refs[i] == 0]
        movers = [i for i in range(n, len(self.refs)) if self.refs[i] > 0]
        for d, s in zip(holes, movers):
            self.values[:, d], self.exps[:, d] = self.values[:, s], self.exps[:, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.table[self.table == s] = d
        return n


def beam_select(logits, scores, k, done=None, eos=-1):
    """logits [n, beams, vocab], scores [n, beams]: (scores, rows, tokens, done) of the k best, best
    first, ties to the lowest (beam, token); float64."""
    x, scores = np.asarray(logits, np.float64), np.asarray(scores, np.float64)
    n, beams, vocab = x.shape
    done = np.zeros((n, beams), bool) if done is None else np.asarray(done, bool)
    out = []
    with np.errstate(all="ignore"):
        for i in range(n):
            c = np.full((beams, vocab), -np.inf)
            for w in range(beams):
                if not np.isfinite(scores[i, w]):
                    continue
                if done[i, w]:
                    c[w, eos] = scores[i, w]
                    continue
                top = x[i, w].max()
                lse = top + np.log(np.exp(x[i, w] - top).sum())
                if np.isfinite(lse):
                    c[w] = scores[i, w] + (x[i, w] - lse)
            flat = np.argsort(-c.reshape(-1), kind="stable")[:k]
            rows, toks = flat // vocab, flat % vocab
            out.append((c.reshape(-1)[flat], rows + i * beams, toks, done[i, rows] | (toks == eos)))
    return tuple(np.stack(v) for v in zip(*out))
