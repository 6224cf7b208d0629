"""Drafted trees, beams, reordered states and pages from their definitions, in 64 bits on the
CPU, one row, node or entry after another."""
import math

import torch

F64 = torch.float64
PAGE = 16


# ---------------------------------------------------------------------- trees
def ancestors(parents, counts=None):
    """(sets of visible nodes, depths) of parents [rows][nodes]."""
    sets, depths = [], []
    for r, row in enumerate(parents.tolist()):
        n = len(row) if counts is None else max(0, min(int(counts[r]), len(row)))
        s, d = [], []
        for t, p in enumerate(row):
            if t >= n:
                s.append(set())
                d.append(0)
                continue
            p = p if -1 <= p < t else -1
            s.append({t} | (s[p] if p >= 0 else set()))
            d.append(d[p] + 1 if p >= 0 else 0)
        sets.append(s)
        depths.append(d)
    return sets, depths


def words(sets, nodes):
    """int64 [rows][nodes][ceil(nodes / 64)] of sets of nodes."""
    out = torch.zeros(len(sets), nodes, -(-nodes // 64), dtype=torch.int64)
    for r, row in enumerate(sets):
        for t, s in enumerate(row):
            for w in range(out.shape[2]):
                v = sum(1 << (n - 64 * w) for n in s if n // 64 == w)
                out[r, t, w] = v - (1 << 64) if v >> 63 else v
    return out


def accept(tokens, parents, picks, counts=None):
    rows, nodes = tokens.shape
    path = torch.full((rows, nodes), -1, dtype=torch.int32)
    accepted, after = [], []
    for r in range(rows):
        n = nodes if counts is None else max(0, min(int(counts[r]), nodes))
        cur, way, want = 0, [], -1
        while n and cur is not None:
            way.append(cur)
            want = int(picks[r, cur])
            cur = next((t for t in range(cur + 1, n) if int(parents[r, t]) == way[-1] and
                        int(tokens[r, t]) == want), None)
        path[r, :len(way)] = torch.tensor(way, dtype=torch.int32)
        accepted.append(len(way))
        after.append(want)
    return path, torch.tensor(accepted, dtype=torch.int32), torch.tensor(after, dtype=torch.int32)


def attention(q, k_pool, v_pool, table, lengths, masks, counts=None, scale=None):
    """(f64 outputs [rows][nodes][heads][dim], the sums of |p v| that bound their rounding);
    NaN where a node is not there."""
    q, k_pool, v_pool = q.cpu().to(F64), k_pool.cpu(), v_pool.cpu()
    table, masks = table.cpu(), masks.cpu()
    rows, nodes, heads, dim = q.shape
    g = heads // k_pool.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=F64)
    size = torch.zeros(q.shape, dtype=F64)
    for b in range(rows):
        n = nodes if counts is None else max(0, min(int(counts[b]), nodes))
        L = int(lengths[b])
        at = torch.arange(L + n)
        page, off = table[b, at // PAGE].long(), at % PAGE
        for t in range(n):
            see = [j for j in range(n) if (int(masks[b, t, j // 64]) >> (j % 64)) & 1]
            idx = torch.cat((torch.arange(L), torch.tensor(see, dtype=torch.int64) + L))
            if not len(idx):
                out[b, t] = 0
                continue
            k = k_pool[page[idx], :, off[idx]].to(F64)
            v = v_pool[page[idx], :, off[idx]].to(F64)
            for h in range(heads):
                p = torch.softmax(scale * (k[:, h // g] @ q[b, t, h]), 0)
                out[b, t, h] = p @ v[:, h // g]
                size[b, t, h] = p @ v[:, h // g].abs()
    return out, size


# ---------------------------------------------------------------------- beams
def beam(logits, scores, lengths, done, *, eos=None, penalty=0.0):
    """(parents, tokens, scores f64, lengths, done) by sorting every candidate."""
    x = logits.cpu().to(F64)
    groups, K = scores.shape
    V = x.shape[1]
    big = torch.finfo(torch.float32).max
    out = ([], [], [], [], [])
    for g in range(groups):
        cands = []
        for b in range(K):
            row = g * K + b
            s = float(scores[g, b])
            n = int(lengths[g, b]) if lengths is not None else 0
            over = bool(done[g, b]) if done is not None else False
            if not math.isfinite(s):
                continue
            if over:
                cands.append((-s / max(n, 1) ** penalty, b, 0.0, -1 if eos is None else eos, s, n,
                              True))
                continue
            l = torch.where(torch.isnan(x[row]), -math.inf, x[row]).clamp(max=big)
            top = float(l.max())
            log_sum = float(torch.log(torch.exp(l - top).sum()))
            order = torch.sort(l, descending=True, stable=True)
            for v, t in zip(order.values[:K].tolist(), order.indices[:K].tolist()):
                if v > -math.inf:
                    c = s + ((v - top) - log_sum)
                    cands.append((-c / max(n + 1, 1) ** penalty, b, -v, t, c, n + 1, t == eos))
        cands.sort(key=lambda c: c[:4])
        for i in range(K):
            if i < len(cands):
                _, b, _, t, c, n, d = cands[i]
                got = (g * K + b, t, c, n, d)
            else:
                got = (g * K + i, -1, -math.inf, int(lengths[g, i]) if lengths is not None else 0,
                       bool(done[g, i]) if done is not None else False)
            for o, v in zip(out, got):
                o.append(v)
    shape = (groups, K)
    return (torch.tensor(out[0], dtype=torch.int32).view(shape),
            torch.tensor(out[1], dtype=torch.int32).view(shape),
            torch.tensor(out[2], dtype=F64).view(shape),
            torch.tensor(out[3], dtype=torch.int32).view(shape),
            torch.tensor(out[4], dtype=torch.bool).view(shape))


# ---------------------------------------------------------------------- pages
class Cache:
    """What ``pages.Pages`` does, entry by entry, over pools on the CPU."""

    def __init__(self, pools, table, refs):
        self.pools, self.table, self.refs = pools, table, refs
        self.rows, self.max_pages = table.shape
        self.pages = refs.numel()
        self.failed = False

    def _held(self, page):
        return 0 <= page < self.pages

    def fork(self, parents, lengths):
        old, new = self.table.clone(), torch.full_like(self.table, -1)
        out = torch.zeros_like(lengths)
        for r in range(self.rows):
            p = int(parents[r])
            if not -1 <= p < self.rows:
                p, self.failed = r, True
            if p >= 0:
                out[r] = lengths[p]
                for c in range(self.max_pages):
                    if p == r or c * PAGE < int(lengths[p]):
                        new[r, c] = old[p, c]
        for t, by in ((old, -1), (new, 1)):
            for page in t.flatten().tolist():
                if self._held(page):
                    self.refs[page] += by
        self.table.copy_(new)
        return out

    def free(self, which):
        own = torch.arange(self.rows)
        self.fork(torch.where(which, -1, own), torch.zeros(self.rows, dtype=torch.int32))

    def take(self, lengths, n):
        wanted = []
        for r in range(self.rows):
            L, k = int(lengths[r]), n if isinstance(n, int) else int(n[r])
            if L < 0:
                self.failed = True
            elif k > 0:
                last = -(-(L + k) // PAGE)
                self.failed |= last > self.max_pages
                wanted += [(r, c) for c in range(L // PAGE, min(last, self.max_pages))]
        held = {}
        for r, c in wanted:
            held.setdefault(int(self.table[r, c]), []).append((r, c))
        before = self.refs.clone()
        free = [i for i in range(self.pages) if before[i] == 0]
        for r, c in wanted:
            page = int(self.table[r, c])
            if self._held(page):
                if before[page] == 1 or (len(held[page]) == before[page] and
                                         held[page][0] == (r, c)):
                    continue
                self.refs[page] -= 1
            elif page != -1:
                self.failed = True
            new = free.pop(0) if free else -1
            self.failed |= new < 0
            self.table[r, c] = new
            if new >= 0:
                self.refs[new] += 1
                if self._held(page) and c == int(lengths[r]) // PAGE and int(lengths[r]) % PAGE:
                    for p in self.pools:
                        p[new] = p[page]

    def keep(self, lengths, path, counts):
        out = lengths.clone()
        for r in range(self.rows):
            L, n = int(lengths[r]), int(counts[r])
            way = path[r, :max(n, 0)].tolist()
            if not 0 <= n <= path.shape[1] or any(
                    not i <= t < path.shape[1] or (i and t <= way[i - 1])
                    for i, t in enumerate(way)) or L < 0 or (
                    n and L + way[-1] >= self.max_pages * PAGE):
                self.failed = True
                continue
            out[r] = L + n
            for i, t in enumerate(way):
                a, b = int(self.table[r, (L + t) // PAGE]), int(self.table[r, (L + i) // PAGE])
                for p in self.pools:
                    p[b, :, (L + i) % PAGE] = p[a, :, (L + t) % PAGE]
        return out

    def compact(self):
        live = int((self.refs > 0).sum())
        moves = [i for i in range(live, self.pages) if self.refs[i] > 0]
        holes = [i for i in range(live) if self.refs[i] == 0]
        for a, b in zip(moves, holes):
            for p in self.pools:
                p[b] = p[a]
            self.refs[b], self.refs[a] = int(self.refs[a]), 0
            self.table[self.table == a] = b
        return live
