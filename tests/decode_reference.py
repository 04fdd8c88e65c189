"""Plain models of the decoding operators for the tests: the paged cache's bookkeeping
in Python, tree attention in 64 bits, beam selection in 64 bits."""
import numpy as np


class PagedModel:
    """The cache's rules, row after row in Python lists."""

    def __init__(self, num_pages, max_seqs, page, width):
        self.page, self.width = page, width
        self.refs = [0] * num_pages
        self.rows = [[] for _ in range(max_seqs)]
        self.lens = [0] * max_seqs
        self.text = {}  # (page, slot) -> the value stored there

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def extend(self, seqs, counts):
        ps, free = self.page, self.free_pages()
        wishes, sharers = [], {}
        for i, (s, n) in enumerate(zip(seqs, counts)):
            last = None
            ok = n >= 0 and -(-(self.lens[s] + n) // ps) <= self.width
            if ok and n > 0 and self.lens[s] % ps:
                last = self.rows[s][self.lens[s] // ps]
                sharers.setdefault(last, []).append(i)
            wishes.append((max(0, -(-(self.lens[s] + n) // ps) - len(self.rows[s])) if ok else 0, last))
        held = list(self.refs)
        taken = 0
        for i, s in enumerate(seqs):
            need, last = wishes[i]
            copy = last is not None and not (held[last] == 1 or (len(sharers[last]) == held[last] and sharers[last][0] == i))
            taken += need + copy
            if not need + copy:
                continue
            if taken > len(free):
                continue
            mine = free[taken - need - copy:taken]
            for p in mine:
                self.refs[p] = 1
            if copy:
                at = self.lens[s] // ps
                self.rows[s][at] = mine[0]
                self.refs[last] -= 1
                for t in range(self.lens[s] % ps):
                    self.text[mine[0], t] = self.text.get((last, t))
            self.rows[s] += mine[copy:]

    def fork(self, src, dst):
        keep = [[] if s < 0 else self.rows[s][:-(-self.lens[s] // self.page)] for s in src]
        lens = [0 if s < 0 else self.lens[s] for s in src]
        for row in keep:
            for p in row:
                self.refs[p] += 1
        for d, row, n in zip(dst, keep, lens):
            for p in self.rows[d]:
                self.refs[p] -= 1
            self.rows[d], self.lens[d] = list(row), n

    def truncate(self, s, n):
        if not 0 <= n <= self.lens[s]:
            return
        keep = -(-n // self.page)
        for p in self.rows[s][keep:]:
            self.refs[p] -= 1
        self.rows[s], self.lens[s] = self.rows[s][:keep], n

    def commit(self, s, n):
        if n >= 0 and self.lens[s] + n <= len(self.rows[s]) * self.page:
            self.lens[s] += n

    def place(self, s, t):
        return self.rows[s][t // self.page], t % self.page

    def store(self, s, values):
        """Past the length; what does not fit is dropped."""
        for t, x in enumerate(values, self.lens[s]):
            if t < len(self.rows[s]) * self.page:
                self.text[self.place(s, t)] = x

    def accept(self, s, parents, tokens, ids):
        n, at, path = len(parents), 0, []
        while at is not None and n:
            path.append(at)
            at = next((j for j in range(at + 1, n) if parents[j] == at and tokens[j] == ids[path[-1]]), None)
        if self.lens[s] + n > len(self.rows[s]) * self.page:
            path = []
        old = [self.text.get(self.place(s, self.lens[s] + j)) for j in path]
        for i, x in enumerate(old):
            self.text[self.place(s, self.lens[s] + i)] = x
        new = self.lens[s] + len(path)
        self.lens[s] = new
        self.truncate(s, new)
        return [ids[j] for j in path]


def tree_reference(c, layer, seqs, lens, q, k, v, masks, n_nodes, scale):
    """In 64 bits from the pools of a PagedCache: out, lse, and for the tolerances the sum of softmax weights times
    |v|, the largest sum of |q k| in a score, and the largest weight."""
    import torch
    B, N, Hq, D = q.shape
    G = Hq // k.shape[2]
    tables = c.tables.cpu().long()
    out = torch.zeros((B, N, Hq, D), dtype=torch.float64)
    weight, lse, spread = torch.zeros_like(out), torch.full((B, N, Hq), float("-inf"), dtype=torch.float64), torch.zeros((B, N, Hq), dtype=torch.float64)
    peak = torch.zeros_like(spread)
    for b in range(B):
        L, m = int(lens[b]), int(n_nodes[b])
        if m == 0:
            continue
        t = torch.arange(L)
        page, slot = tables[int(seqs[b]), t // c.page_size].to(c.k.device), (t % c.page_size).to(c.k.device)
        kk = torch.cat([c.k[layer, page, :, slot], k[b, :m]]).double().cpu().permute(1, 0, 2)
        vv = torch.cat([c.v[layer, page, :, slot], v[b, :m]]).double().cpu().permute(1, 0, 2)
        qq = q[b, :m].double().cpu().permute(1, 0, 2)
        sees = torch.ones((m, L + m), dtype=torch.bool)
        for i in range(m):
            bits = int(masks[b][i])
            for j in range(m):
                sees[i, L + j] = bool(bits >> j & 1)
        for h in range(Hq):
            z = (qq[h] @ kk[h // G].T * scale).masked_fill(~sees, float("-inf"))
            w = torch.softmax(z, 1)
            w = torch.where(sees.any(1, keepdim=True), w, torch.zeros_like(w))
            use = w > 0
            vh = vv[h // G]
            for i in range(m):
                sel = use[i] if torch.isfinite(z[i][sees[i]]).all() else sees[i]
                out[b, i, h] = w[i, sel] @ vh[sel]
                weight[b, i, h] = w[i, sel] @ vh[sel].abs()
            lse[b, :m, h] = torch.logsumexp(z, 1)
            peak[b, :m, h] = w.max(1).values
            mags = (qq[h].abs() @ kk[h // G].abs().T * abs(scale)).masked_fill(~sees, 0.0)
            spread[b, :m, h] = mags.max(1).values if L + m else 0.0
    return out, lse, weight, spread, peak


def beam_reference(x, scores, finished, allowed, pad):
    """Scores in 64 bits, [batch, beams * vocab], from logits as float64."""
    B, W = scores.shape
    V = x.shape[1]
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    if allowed is not None:
        x = np.where(allowed, x, -np.inf)
    top = x.max(1, keepdims=True)
    base = np.where(np.isfinite(top), top, 0.0)
    with np.errstate(divide="ignore"):
        lse = base + np.log(np.exp(x - base).sum(1, keepdims=True))
    s = np.where(np.isfinite(lse), x - np.where(np.isfinite(lse), lse, 0.0), -np.inf).reshape(B, W, V) + scores.astype(np.float64)[:, :, None]
    if finished is not None:
        f = finished.astype(bool)
        s[f] = -np.inf
        s[f, pad] = scores.astype(np.float64)[f]
    return np.where(np.isnan(s), -np.inf, s).reshape(B, W * V)
