"""A plain model of the paged cache on lists and CPU tensors: what the device calls are compared with."""

import torch


class ModelCache:
    def __init__(self, cache):
        self.k, self.v = cache.k.cpu().clone(), cache.v.cpu().clone()
        self.table, self.lens, self.refs = cache.page_table.cpu().tolist(), cache.seq_lens.cpu().tolist(), cache.ref_counts.cpu().tolist()
        self.page = self.k.shape[3]
        self.scale = None if cache.k_scale is None else (cache.k_scale.cpu(), cache.v_scale.cpu())

    def pages(self, n):
        return -(-n // self.page)

    def bytes(self, pool):
        return pool.view(torch.uint8) if pool.element_size() == 1 else pool.view(torch.int16)

    def move(self, src, dst, tokens):
        for pool in (self.bytes(self.k), self.bytes(self.v)):
            pool[:, dst, :, :tokens] = pool[:, src, :, :tokens].clone()

    def claim(self, n):
        got = [p for p, r in enumerate(self.refs) if r == 0][:n]
        if len(got) < n:
            return None
        for p in got:
            self.refs[p] = 1
        return got

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < len(self.lens):
                continue
            for j in range(self.pages(self.lens[s])):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = 0

    def extend(self, seqs, n_new):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.lens) for s in seqs) or any(x < 0 for x in n_new):
            return False
        if any(self.lens[s] + x > len(self.table[s]) * self.page for s, x in zip(seqs, n_new)):
            return False
        need = [self.pages(self.lens[s] + x) - self.pages(self.lens[s]) for s, x in zip(seqs, n_new)]
        got = self.claim(sum(need))
        if got is None:
            return False
        for s, x, m in zip(seqs, n_new, need):
            first = self.pages(self.lens[s])
            self.table[s][first:first + m], got = got[:m], got[m:]
            self.lens[s] += x
        return True

    def stored(self, x, which, layer):
        """What the pool holds for values [Hkv, D] of one token."""
        if self.scale is None:
            return x
        q = x.float() / self.scale[which][layer][:, None]
        codes = q.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return codes.masked_fill(q.isnan(), 0x7f).view(torch.float8_e4m3fn)  # NaN has two codes: the one without a sign

    def write(self, k, v, seqs, n_new, layer):
        for i, s in enumerate(seqs):
            if not 0 <= s < len(self.lens):
                continue
            n = k.shape[2] if n_new is None else n_new[i]
            for t in range(min(n, k.shape[2])):
                pos = self.lens[s] - n + t
                if pos < 0:
                    continue
                p = self.table[s][pos // self.page]
                for which, (pool, x) in enumerate(((self.k, k), (self.v, v))):
                    self.bytes(pool)[layer, p, :, pos % self.page] = self.bytes(self.stored(x[i, :, t].cpu(), which, layer))

    def fork(self, parents, children):
        if len(set(children)) < len(children) or set(parents) & set(children):
            return False
        if any(not 0 <= s < len(self.lens) for s in parents + children) or any(self.lens[c] for c in children):
            return False
        parts = [self.lens[p] % self.page for p in parents]
        got = self.claim(sum(x > 0 for x in parts))
        if got is None:
            return False
        for p, c, part in zip(parents, children, parts):
            full = self.lens[p] // self.page
            self.table[c][:full] = self.table[p][:full]
            for x in self.table[p][:full]:
                self.refs[x] += 1
            if part:
                self.table[c][full] = got.pop(0)
                self.move(self.table[p][full], self.table[c][full], part)
            self.lens[c] = self.lens[p]
        return True

    def copy_pages(self, src, dst):
        live = [(s, d) for s, d in zip(src, dst)]
        for i, (s, d) in enumerate(live):
            if s < 0 or d < 0 or s >= len(self.refs) or d >= len(self.refs):
                continue
            if d in src or s in dst or any(j != i and x == d for j, (_, x) in enumerate(live)):
                continue
            self.move(s, d, self.page)

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] == 0]
        to = {}
        for p in range(n, len(self.refs)):
            if self.refs[p] > 0:
                to[p] = holes[len(to)]
                self.move(p, to[p], self.page)
                self.refs[to[p]], self.refs[p] = self.refs[p], 0
        self.table = [[to.get(x, x) for x in row] for row in self.table]

    def check(self, cache, what=""):
        """Every byte of the cache's state."""
        assert cache.page_table.cpu().tolist() == self.table, what
        assert cache.seq_lens.cpu().tolist() == self.lens, what
        assert cache.ref_counts.cpu().tolist() == self.refs, what
        for name, pool, mine in (("k", cache.k, self.k), ("v", cache.v, self.v)):
            assert torch.equal(self.bytes(pool.cpu().contiguous()), self.bytes(mine)), f"{what}: {name}"

    def invariants(self):
        held = [0] * len(self.refs)
        for row, n in zip(self.table, self.lens):
            m = self.pages(n)
            assert all(p >= 0 for p in row[:m]) and all(p == -1 for p in row[m:])
            for j, p in enumerate(row[:m]):
                held[p] += 1
        assert held == self.refs
        for row, n in zip(self.table, self.lens):
            if n % self.page:
                assert self.refs[row[n // self.page]] == 1  # a page still being filled is nobody else's
