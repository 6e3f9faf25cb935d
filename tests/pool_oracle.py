"""A page pool in plain Python lists: what fork, extend, free and compact have to leave in the tables,
lengths, counts and caches. Written from the operators' contract (include/pagedkv.h), for tests."""
import torch


class Pool:
    def __init__(self, tables, lens, refs, k, v, block_size):
        self.tables = [list(r) for r in tables.tolist()]
        self.lens, self.refs = lens.tolist(), refs.tolist()
        self.k, self.v = k.clone(), v.clone()  # (L, NB, BS, Hkv, D)
        self.bs = block_size
        self.width = tables.shape[1]

    def pages(self, row):
        return -(-min(self.lens[row], self.width * self.bs) // self.bs)

    def _take(self):
        for b, n in enumerate(self.refs):
            if n == 0:
                self.refs[b] = 1
                return b
        return -2

    def copy(self, src, dst, tokens):
        for s, d, n in zip(src, dst, tokens):
            if 0 <= s < len(self.refs) and 0 <= d < len(self.refs):
                for c in (self.k, self.v):
                    c[:, d, :max(n, 0)] = c[:, s, :max(n, 0)]

    def fork(self, parents, children):
        lens, tables = list(self.lens), [list(r) for r in self.tables]  # parents as they were before the call
        out, seen = [], set()
        for p, c in zip(parents, children):
            if not 0 <= c < len(lens) or lens[c] != 0 or c in seen:
                out.append(-3)
                seen.add(c)
                continue
            seen.add(c)
            n = lens[p] if 0 <= p < len(lens) else 0
            full, tail = divmod(n, self.bs)
            new = self._take() if tail else -1
            out.append(new)
            if new == -2:
                continue
            self.lens[c] = n
            self.tables[c] = [-1] * self.width
            self.tables[c][:full] = tables[p][:full] if full else []
            for b in self.tables[c][:full]:
                self.refs[b] += 1
            if tail:
                self.tables[c][full] = new
                self.copy([tables[p][full]], [new], [tail])
        return out

    def extend(self, rows):
        out, seen = [], set()
        for r in rows:
            slot = -1
            if 0 <= r < len(self.lens) and r not in seen and self.lens[r] < self.width * self.bs:
                page, off = divmod(self.lens[r], self.bs)
                block = self.tables[r][page] if off else self._take()
                if block >= 0:
                    self.tables[r][page] = block
                    self.lens[r] += 1
                    slot = block * self.bs + off
            seen.add(r)
            out.append(slot)
        return out

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.lens):
                for j in range(self.pages(r)):
                    self.refs[self.tables[r][j]] -= 1
                    self.tables[r][j] = -1
                self.lens[r] = 0

    def compact(self):
        live = [b for b, n in enumerate(self.refs) if n > 0]
        to = {b: b for b in live}
        holes = [b for b in range(len(live)) if self.refs[b] == 0]
        for s, d in zip([b for b in live if b >= len(live)], holes):
            to[s], self.refs[d], self.refs[s] = d, self.refs[s], 0
            self.copy([s], [d], [self.bs])
        for r in range(len(self.lens)):
            for j in range(self.pages(r)):
                self.tables[r][j] = to[self.tables[r][j]]
        return [to.get(b, -1) for b in range(len(self.refs))], len(live)

    def same(self, tables, lens, refs, k, v):
        assert tables.cpu().tolist() == self.tables
        assert lens.cpu().tolist() == self.lens
        assert refs.cpu().tolist() == self.refs
        assert torch.equal(k.cpu().view(torch.int16), self.k.view(torch.int16))
        assert torch.equal(v.cpu().view(torch.int16), self.v.view(torch.int16))


def make_pool(seed, lens, block_size, num_blocks, width, layers=2, heads=1, head_dim=8, dtype=torch.bfloat16):
    """Random placement of rows of the given lengths: (tables, lens, refs, k, v) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(num_blocks, generator=g).tolist()
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    refs = torch.zeros(num_blocks, dtype=torch.int32)
    for r, n in enumerate(lens):
        for j in range(-(-n // block_size)):
            b = order.pop()
            tables[r, j] = b
            refs[b] = 1
    kv = torch.randn(2, layers, num_blocks, block_size, heads, head_dim, generator=g).to(dtype)
    return tables, torch.tensor(lens, dtype=torch.int32), refs, kv[0], kv[1]
