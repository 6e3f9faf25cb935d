"""What serving many requests from one set of weights and one paged cache needs beside the attention path: the
requests' low-rank adapters next to the shared projections, and the cache's pages shared, grown, freed and moved.

Every case is a dict of plain values with a "kind":

  linear   one projection of a decode step with every row's own adapter: out = x W^T + s (x A^T) B^T
  add      the adapters of a prefill step, added to a projection's output: out = y + s (x A^T) B^T
  copy     pages copied in every layer's K and V cache, whole or their first tokens
  fork     a step of parallel candidates: sequences forked, their forks grown by one token, the parents freed
  compact  live pages moved to the front of the cache, with the tables that name them

Geometry: the 0.6B model's projections (hidden 1024, FFN 3072, 16 query and 8 kv heads of 128, 28 layers) or one
tensor-parallel rank's share of its kv heads. Which row has which adapter and how long a sequence is come from the
case ("pick" seeds them), tensor values and the placement of pages from the seed.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
D = 128
# projection: (input width, output widths of the projections merged in it)
PROJ = {"qkv": (1024, (2048, 1024, 1024)), "o": (2048, (1024,)), "gate_up": (1024, (3072, 3072)),
        "down": (3072, (1024,))}


def listed():
    return [
        # one chat with one adapter: a step bound by latency and launches
        dict(name="linear_qkv_1", kind="linear", proj="qkv", rows=1, adapters=4, rank=16, pick=1),
        # a ragged decode batch on a few adapters, the widest projection
        dict(name="linear_gate_up_97", kind="linear", proj="gate_up", rows=97, adapters=8, rank=16, pick=2),
        # the full decode batch, almost every request an adapter of its own, large ranks, the longest rows
        dict(name="linear_down_128", kind="linear", proj="down", rows=128, adapters=100, rank=64, pick=3),
        # a mixed step: the live sequences' decode rows and one short chunk
        dict(name="add_o_300", kind="add", proj="o", decodes=120, chunks=1, tokens=300, adapters=24, rank=8, pick=4),
        # the serving run's first step: as many fresh prompts as the 16384-token budget takes
        dict(name="add_qkv_16384", kind="add", proj="qkv", decodes=0, chunks=31, tokens=16384, adapters=8, rank=16,
             pick=5),
        # a ragged step of long prompts, large ranks, the widest projection
        dict(name="add_gate_up_13001", kind="add", proj="gate_up", decodes=0, chunks=9, tokens=13001, adapters=20,
             rank=64, pick=6),
        # one sequence's last page made private before it is written to (37 tokens of it in use)
        dict(name="copy_tail_1", kind="copy", layers=28, kv=8, bs=256, blocks=8, pairs=1, lo=37, hi=37, pick=7),
        # pages of preempted prompts copied whole
        dict(name="copy_pages_16", kind="copy", layers=28, kv=8, bs=256, blocks=40, pairs=16, lo=256, hi=256, pick=8),
        # one request, four candidates
        dict(name="fork_1x4", kind="fork", layers=28, kv=8, bs=256, parents=1, each=4, lo=700, hi=700, free=8, pick=9),
        # a decode batch of sixteen requests with eight candidates each, a rank's share of the heads
        dict(name="fork_16x8", kind="fork", layers=28, kv=2, bs=256, parents=16, each=8, lo=100, hi=2048, free=200,
             pick=10),
        # a few holes closed after one request ended
        dict(name="compact_3", kind="compact", layers=4, kv=8, bs=256, blocks=60, live=40, moves=3, seqs=8, pick=11),
        # a long-running cache with half of its pages live, anywhere
        dict(name="compact_40", kind="compact", layers=28, kv=4, bs=256, blocks=160, live=80, moves=40, seqs=64,
             pick=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "add", "add", "add", "copy", "fork", "fork", "compact"])
    pick = rng.randrange(1 << 20)
    if kind in ("linear", "add"):
        proj, rank, adapters = rng.choice(sorted(PROJ)), 8 * _log_int(rng, 1, 8), _log_int(rng, 1, 100)
        if kind == "linear":
            return dict(kind=kind, proj=proj, rows=_log_int(rng, 1, 128), adapters=adapters, rank=rank, pick=pick)
        # a step's prompts stay within what the largest step holds
        tokens = _log_int(rng, 2, 13001)
        chunks = _log_int(rng, 1, min(40, tokens // 2))
        decodes = rng.choice([0, rng.randint(0, min(128, tokens - 2 * chunks))])
        return dict(kind=kind, proj=proj, decodes=decodes, chunks=chunks, tokens=tokens, adapters=adapters, rank=rank,
                    pick=pick)
    layers, kv, bs = rng.randint(1, 28), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    if kind == "copy":
        pairs = _log_int(rng, 1, 16)
        lo, hi = sorted((rng.randint(1, bs), rng.randint(1, bs)))
        return dict(kind=kind, layers=layers, kv=kv, bs=bs, blocks=2 * pairs + rng.randint(0, 8), pairs=pairs, lo=lo,
                    hi=hi, pick=pick)
    if kind == "fork":
        lo, hi = sorted((_log_int(rng, 1, 2048), _log_int(rng, 64, 2048)))
        parents, each = _log_int(rng, 1, 16), rng.randint(1, 8)
        return dict(kind=kind, layers=layers, kv=min(kv, 2), bs=bs, parents=parents, each=each, lo=lo, hi=hi,
                    free=2 * parents * each + rng.randint(0, 40), pick=pick)
    blocks = _log_int(rng, 8, 160)
    live = rng.randint(2, blocks - 2)
    return dict(kind=kind, layers=layers, kv=min(kv, 4), bs=bs, blocks=blocks, live=live,
                moves=rng.randint(0, min(live, blocks - live, 40)), seqs=_log_int(rng, 1, 64), pick=pick)


# ---------------------------------------------------------------- shapes of a case ---
def _segments(case):
    """(first row, end row, adapter) of a step's sequences in batch order; adapter -1: the base model."""
    r = random.Random(case["pick"])
    if case["kind"] == "linear":
        lens = [1] * case["rows"]
    else:
        rest = case["tokens"] - case["decodes"] - 2 * case["chunks"]  # a chunk has two tokens or more
        cuts = sorted(r.randint(0, rest) for _ in range(case["chunks"] - 1))
        lens = [1] * case["decodes"] + [2 + b - a for a, b in zip([0] + cuts, cuts + [rest])]
    out, at = [], 0
    for n in lens:
        out.append((at, at + n, -1 if r.random() < 0.1 and len(lens) > 1 else r.randrange(case["adapters"])))
        at += n
    return out


def _copy_tokens(case):
    r = random.Random(case["pick"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["pairs"])]


def _fork_lens(case):
    r = random.Random(case["pick"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["parents"])]


def work(case):
    """Bytes: inputs read once, outputs written once (the adapters that a row has; the pages' tokens that are
    copied, read and written; tables, lengths and counts of the sequences). Flops: multiplies and adds."""
    kind = case["kind"]
    if kind in ("linear", "add"):
        k, widths = PROJ[case["proj"]]
        n, r, s = sum(widths), case["rank"], len(widths)
        seg = _segments(case)
        m = seg[-1][1]
        with_adapter = sum(b - a for a, b, i in seg if i >= 0)
        used = len({i for _, _, i in seg if i >= 0})
        low = s * r * k + n * r
        base = n * k if kind == "linear" else m * n
        return {"bytes": 2 * (base + m * k + m * n + used * low) + 4 * m,
                "flops": 2 * with_adapter * low + (2 * m * n * k if kind == "linear" else m * n)}
    token = 2 * 2 * case["layers"] * case["kv"] * D  # K and V of one token in every layer
    if kind == "copy":
        return {"bytes": 2 * token * sum(_copy_tokens(case)) + 12 * case["pairs"], "flops": 0}
    if kind == "fork":
        lens, bs, each = _fork_lens(case), case["bs"], case["each"]
        return {"bytes": 2 * token * each * sum(x % bs for x in lens) + 8 * (each + 1) * sum(-(-x // bs) for x in lens),
                "flops": 0}
    return {"bytes": 2 * token * case["bs"] * case["moves"] + 16 * case["blocks"], "flops": 0}


# ---------------------------------------------------------------- inputs ---
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _caches(case, blocks, g):
    # K and V as the runner keeps them: (layers, blocks, block size, kv heads, 128), two halves of one tensor
    kv = torch.empty(2, case["layers"], blocks, case["bs"], case["kv"], D, dtype=torch.bfloat16, device=DEV)
    kv.normal_(generator=g)
    return kv[0], kv[1]


def prepare(case, seed):
    kind, g, rng = case["kind"], _gen(seed), random.Random(seed)
    st = {"case": case}
    if own:
        root = os.path.join(os.getcwd(), "nano-vllm-diy_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        import pagedkv
        st["lib"] = pagedkv
    if kind in ("linear", "add"):
        k, widths = PROJ[case["proj"]]
        n, r, na = sum(widths), case["rank"], case["adapters"]
        seg = _segments(case)
        m = seg[-1][1]
        st.update(x=_randn(g, m, k), a=_randn(g, na, len(widths) * r, k, std=k ** -0.5),
                  b=_randn(g, na, n, r, std=0.05), ids=_i32([i for a, b, i in seg for _ in range(b - a)]), widths=widths,
                  scales=torch.tensor([rng.choice([0.5, 1.0, 2.0]) for _ in range(na)], device=DEV))
        if kind == "linear":
            st["w"] = _randn(g, n, k, std=0.02)
        else:
            st["y"] = _randn(g, m, n)
            # the plain form's plan: the rows of every adapter in use
            st["rows"] = [(i, torch.tensor([x for a, b, j in seg if j == i for x in range(a, b)], device=DEV))
                          for i in sorted({j for _, _, j in seg if j >= 0})]
        return st
    if kind == "copy":
        st["k"], st["v"] = _caches(case, case["blocks"], g)
        order = rng.sample(range(case["blocks"]), 2 * case["pairs"])
        st.update(src=_i32(order[:case["pairs"]]), dst=_i32(order[case["pairs"]:]), tokens=_i32(_copy_tokens(case)))
        return st
    if kind == "fork":
        lens, bs, each = _fork_lens(case), case["bs"], case["each"]
        used = sum(-(-x // bs) for x in lens)
        nb, rows = used + case["free"], len(lens) * (1 + each)
        width = -(-case["hi"] // bs) + 1
        st["k"], st["v"] = _caches(case, nb, g)
        ids = rng.sample(range(nb), used)
        place = rng.sample(range(rows), rows)  # which row of the tables a sequence has
        tables = torch.full((rows, width), -1, dtype=torch.int32)
        refs, lrow = torch.zeros(nb, dtype=torch.int32), [0] * rows
        for i, x in enumerate(lens):
            mine = [ids.pop() for _ in range(-(-x // bs))]
            tables[place[i], :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            refs[mine] = 1
            lrow[place[i]] = x
        parents = [i for i in range(len(lens)) for _ in range(each)]
        st.update(tables=tables.to(DEV), lens=_i32(lrow), refs=refs.to(DEV), parents=_i32([place[i] for i in parents]),
                  children=_i32(place[len(lens):]), done=_i32(place[:len(lens)]), part=[lens[i] % bs for i in parents])
        return st
    # compact: `moves` of the live pages lie behind the first `live` pages
    nb, live, moves, seqs = case["blocks"], case["live"], case["moves"], case["seqs"]
    st["k"], st["v"] = _caches(case, nb, g)
    ids = rng.sample(range(live), live - moves) + rng.sample(range(live, nb), moves)
    rng.shuffle(ids)
    # the pages in the tables of the sequences, every fourth of them in a second sequence's too
    width = -(-live // seqs) * 2 + 1
    rows = [[] for _ in range(seqs)]
    refs = torch.zeros(nb, dtype=torch.int32)
    for j, b in enumerate(ids):
        rows[j % seqs].append(b)
        refs[b] += 1
        if j % 4 == 0 and seqs > 1:
            rows[(j + 1) % seqs].append(b)
            refs[b] += 1
    tables = torch.full((seqs, width), -1, dtype=torch.int32)
    for i, row in enumerate(rows):
        tables[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
    lens = [len(row) * case["bs"] - (rng.randrange(case["bs"]) if row else 0) for row in rows]
    st.update(tables=tables.to(DEV), refs=refs.to(DEV), lens=_i32(lens))
    return st


# ---------------------------------------------------------------- one pass ---
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    kind, lib, bs = st["case"]["kind"], st["lib"], st["case"].get("bs")
    if kind == "linear":
        return lib.lora_linear(st["x"], st["w"], st["a"], st["b"], st["ids"], st["scales"], slices=st["widths"])
    if kind == "add":
        return lib.lora_add(st["y"], st["x"], st["a"], st["b"], st["ids"], st["scales"], slices=st["widths"])
    if kind == "copy":
        lib.copy_blocks(st["k"], st["v"], st["src"], st["dst"], st["tokens"])
        return st["k"], st["v"]
    tables, lens, refs = st["tables"].clone(), st["lens"].clone(), st["refs"].clone()
    if kind == "fork":
        new = lib.fork_sequences(st["k"], st["v"], tables, lens, refs, st["parents"], st["children"])
        slots = lib.extend_sequences(tables, lens, refs, bs, st["children"])
        lib.free_sequences(tables, lens, refs, bs, st["done"])
        return st["k"], st["v"], tables, lens, refs, new, slots
    block_map, num_live = lib.compact_blocks(st["k"], st["v"], tables, lens, refs)
    return st["k"], st["v"], tables, refs, block_map, num_live


def _lowest_free(refs, need):
    """For every true entry of need, in order, the lowest block that nobody holds; -1 where false, -2 where none is
    left."""
    order = torch.argsort((refs > 0).to(torch.int8), stable=True)  # the free blocks first, each kind ascending
    nth = torch.cumsum(need, 0) - 1
    got = order[nth.clamp(0, refs.numel() - 1)]
    got = torch.where(nth < (refs == 0).sum(), got, torch.full_like(got, -2))
    return torch.where(need, got, torch.full_like(got, -1)).to(torch.int32)


def _count(refs, blocks, live, step):
    """refs[blocks] += step where live."""
    refs.index_add_(0, blocks.clamp(min=0).reshape(-1).long(), (live.to(torch.int32) * step).reshape(-1))


def _run_plain(st):
    case = st["case"]
    kind, bs = case["kind"], case.get("bs")
    if kind == "linear":
        # every row with its own adapter's matrices; rows without one multiply by a scale of zero
        x, ids = st["x"].float(), st["ids"].long()
        pick, r = ids.clamp(min=0), case["rank"]
        t = torch.bmm(st["a"][pick].float(), x.unsqueeze(2)).squeeze(2)
        t = t * torch.where(ids >= 0, st["scales"][pick], torch.zeros_like(st["scales"][pick])).unsqueeze(1)
        delta, at = [], 0
        for q, n in enumerate(st["widths"]):
            delta.append(torch.bmm(st["b"][pick, at:at + n].float(), t[:, q * r:(q + 1) * r].unsqueeze(2)).squeeze(2))
            at += n
        return (x @ st["w"].float().t() + torch.cat(delta, 1)).to(torch.bfloat16)
    if kind == "add":
        # adapter by adapter, whose rows the program knows
        out, r = st["y"].clone(), case["rank"]
        for i, rows in st["rows"]:
            t = (st["x"][rows].float() @ st["a"][i].float().t()) * st["scales"][i]
            b, at, parts = st["b"][i].float(), 0, []
            for q, n in enumerate(st["widths"]):
                parts.append(t[:, q * r:(q + 1) * r] @ b[at:at + n].t())
                at += n
            out[rows] = (st["y"][rows].float() + torch.cat(parts, 1)).to(torch.bfloat16)
        return out
    k, v = st["k"], st["v"]
    if kind == "copy":
        src, dst = st["src"].long(), st["dst"].long()
        keep = (torch.arange(bs, device=DEV) < st["tokens"].unsqueeze(1))[None, :, :, None, None]
        for c in (k, v):
            c[:, dst] = torch.where(keep, c[:, src], c[:, dst])
        return k, v
    tables, lens, refs = st["tables"].clone(), st["lens"].clone(), st["refs"].clone()
    cols = torch.arange(tables.shape[1], dtype=torch.int32, device=DEV)
    if kind == "fork":
        parents, children, done = st["parents"].long(), st["children"].long(), st["done"].long()
        # fork
        length = lens[parents]
        full, part = length // bs, length % bs
        new = _lowest_free(refs, part > 0)
        row = tables[parents]
        shared = cols < full.unsqueeze(1)
        _count(refs, row, shared, 1)
        _count(refs, new, new >= 0, 1)
        last = row.gather(1, full.unsqueeze(1).long().clamp(max=row.shape[1] - 1)).squeeze(1)
        row = torch.where(shared, row, torch.where(cols == full.unsqueeze(1), new.clamp(min=-1).unsqueeze(1),
                                                   torch.full_like(row, -1)))
        tables[children] = row
        lens[children] = length
        some = [i for i, x in enumerate(st["part"]) if x]  # the forks with a page of their own
        if some:
            src, dst = last[some].long(), new[some].long()
            keep = (torch.arange(bs, device=DEV) < part[some].unsqueeze(1))[None, :, :, None, None]
            for c in (k, v):
                c[:, dst] = torch.where(keep, c[:, src], c[:, dst])
        # grow every fork by a token
        length = lens[children]
        at = (length // bs).unsqueeze(1)
        grown = _lowest_free(refs, length % bs == 0)
        _count(refs, grown, grown >= 0, 1)
        row = tables[children]
        row = torch.where((cols == at) & (length % bs == 0).unsqueeze(1), grown.unsqueeze(1), row)
        tables[children] = row
        slots = row.gather(1, at.long()).squeeze(1) * bs + length % bs
        lens[children] = length + 1
        # free the parents
        row = tables[done]
        _count(refs, row, row >= 0, -1)
        tables[done] = torch.full_like(row, -1)
        lens[done] = 0
        return k, v, tables, lens, refs, new, slots
    ids = torch.arange(refs.numel(), dtype=torch.int32, device=DEV)
    live = refs > 0
    num_live = live.sum(0, keepdim=True).to(torch.int32)
    src = torch.argsort((live & (ids >= num_live)).to(torch.int8), stable=True, descending=True)[:case["moves"]]
    dst = torch.argsort((~live & (ids < num_live)).to(torch.int8), stable=True, descending=True)[:case["moves"]]
    block_map = torch.where(live, ids, torch.full_like(ids, -1))
    block_map[src] = dst.to(torch.int32)
    refs[dst] = refs[src]
    refs[src] = 0
    tables = torch.where(tables >= 0, block_map[tables.clamp(min=0).long()], tables)
    for c in (k, v):
        c[:, dst] = c[:, src]
    return k, v, tables, refs, block_map, num_live


# ---------------------------------------------------------------- from the definition, in 64 bits ---
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("linear", "add"):
        x = st["x"].double()
        out = x @ st["w"].double().t() if kind == "linear" else st["y"].double()
        r, ids = case["rank"], st["ids"].cpu().tolist()
        for i in sorted(set(ids)):
            if i < 0:
                continue
            rows = torch.tensor([m for m, j in enumerate(ids) if j == i], device=DEV)
            t = x[rows] @ st["a"][i].double().t()
            at = 0
            for q, n in enumerate(st["widths"]):
                b = st["b"][i, at:at + n].double()
                out[rows, at:at + n] += st["scales"][i].double() * (t[:, q * r:(q + 1) * r] @ b.t())
                at += n
        return out
    k, v, bs = st["k"], st["v"], case["bs"]
    if kind == "copy":
        for s, d, n in zip(st["src"].tolist(), st["dst"].tolist(), st["tokens"].tolist()):
            k[:, d, :n] = k[:, s, :n]
            v[:, d, :n] = v[:, s, :n]
        return k, v
    tables, lens, refs = st["tables"].tolist(), st["lens"].tolist(), st["refs"].tolist()
    if kind == "fork":
        new, slots, children = [], [], st["children"].tolist()
        free = [b for b, n in enumerate(refs) if n == 0]
        for p, c in zip(st["parents"].tolist(), children):
            full, part = divmod(lens[p], bs)
            tables[c][:full] = tables[p][:full]
            for b in tables[p][:full]:
                refs[b] += 1
            new.append(free.pop(0) if part else -1)
            if part:
                tables[c][full] = new[-1]
                refs[new[-1]] = 1
                for cache in (k, v):
                    cache[:, new[-1], :part] = cache[:, tables[p][full], :part]
            lens[c] = lens[p]
        for c in children:
            j, off = divmod(lens[c], bs)
            if off == 0:
                tables[c][j] = free.pop(0)
                refs[tables[c][j]] = 1
            slots.append(tables[c][j] * bs + off)
            lens[c] += 1
        for p in st["done"].tolist():
            for j, b in enumerate(tables[p]):
                if b >= 0:
                    refs[b] -= 1
                tables[p][j] = -1
            lens[p] = 0
        return k, v, _i32(tables), _i32(lens), _i32(refs), _i32(new), _i32(slots)
    live = [b for b, n in enumerate(refs) if n > 0]
    holes = [b for b in range(len(live)) if refs[b] == 0]
    to = {b: b for b in live}
    for s, d in zip([b for b in live if b >= len(live)], holes):
        to[s], refs[d], refs[s] = d, refs[s], 0
        k[:, d] = k[:, s]
        v[:, d] = v[:, s]
    tables = [[to[b] if b >= 0 else b for b in row] for row in tables]
    return k, v, _i32(tables), _i32(refs), _i32([to.get(b, -1) for b in range(len(refs))]), _i32([len(live)])
