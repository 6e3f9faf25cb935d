"""What a paged K/V cache held in 4 bits needs: new tokens appended to it (q/k norm and rotation on the way, or rows
as given) and attention over it, for single tokens, a few tokens of every sequence, chunks of prompts and mixtures.

A token's row of such a cache (uint8) is, for Hkv kv heads of 128: Hkv x 64 bytes of values, two to a byte (the lower
dimension in the low four bits), then Hkv x 4 scale bytes, one per 32 dimensions, then zero to 15 bytes up to a
multiple of 16 that nothing reads or writes. A value is sign, two bits of exponent and one of mantissa (0, 0.5, 1,
1.5, 2, 3, 4, 6 and their negatives) times 2^(scale byte - 127). Of 32 values with the largest magnitude a, the scale
is the smallest power of two s with a <= 7 s (within 2^-126 .. 2^125); values are divided by it and rounded to
nearest, ties to even, at most 6.

Every case is a dict of plain values with a "kind":

  append   qk_norm_rope_store_fp4: one step's tokens from the fused qkv projection, q returned, k and v rows stored;
           the stored rows are returned as values too (a fresh prompt's attention takes them)
  store    store_kvcache_fp4, rows as given, and gather_kv_fp4, the sequences' rows read back as values
  attend   varlen_attention_fp4: "ones" sequences of one query row, "chunks" sequences of several rows behind a prefix

Geometry: the 0.6B model's heads (16 query heads, 8 kv heads of 128), one tensor-parallel rank's share of them, or
another GQA group. Lengths and which tokens are padding come from the case ("pick" seeds them), tensor values and the
placement of pages from the seed.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
D = 128
EPS = 1e-6
MAX_POSITION = 40960


def listed():
    return [
        # one chat's decode step: latency
        dict(name="append_1", kind="append", heads=16, kv=8, bs=256, seqs=1, lo=1, hi=1, pad=0, pick=1),
        # a decode step of 97 sequences in a graph captured for 112
        dict(name="append_97", kind="append", heads=16, kv=8, bs=256, seqs=97, lo=1, hi=1, pad=15, pick=2),
        # the serving run's first step: fresh prompts up to the 16384-token budget
        dict(name="append_16384", kind="append", heads=16, kv=8, bs=256, seqs=32, lo=512, hi=512, pad=0, pick=3),
        # a mixed step at a rank's share of the heads, stored by the attention layer
        dict(name="store_301", kind="store", heads=8, kv=4, bs=64, seqs=7, lo=1, hi=85, pad=3, pick=4),
        # long prompts' rows, stored and read back
        dict(name="store_8191", kind="store", heads=16, kv=8, bs=256, seqs=5, lo=300, hi=3000, pad=0, pick=5),
        # a small decode batch
        dict(name="attend_8", kind="attend", heads=16, kv=8, bs=256, ones=8, one_lo=256, one_hi=2048, chunks=0,
             rows_lo=0, rows_hi=0, pre_lo=0, pre_hi=0, pick=6),
        # the serving run's decode step
        dict(name="attend_128", kind="attend", heads=16, kv=8, bs=256, ones=128, one_lo=100, one_hi=2048, chunks=0,
             rows_lo=0, rows_hi=0, pre_lo=0, pre_hi=0, pick=7),
        # the large decode batch of long contexts
        dict(name="attend_256", kind="attend", heads=16, kv=8, bs=256, ones=256, one_lo=1024, one_hi=8192, chunks=0,
             rows_lo=0, rows_hi=0, pre_lo=0, pre_hi=0, pick=8),
        # one very long context on one kv head, eight query heads on it
        dict(name="attend_long_1", kind="attend", heads=8, kv=1, bs=256, ones=1, one_lo=100003, one_hi=100003, chunks=0,
             rows_lo=0, rows_hi=0, pre_lo=0, pre_hi=0, pick=9),
        # drafted tokens checked: a few rows of every sequence, a rank's share of the heads
        dict(name="attend_verify_48", kind="attend", heads=8, kv=4, bs=128, ones=0, one_lo=0, one_hi=0, chunks=48,
             rows_lo=2, rows_hi=8, pre_lo=300, pre_hi=4000, pick=10),
        # a mixed step: decode rows and chunks of 512 tokens of new prompts
        dict(name="attend_mixed_124", kind="attend", heads=16, kv=8, bs=256, ones=120, one_lo=100, one_hi=2048, chunks=4,
             rows_lo=300, rows_hi=512, pre_lo=0, pre_hi=2048, pick=11),
        # chunks of long prompts behind what is cached of them
        dict(name="attend_chunks_16", kind="attend", heads=16, kv=8, bs=256, ones=0, one_lo=0, one_hi=0, chunks=16,
             rows_lo=1024, rows_hi=1024, pre_lo=4096, pre_hi=4096, pick=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _span(rng, lo, hi):
    return sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))


def draw(rng):
    kind = rng.choice(["append", "append", "store", "attend", "attend", "attend", "attend", "attend"])
    kv, group, bs = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    c = dict(kind=kind, heads=kv * min(group, 16 // kv), kv=kv, bs=bs)
    pick = rng.randrange(1 << 20)
    if kind != "attend":
        seqs = _log_int(rng, 1, 128)
        lo, hi = rng.choice([(1, 1), _span(rng, 1, 16384 // seqs)])
        return dict(c, seqs=seqs, lo=lo, hi=hi, pad=rng.choice([0, rng.randint(1, 16)]), pick=pick)
    what = rng.choice(["ones", "ones", "few", "chunks", "mixed"])
    ones = chunks = one_lo = one_hi = rows_lo = rows_hi = pre_lo = pre_hi = 0
    if what in ("ones", "mixed"):
        ones = _log_int(rng, 1, 256 if what == "ones" else 120)
        one_lo, one_hi = _span(rng, 1, min(8192, 1 << 20) if ones > 4 else 100000)
    if what == "few":
        chunks = _log_int(rng, 1, 64)
        rows_lo, rows_hi = sorted((rng.randint(2, 16), rng.randint(2, 16)))
        pre_lo, pre_hi = _span(rng, 1, 4000)
    elif what in ("chunks", "mixed"):
        chunks = _log_int(rng, 1, 16 if what == "chunks" else 4)
        rows_lo, rows_hi = _span(rng, 2, 1024 if what == "chunks" else 512)
        pre_lo, pre_hi = rng.choice([(0, 0), _span(rng, 1, 4096)])
    return dict(c, ones=ones, one_lo=one_lo, one_hi=one_hi, chunks=chunks, rows_lo=rows_lo, rows_hi=rows_hi,
                pre_lo=pre_lo, pre_hi=pre_hi, pick=pick)


# ---------------------------------------------------------------- shapes of a case ---
def _row_bytes(kv):
    return (68 * kv + 15) // 16 * 16


def _new_lens(case):
    """append and store: tokens of every sequence"""
    r = random.Random(case["pick"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _attend_lens(case):
    """(query rows, keys) of every sequence, the single rows first"""
    r = random.Random(case["pick"])
    out = [(1, r.randint(case["one_lo"], case["one_hi"])) for _ in range(case["ones"])]
    for _ in range(case["chunks"]):
        rows = r.randint(case["rows_lo"], case["rows_hi"])
        out.append((rows, rows + r.randint(case["pre_lo"], case["pre_hi"])))
    return out


def work(case):
    """Bytes: inputs read once, outputs written once (a key's 4-bit row once for all the rows that see it).
    Flops: the two products over the keys that a row sees, the roundings of an append not counted."""
    h, kv = case["heads"], case["kv"]
    if case["kind"] == "attend":
        lens = _attend_lens(case)
        rows, keys = sum(q for q, _ in lens), sum(k for _, k in lens)
        seen = sum(q * k - q * (q - 1) // 2 for q, k in lens)
        return {"bytes": 2 * 68 * kv * keys + 2 * 2 * D * h * rows + 8 * len(lens), "flops": 4 * D * h * seen}
    n = sum(_new_lens(case))
    new = 2 * (2 * D + 68) * kv * n  # K and V rows read, and written in 4 bits
    if case["kind"] == "append":  # q read and written, the stored rows' values written, table row, position, slot
        return {"bytes": new + 2 * 2 * D * h * n + 2 * 2 * D * kv * n + (4 * D + 12) * n, "flops": 8 * D * (h + kv) * n}
    return {"bytes": new + 2 * (2 * D + 68) * kv * n + 4 * n, "flops": 2 * D * kv * n}  # and read back


# ---------------------------------------------------------------- inputs ---
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prefix(values):
    out = [0]
    for x in values:
        out.append(out[-1] + x)
    return out


def _tables(lens, bs, rng):
    """Block tables of sequences of these lengths over a pool with a few blocks that nobody has, and its size."""
    need = [-(-x // bs) for x in lens]
    nb = sum(need) + 2
    ids = rng.sample(range(nb), sum(need))
    tables = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        tables[i, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return tables, nb


def prepare(case, seed):
    kind, g, rng = case["kind"], _gen(seed), random.Random(seed)
    h, kv, bs, row = case["heads"], case["kv"], case["bs"], _row_bytes(case["kv"])
    st = {"case": case}
    if own:
        root = os.path.join(os.getcwd(), "nano-vllm-diy_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        import pagedkv
        st["lib"] = pagedkv
    if kind != "attend":
        lens, pad = _new_lens(case), case["pad"]
        n = sum(lens)
        tables, nb = _tables(lens, bs, rng)
        slots = [int(tables[i, t // bs]) * bs + t % bs for i, x in enumerate(lens) for t in range(x)]
        qkv = _randn(g, n + pad, (h + 2 * kv) * D)
        st.update(slots=_i32(slots + [-1] * pad), n=n, rows=torch.tensor(slots, device=DEV), tables=tables.to(DEV),
                  cu=_i32(_prefix(lens)), max_k=max(lens))
        for name in ("k", "v"):
            st[name] = torch.randint(0, 256, (nb, bs, row), generator=g, device=DEV, dtype=torch.uint8)
        if kind == "store":
            st.update(key=_randn(g, n + pad, kv, D), value=qkv[:, (h + kv) * D:].view(-1, kv, D))
            return st
        freq = 1.0 / 1000000.0 ** (torch.arange(0, D, 2, device=DEV).double() / D)
        angle = torch.outer(torch.arange(MAX_POSITION, device=DEV).double(), freq)
        positions = [p for x in lens for p in (range(x) if x > 1 else [rng.randrange(MAX_POSITION)])]
        st.update(qkv=qkv, positions=torch.tensor(positions + [0] * pad, device=DEV),
                  table=torch.cat((angle.cos(), angle.sin()), 1).float().contiguous(),
                  qw=_randn(g, D, std=0.1) + 1, kw=_randn(g, D, std=0.1) + 1)
        return st
    lens = _attend_lens(case)
    tables, nb = _tables([k for _, k in lens], bs, rng)
    n = sum(q for q, _ in lens)
    # keys with a few dimensions far larger than the others, as rotated keys have them
    wide = torch.ones(kv, D, device=DEV)
    wide[:, torch.tensor(rng.sample(range(D), 6), device=DEV)] = 6.0
    for name, scale in (("k", wide), ("v", 1.0)):
        x = torch.empty(nb, bs, kv, D, device=DEV).normal_(generator=g)
        st[name] = _quantise((x * scale).to(torch.bfloat16), row)
        del x
    st.update(q=_randn(g, n, h, D), tables=tables.to(DEV), cu_q=_i32(_prefix([q for q, _ in lens])),
              cu_k=_i32(_prefix([k for _, k in lens])), max_q=max(q for q, _ in lens), max_k=max(k for _, k in lens))
    # the plain form's plan: sequences of one row, and of several, padded to their longest
    st["groups"], first = [], _prefix([q for q, _ in lens])
    for which in (range(case["ones"]), range(case["ones"], len(lens))):
        if len(which):
            rows, keys = max(lens[i][0] for i in which), max(lens[i][1] for i in which)
            st["groups"].append(dict(
                rows=torch.tensor([[first[i] + min(j, lens[i][0] - 1) for j in range(rows)] for i in which], device=DEV),
                real=torch.tensor([[j < lens[i][0] for j in range(rows)] for i in which], device=DEV),
                pages=st["tables"][which.start:which.stop, :-(-keys // bs)].clamp(min=0).long(),
                lq=torch.tensor([lens[i][0] for i in which], device=DEV),
                lk=torch.tensor([lens[i][1] for i in which], device=DEV)))
    return st


# ---------------------------------------------------------------- the plain form ---
def _quantise(x, row):
    """(..., Hkv, 128) values as rows of `row` bytes (the last ones zero)."""
    lead, kv = x.shape[:-2], x.shape[-2]
    x = x.float().view(*lead, kv, 4, 32)
    bits = x.abs().amax(-1).view(torch.int32)
    scale = ((bits >> 23) - 2 + ((bits & 0x7fffff) > 0x600000).int()).clamp(1, 252)
    a = x.abs() * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)
    code = (torch.signbit(x).to(torch.uint8) * 8 + (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5))
    code = code.view(*lead, kv * 64, 2)
    parts = [code[..., 0] + code[..., 1] * 16, scale.to(torch.uint8).view(*lead, kv * 4)]
    if row > 68 * kv:
        parts.append(torch.zeros(*lead, row - 68 * kv, dtype=torch.uint8, device=x.device))
    return torch.cat(parts, -1)


def _values(rows, kv):
    """The fp32 values (..., Hkv, 128) of rows of bytes."""
    lead = rows.shape[:-1]
    code = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=rows.device)
    pairs = torch.stack((code.repeat(16), code.repeat_interleave(16)), 1)  # of every byte: low bits, high bits
    x = pairs[rows[..., :64 * kv].int()].view(*lead, kv, 4, 32)
    scale = (rows[..., 64 * kv:68 * kv].int() << 23).view(torch.float32).view(*lead, kv, 4, 1)
    return (x * scale).view(*lead, kv, D)


def _put(cache, rows, x):
    """Values into token rows of a cache, its last bytes left as they are."""
    kv = x.shape[-2]
    cache.view(-1, cache.shape[-1])[rows, :68 * kv] = _quantise(x, _row_bytes(kv))[:, :68 * kv]


def _norm_rope(x, weight, positions, table):
    """RMSNorm and rotation of (N, heads, 128) bf16, rounded to bf16 after each; the root in 64 bits, since a value
    next to a rounding border decides which of two 4-bit values a key gets."""
    root = (x.double().square().mean(-1, keepdim=True) + torch.tensor(EPS).double()).sqrt().reciprocal().float()
    x = (weight.float() * (x.float() * root)).to(torch.bfloat16).float()
    cos, sin = table[positions].unsqueeze(1).split(D // 2, -1)
    a, b = x.split(D // 2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).to(torch.bfloat16)


def _attend(st, grp):
    """(rows, heads, 128) outputs of one group's padded query rows."""
    h, kv = st["case"]["heads"], st["case"]["kv"]
    q = st["q"][grp["rows"]].float()
    s, r = q.shape[:2]
    q = q.view(s, r, kv, h // kv, D).permute(0, 2, 1, 3, 4).reshape(s, kv, -1, D)
    k = _values(st["k"][grp["pages"]].flatten(1, 2), kv).permute(0, 2, 3, 1).contiguous()
    p = torch.matmul(q, k) * D ** -0.5
    del k
    last = grp["lk"].unsqueeze(1) - grp["lq"].unsqueeze(1) + torch.arange(r, device=DEV)  # a row's last key
    last = torch.minimum(last, grp["lk"].unsqueeze(1) - 1).repeat_interleave(h // kv, 1)
    hidden = torch.arange(p.shape[-1], device=DEV) > last.unsqueeze(-1)
    p = p.masked_fill_(hidden.unsqueeze(1), float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    # keys behind a sequence's end may be anything: their weights are zero, their values taken as zero
    v = _values(st["v"][grp["pages"]].flatten(1, 2), kv)
    v = v.masked_fill_((torch.arange(v.shape[1], device=DEV) >= grp["lk"].unsqueeze(1))[:, :, None, None], 0)
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()) / total
    return o.view(s, kv, r, h // kv, D).permute(0, 2, 1, 3, 4).reshape(s, r, h, D)


def _run_plain(st):
    case = st["case"]
    h, kv, n = case["heads"], case["kv"], st.get("n")
    if case["kind"] == "append":
        qkv = st["qkv"].view(-1, h + 2 * kv, D)
        q = _norm_rope(qkv[:, :h], st["qw"], st["positions"], st["table"])
        k = _norm_rope(qkv[:, h:h + kv], st["kw"], st["positions"], st["table"])
        stored = [_values(_quantise(x, _row_bytes(kv)), kv).to(torch.bfloat16) for x in (k, qkv[:, h + kv:])]
        _put(st["k"], st["rows"], k[:n])
        _put(st["v"], st["rows"], qkv[:n, h + kv:])
        return q, stored[0], stored[1], st["k"], st["v"]
    if case["kind"] == "store":
        _put(st["k"], st["rows"], st["key"][:n])
        _put(st["v"], st["rows"], st["value"][:n])
        return [_values(c.view(-1, c.shape[-1])[st["rows"]], kv).to(torch.bfloat16) for c in (st["k"], st["v"])]
    out = torch.empty_like(st["q"])
    outs = [(grp["rows"][grp["real"]], _attend(st, grp)[grp["real"]]) for grp in st["groups"]]
    out[torch.cat([i for i, _ in outs])] = torch.cat([o for _, o in outs]).to(torch.bfloat16)
    return out


# ---------------------------------------------------------------- one pass ---
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    case, lib = st["case"], st["lib"]
    if case["kind"] == "append":
        q, k, v = lib.qk_norm_rope_store_fp4(st["qkv"], st["positions"], st["table"], case["heads"], case["kv"], D,
                                             st["qw"], st["kw"], EPS, st["k"], st["v"], st["slots"], return_kv=True)
        return q, k, v, st["k"], st["v"]
    if case["kind"] == "store":
        lib.store_kvcache_fp4(st["key"], st["value"], st["k"], st["v"], st["slots"])
        return [lib.gather_kv_fp4(c, st["tables"], st["cu"], st["max_k"], st["n"]) for c in (st["k"], st["v"])]
    return lib.varlen_attention_fp4(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["max_q"], st["max_k"],
                                    st["tables"])


# ---------------------------------------------------------------- from the definition, in 64 bits ---
def exact(case, seed):
    """None for an append's keys, whose 4-bit values its roundings to bf16 decide, and for whole caches (bytes)."""
    st = prepare(case, seed)
    h, kv, bs = case["heads"], case["kv"], case["bs"]

    def held(x):  # values as the cache holds them
        x = x.double().view(-1, kv, 4, 32)
        top = x.abs().amax(-1, keepdim=True)
        s = torch.pow(2.0, torch.ceil(torch.log2(top / 7)).clamp(-126, 125))
        step = torch.where(x.abs() < 2 * s, s / 2, torch.where(x.abs() < 4 * s, s, 2 * s))
        return torch.minimum(torch.maximum(torch.round(x / step) * step, -6 * s), 6 * s).view(-1, kv, D)

    if case["kind"] == "store":
        return [held(st[name][:st["n"]]) for name in ("key", "value")]
    if case["kind"] == "append":
        x = st["qkv"].double().view(-1, h + 2 * kv, D)[:, :h]
        x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * st["qw"].double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                           torch.atan2(st["table"][:, D // 2:].double(), st["table"][:, :D // 2].double()))
        z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn[st["positions"]].unsqueeze(1)
        return torch.cat((z.real, z.imag), -1), None, held(st["qkv"][:, (h + kv) * D:]), None, None
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    dims = torch.arange(D, device=DEV)

    def read(cache, row):
        x = cache[row]  # (blocks, bs, row bytes)
        x = x.view(-1, x.shape[-1])
        heads = torch.arange(kv, device=DEV).unsqueeze(1)
        nib = (x[:, heads * 64 + dims // 2].long() >> (dims % 2 * 4)) & 15
        exp, man = nib >> 1 & 3, (nib & 1).double()
        mag = torch.where(exp == 0, man / 2, (1 + man / 2) * torch.pow(2.0, (exp - 1).double()))
        power = torch.pow(2.0, x[:, kv * 64 + heads * 4 + dims // 32].double() - 127)
        return torch.where(nib >= 8, -mag, mag) * power

    at = 0
    for i, (lq, lk) in enumerate(_attend_lens(case)):
        row = st["tables"][i, :-(-lk // bs)].long()
        k, v = read(st["k"], row)[:lk], read(st["v"], row)[:lk]
        for j in range(kv):
            q = st["q"][at:at + lq, j * (h // kv):(j + 1) * (h // kv)].double().transpose(0, 1)
            s = (q @ k[:, j].t()) / D ** 0.5
            seen = torch.ones(lq, lk, dtype=torch.bool, device=DEV).tril(lk - lq)
            out[at:at + lq, j * (h // kv):(j + 1) * (h // kv)] = \
                (torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v[:, j]).transpose(0, 1)
        at += lq
    return out
