"""The page operators and the adapters together, as a step of parallel candidates uses them: prompts with
an adapter each go through a two-layer model of the 0.6B geometry into a paged cache, their pages
are forked into candidates, the candidates grow page by page and decode with their prompt's
adapter, some are freed, the cache is compacted, the others go on. Every step's logits are compared
with the CPU oracle run over the candidate's whole token list with the adapter merged into the weights
(in fp32, unrounded).

Tolerance on the logits: a row passes about 20 roundings to bf16 in two layers on either side, each
with a standard deviation of 2^-9 / sqrt(3) to 2^-8 / sqrt(3) of what it rounds, which add like
independent errors: sqrt(40) 2^-8 / sqrt(3) = 1.4% of the final hidden row at most, whose logits
spread by 0.02 sqrt(1024) = 0.64: 0.009, and over some 10^5 compared values 5 standard deviations,
0.045. A candidate with another one's adapter, page or position is off by 0.3 and more, which the
test checks on the oracle's side.
"""
from types import SimpleNamespace

import pytest
import torch

import pagedkv
from oracle import qwen3 as Q
from pagedkv.qwen3 import Qwen3Adapters, Qwen3Config, Qwen3Model, Qwen3Weights

pytestmark = pytest.mark.gpu

BS, TOL = 64, 0.05


def _merged(w, ad, adapter):
    """CPU weights with one adapter (-1: none) added, in fp32."""
    layers = []
    for L, A in zip(w.layers, ad.layers):
        out = {n: t.cpu() for n, t in L.items()}
        if adapter >= 0:
            for name, widths in ad.slices.items():
                a, b = A[name][0][adapter].cpu().float(), A[name][1][adapter].cpu().float()
                r, at, rows = b.shape[1], 0, []
                for q, n in enumerate(widths):
                    rows.append(b[at:at + n] @ a[q * r:(q + 1) * r])
                    at += n
                out[name] = out[name].float() + float(ad.scales[adapter]) * torch.cat(rows)
        layers.append(out)
    return SimpleNamespace(embed=w.embed.cpu(), final_norm=w.final_norm.cpu(), layers=layers)


class _Run:
    def __init__(self, gpu, cfg, adapters, rows=16, blocks=48):
        self.gpu, self.cfg = gpu, cfg
        self.w = Qwen3Weights(cfg, gpu)
        self.ad = adapters
        kv = torch.zeros(2, cfg.num_hidden_layers, blocks, BS, cfg.num_key_value_heads, cfg.head_dim,
                         dtype=torch.bfloat16, device=gpu)
        self.k, self.v = kv[0], kv[1]
        self.model = Qwen3Model(cfg, self.w, self.k, self.v, 1024)
        self.model.bind_adapters(adapters)
        self.tables = torch.full((rows, 6), -1, dtype=torch.int32, device=gpu)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=gpu)
        self.refs = torch.zeros(blocks, dtype=torch.int32, device=gpu)
        self.tokens, self.adapter = {}, {}
        self.oracle = {a: _merged(self.w, adapters, a) for a in range(-1, adapters.scales.numel())}

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.gpu)

    def check(self, rows, hidden, what):
        got = (hidden.float() @ self.w.embed.float().T).cpu()
        for i, r in enumerate(rows):
            want = Q.forward_logits(self.oracle[self.adapter[r]], self.cfg, self.tokens[r])[-1]
            err = float((got[i] - want).abs().max())
            assert err <= TOL, f"{what}: row {r} (adapter {self.adapter[r]}) off by {err:.3f}"

    def prefill(self, prompts, adapters):
        """Rows 0 .. get the prompts, in blocks from the end of the cache."""
        free, cu, slots = self.refs.numel() - 1, [0], []
        for r, (p, a) in enumerate(zip(prompts, adapters)):
            self.tokens[r], self.adapter[r] = list(p), a
            for j in range(-(-len(p) // BS)):
                self.tables[r, j] = free
                self.refs[free] = 1
                free -= 2  # with holes
            self.lens[r] = len(p)
            slots += [int(self.tables[r, t // BS]) * BS + t % BS for t in range(len(p))]
            cu.append(cu[-1] + len(p))
        ids = self.i32([a for p, a in zip(prompts, adapters) for _ in p])
        ctx = pagedkv.Context(True, self.i32(cu), self.i32(cu), max(map(len, prompts)), max(map(len, prompts)),
                              self.i32(slots), None, None, adapter_ids=ids)
        hidden = self.model.forward(torch.tensor([t for p in prompts for t in p], device=self.gpu),
                                    torch.cat([torch.arange(len(p)) for p in prompts]).to(self.gpu), ctx)
        self.check(range(len(prompts)), hidden[self.i32(cu[1:]).long() - 1], "prefill")

    def decode(self, rows, new_tokens):
        """One more token for every row, all on the device but the tokens' choice."""
        at = self.i32(rows)
        slots = pagedkv.extend_sequences(self.tables, self.lens, self.refs, BS, at)
        lens = self.lens[at.long()]
        cu_k = torch.cat([torch.zeros_like(lens[:1]), torch.cumsum(lens, 0, dtype=torch.int32)])
        ctx = pagedkv.Context(False, torch.arange(len(rows) + 1, dtype=torch.int32, device=self.gpu), cu_k, 1, 384,
                              slots, None, self.tables[at.long()].contiguous(),
                              adapter_ids=self.i32([self.adapter[r] for r in rows]))
        hidden = self.model.forward(torch.tensor(new_tokens, device=self.gpu), (lens - 1).long(), ctx)
        for r, t in zip(rows, new_tokens):
            self.tokens[r].append(t)
        assert int(slots.min()) >= 0
        self.check(rows, hidden, f"decode of {rows}")


def test_candidates_of_adapted_prompts(gpu):
    cfg = Qwen3Config(num_hidden_layers=2, vocab_size=2048)
    ad = Qwen3Adapters(cfg, 3, 16, gpu, std=0.04)
    run = _Run(gpu, cfg, ad)
    g = torch.Generator().manual_seed(11)

    def tokens(n):
        return torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()

    prompts = [tokens(n) for n in (61, 64, 130, 20)]  # a page to fill, a full one, several, short
    print("[candidates] prefill", flush=True)
    run.prefill(prompts, [2, 0, -1, 1])
    # what the comparison would see of a mix-up of adapters
    a, b = (Q.forward_logits(run.oracle[i], cfg, run.tokens[0])[-1] for i in (2, 0))
    assert float((a - b).abs().max()) > 4 * TOL
    parents, kids = [0, 0, 0, 1, 1, 2, 3, 3], [4, 5, 6, 7, 8, 9, 10, 11]
    print("[candidates] fork", flush=True)
    new = pagedkv.fork_sequences(run.k, run.v, run.tables, run.lens, run.refs, run.i32(parents), run.i32(kids))
    assert [int(x) >= 0 for x in new] == [True, True, True, False, False, True, True, True]
    for p, c in zip(parents, kids):
        run.tokens[c], run.adapter[c] = list(run.tokens[p]), run.adapter[p]
    # children and parents grow in one batch: 61 + 5 tokens cross into a new page
    rows = [0, 1, 2, 3] + kids
    for step in range(5):
        print(f"[candidates] decode {step}", flush=True)
        run.decode(rows, tokens(len(rows)))
    done = [0, 2, 5, 7, 10]
    print("[candidates] free, compact", flush=True)
    pagedkv.free_sequences(run.tables, run.lens, run.refs, BS, run.i32(done))
    _, live = pagedkv.compact_blocks(run.k, run.v, run.tables, run.lens, run.refs)
    rows = [r for r in rows if r not in done]
    used = run.tables[run.tables >= 0]
    assert int(live) == int((run.refs > 0).sum()) == int(used.unique().numel()) == int(used.max()) + 1
    for step in range(3):
        print(f"[candidates] decode after compaction {step}", flush=True)
        run.decode(rows, tokens(len(rows)))
    pagedkv.free_sequences(run.tables, run.lens, run.refs, BS, run.i32(rows))
    assert not bool(run.refs.any()) and bool((run.tables == -1).all())


@pytest.mark.parametrize("n", [5, 200])
def test_tokens_without_an_adapter_are_the_base_model(gpu, n):
    """A step whose tokens have no adapter gives the base model's bits, adapters bound or not."""
    cfg = Qwen3Config(num_hidden_layers=2, vocab_size=2048)
    model = Qwen3Model(cfg, Qwen3Weights(cfg, gpu), None, None, 512)
    ids = torch.randint(0, 2048, (n,), generator=torch.Generator().manual_seed(1)).to(gpu)
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    ctx = pagedkv.Context(True, cu, cu, n, n, None, None, None)
    pos = torch.arange(n, device=gpu)
    print(f"[adapters] none, {n} tokens", flush=True)
    base = model.forward(ids, pos, ctx)
    model.bind_adapters(Qwen3Adapters(cfg, 2, 8, gpu))
    assert torch.equal(model.forward(ids, pos, ctx), base)
    ctx.adapter_ids = torch.full((n,), -1, dtype=torch.int32, device=gpu)
    assert torch.equal(model.forward(ids, pos, ctx), base)
    ctx.adapter_ids[0] = 1
    assert not torch.equal(model.forward(ids, pos, ctx), base)
