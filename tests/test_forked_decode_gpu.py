"""Decode steps of forked sequences whose Context states what they share: the model's attention computes the
shared pages once. Logits against the CPU oracle as in the test of candidates (same tolerance, derived
there), and against the same step without the statement."""
import pytest
import torch

import pagedkv
from pagedkv.qwen3 import Qwen3Adapters, Qwen3Config, Qwen3Model
from test_candidates_gpu import BS, TOL, _Run

pytestmark = pytest.mark.gpu


class _Forked(_Run):
    """Room for long prompts."""

    def __init__(self, gpu, cfg, adapters):
        super().__init__(gpu, cfg, adapters, rows=12, blocks=96)
        self.model = Qwen3Model(cfg, self.w, self.k, self.v, 2048)
        self.model.bind_adapters(adapters)
        self.tables = torch.full((12, 20), -1, dtype=torch.int32, device=gpu)

    def decode(self, rows, new_tokens):
        at = self.i32(rows)
        slots = pagedkv.extend_sequences(self.tables, self.lens, self.refs, BS, at)
        lens, tables = self.lens[at.long()], self.tables[at.long()].contiguous()
        shared = pagedkv.shared_prefix_keys(tables, BS)
        assert shared == 1024
        cu_q = torch.arange(len(rows) + 1, dtype=torch.int32, device=self.gpu)
        cu_k = torch.cat([torch.zeros_like(lens[:1]), torch.cumsum(lens, 0, dtype=torch.int32)])
        ids, pos = torch.tensor(new_tokens, device=self.gpu), (lens - 1).long()
        hidden = {}
        for hint in (None, shared):
            print(f"[forked decode] cached_prefix_keys={hint}", flush=True)
            ctx = pagedkv.Context(False, cu_q, cu_k, 1, 20 * BS, slots, None, tables, hint,
                                  self.i32([self.adapter[r] for r in rows]))
            hidden[hint] = self.model.forward(ids, pos, ctx)
        for r, t in zip(rows, new_tokens):
            self.tokens[r].append(t)
        for hint, h in hidden.items():
            self.check(rows, h, f"decode, cached_prefix_keys={hint}")
        a, b = (h.float() @ self.w.embed.float().T for h in hidden.values())
        assert float((a - b).abs().max()) <= TOL and not torch.equal(a, b)  # summed in another order


def _forked(gpu):
    """Two prompts, six forks: (run, rows, a function that draws tokens)."""
    cfg = Qwen3Config(num_hidden_layers=2, vocab_size=2048)
    run = _Forked(gpu, cfg, Qwen3Adapters(cfg, 2, 16, gpu, std=0.04))
    g = torch.Generator().manual_seed(5)

    def tokens(n):
        return torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()

    print("[forked decode] prefill", flush=True)
    run.prefill([tokens(1030), tokens(700)], [1, -1])
    parents, kids = [0, 0, 0, 0, 1, 1], [2, 3, 4, 5, 6, 7]
    pagedkv.fork_sequences(run.k, run.v, run.tables, run.lens, run.refs, run.i32(parents), run.i32(kids))
    for p, c in zip(parents, kids):
        run.tokens[c], run.adapter[c] = list(run.tokens[p]), run.adapter[p]
    return run, [0, 1] + kids, tokens


def test_forked_decode_with_a_stated_prefix(gpu):
    run, rows, tokens = _forked(gpu)
    for _ in range(2):
        run.decode(rows, tokens(len(rows)))


def test_captured_padded_step_with_a_stated_prefix(gpu):
    """The step captured with four padding rows, as the runner pads (slot -1, cu_seqlens tails of 0, tables
    and adapters of -1): every replay, with eager work between the replays, gives the eager call's bits."""
    run, rows, tokens = _forked(gpu)
    n, width = len(rows), 12
    at = run.i32(rows)
    slots, tables = torch.full((width,), -1, dtype=torch.int32, device=gpu), torch.full((width, 20), -1,
                                                                                       dtype=torch.int32, device=gpu)
    slots[:n] = pagedkv.extend_sequences(run.tables, run.lens, run.refs, BS, at)
    tables[:n] = run.tables[at.long()]
    lens = run.lens[at.long()]
    cu_q, cu_k = torch.zeros(2, width + 1, dtype=torch.int32, device=gpu)
    cu_q[:n + 1], cu_k[1:n + 1] = torch.arange(n + 1), torch.cumsum(lens, 0, dtype=torch.int32)
    ids, pos = torch.zeros(2, width, dtype=torch.int64, device=gpu)
    new = tokens(n)
    ids[:n], pos[:n] = torch.tensor(new), (lens - 1).long()
    ctx = pagedkv.Context(False, cu_q, cu_k, 1, 20 * BS, slots, None, tables, 1024,
                          run.i32([run.adapter[r] for r in rows] + [-1] * (width - n)))
    for r, t in zip(rows, new):
        run.tokens[r].append(t)
    print("[forked decode] eager, padded", flush=True)
    want = run.model.forward(ids, pos, ctx)[:n].clone()
    run.check(rows, want, "padded decode")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run.model.forward(ids, pos, ctx)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run.model.forward(ids, pos, ctx)
    for i in range(4):
        print(f"[forked decode] replay {i}", flush=True)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:n].view(torch.int16), want.view(torch.int16))
        run.model.forward(ids, pos, ctx)
        torch.cuda.synchronize()
