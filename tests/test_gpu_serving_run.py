"""The serving operators together: rope_paged_kv fills the cache, paged_attn (or paged_attn_shared) reads it, the logits
of its output go to argmax_sample and token_logprobs; eagerly and from one captured graph, token after token."""
import math

import pytest
import torch

import exl3r.ffi as ffi
from exl3r import ROPE_NEOX

pytestmark = pytest.mark.gpu

HQ, HK, HD, PAGE, VOCAB, TOP = 16, 4, 64, 32, 4001, 5


class Decoder:
    """One attention layer over a paged cache and logits of its output; every tensor is kept, as a graph needs it."""

    def __init__(self, lens, blocks, dtype, shared, window, sinks, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.bsz, self.shared, self.window, self.sinks = len(lens), shared, window, sinks
        pages = len(lens) * blocks
        self.kc, self.vc = (torch.randn((pages, PAGE, HK, HD), generator=g, device="cuda").to(dtype) for _ in range(2))
        table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).view(len(lens), blocks)
        table[:, :shared // PAGE] = table[0, :shared // PAGE]
        self.table = table.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.inv = 1.0 / 10000.0 ** (torch.arange(0, HD, 2, device="cuda").float() / HD)
        self.pick = torch.randint(0, HQ * HD, (VOCAB,), generator=g, device="cuda")      # a logit is one output's multiple
        self.gain = 4 * torch.randn(VOCAB, generator=g, device="cuda")
        self.q = torch.empty((self.bsz, 1, HQ, HD), dtype=dtype, device="cuda")
        self.k, self.v = (torch.empty((self.bsz, 1, HK, HD), dtype=dtype, device="cuda") for _ in range(2))
        self.out, self.roped = torch.empty_like(self.q), torch.empty_like(self.q)
        self.logits = torch.empty((self.bsz, VOCAB), device="cuda")
        self.ids = torch.empty(self.bsz, dtype=torch.int64, device="cuda")
        self.lp, self.ent = (torch.empty(self.bsz, device="cuda") for _ in range(2))
        self.top_ids = torch.empty((self.bsz, TOP), dtype=torch.int64, device="cuda")
        self.top_lp = torch.empty((self.bsz, TOP), device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.ws = torch.empty(max(256, ffi.paged_attn_workspace_bytes(self.q, self.kc, self.table, shared)), dtype=torch.uint8, device="cuda")
        self.lws = torch.empty(max(256, ffi.token_logprobs_workspace_bytes(self.bsz, VOCAB)), dtype=torch.uint8, device="cuda")

    def draw(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))

    def step(self):
        ffi.rope_paged_kv(self.q, self.roped, self.k, None, self.v, self.inv, 0, self.lens, None, None, 1e-6, 0.0,
                          ROPE_NEOX, 1.0, self.kc, self.vc, self.table, self.lens, err_flag=self.err)
        if self.shared:
            ffi.paged_attn_shared(self.roped, self.kc, self.vc, self.table, self.lens, self.out, self.shared, window=self.window,
                                  sinks=self.sinks, workspace=self.ws, err_flag=self.err)
        else:
            ffi.paged_attn(self.roped, self.kc, self.vc, self.table, self.lens, self.out, window=self.window, sinks=self.sinks,
                           workspace=self.ws, err_flag=self.err)
        self.logits.copy_(self.out.view(self.bsz, -1).float()[:, self.pick] * self.gain)
        ffi.argmax_sample(self.logits, self.ids)
        ffi.token_logprobs(self.logits, self.ids, self.lp, self.ent, self.top_ids, self.top_lp, workspace=self.lws,
                           err_flag=self.err)

    def results(self):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.out, self.logits, self.ids, self.lp, self.ent, self.top_ids, self.top_lp, self.kc, self.vc)]

    def check(self):
        """The attention from the cache in 64 bits, the log probabilities from the logits in 64 bits."""
        u = torch.finfo(self.q.dtype).eps / 2
        lens = self.lens.tolist()
        for b, n in enumerate(lens):
            j = torch.arange(n + 1, device="cuda")
            pg = self.table[b].long()[j // PAGE]
            k, v = self.kc[pg, j % PAGE].double(), self.vc[pg, j % PAGE].double()
            # the new token's keys and values are where the append put them
            assert torch.equal(self.vc[pg[-1], n % PAGE], self.v[b, 0])
            see = (n - j < self.window) | (j < self.sinks) if self.window else torch.ones_like(j, dtype=torch.bool)
            for h in range(HQ):
                kh, vh = k[see, h // (HQ // HK)], v[see, h // (HQ // HK)]
                qh = self.roped[b, 0, h].double()
                s = (kh * qh).sum(1) / math.sqrt(HD)
                w = torch.softmax(s, 0)
                want = (w[:, None] * vh).sum(0)
                # u for a weight's rounding, a score's error twice, fp32 sums; u for the output's rounding
                d = 2 * (HD + 2) * 2.0 ** -24 * ((kh * qh).abs().sum(1) / math.sqrt(HD)).max() + 2.0 ** -21 + 2.0 ** -22 * (s.max() - s.min())
                tol = (u + 2 * d + 2.0 ** -19) * (w[:, None] * vh.abs()).sum(0) + u * want.abs() + 2.0 ** -25 + 2.0 ** -31 * vh.abs().sum(0)
                got = self.out[b, 0, h].double()
                assert ((got - want).abs() <= tol).all(), (b, h, ((got - want).abs() / tol).max().item())
        x = self.logits.double()
        lp = torch.log_softmax(x, 1)
        assert torch.equal(self.ids, x.argmax(1))
        assert torch.equal(self.top_ids[:, 0], self.ids) and torch.equal(self.top_lp[:, 0], self.lp)
        v, _ = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(x.gather(1, self.top_ids), v[:, :TOP])
        # e: 48 fp32 additions and an exponential's 2^-22 in the sum; one rounding of a value below 64; the entropy is
        # ln l - t / l, the second below 64 with twice that relative error
        e = 48 * 2.0 ** -24 + 2.0 ** -22
        assert ((self.top_lp - lp.gather(1, self.top_ids)).abs() <= e + 2.0 ** -19).all()
        ent = -(lp.exp() * lp).sum(1)
        assert ((self.ent - ent).abs() <= e + 64 * 2 * e + 2.0 ** -19).all()
        assert self.err.item() == 0


RUNS = [
    # lens, dtype, shared, window, sinks
    ([63, 0, 31, 200], torch.float16, 0, 0, 0),
    ([63, 0, 31, 200], torch.bfloat16, 0, 40, 3),
    ([64, 100, 95, 70, 64, 127], torch.bfloat16, 64, 0, 0),
    ([130], torch.float16, 0, 0, 0),
]


@pytest.mark.parametrize("lens,dtype,shared,window,sinks", RUNS)
def test_tokens_one_after_the_other(lens, dtype, shared, window, sinks):
    d = Decoder(lens, 9, dtype, shared, window, sinks, seed=7)
    for t in range(4):
        d.draw(100 + t)
        d.step()
        torch.cuda.synchronize()
        d.check()
        d.lens += 1


@pytest.mark.parametrize("lens,dtype,shared,window,sinks", RUNS[1:3])
def test_captured_step(lens, dtype, shared, window, sinks):
    """One captured step, replayed for token after token, against eager steps of a second decoder in between."""
    d, e = (Decoder(lens, 9, dtype, shared, window, sinks, seed=8) for _ in range(2))
    cache = d.kc.clone(), d.vc.clone()
    side = torch.cuda.Stream()
    d.draw(0)
    with torch.cuda.stream(side):
        d.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.step()
    d.kc.copy_(cache[0])
    d.vc.copy_(cache[1])
    for t in range(4):
        for x in (d, e):
            x.draw(200 + t)
        graph.replay()
        torch.cuda.synchronize()
        d.check()
        e.step()
        for a, b in zip(d.results(), e.results()):
            assert torch.equal(a, b)
        for x in (d, e):
            x.lens += 1


def test_two_captured_steps_at_once():
    """Two graphs with workspaces of their own, replayed on two streams."""
    a, b = (Decoder([150 + 30 * i, 9, 200], 9, torch.float16, 0, 0, 0, seed=9 + i) for i in range(2))
    graphs = []
    for x in (a, b):
        x.draw(1)
        x.step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.step()
        graphs.append(g)
    want = [x.results() for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, w in zip((a, b), want):
            for p, q in zip(x.results(), w):
                assert torch.equal(p, q)
