"""The operators around the paged cache and the logits: attention over the pages that the RoPE append wrote
(`paged_attn`), the same for a batch whose sequences share a long prefix (`paged_attn_shared`), and the log
probabilities of given tokens with entropy and top alternatives (`token_logprobs`).

Sizes are the repository's configurations: 64 / 8 heads of 128 (the large dense model), 16 / 8 heads of 128 (the
small one), 16 / 2 heads of 256 (the hybrid model's gated attention), pages of 256 tokens, vocabulary 151936.
`draw` spreads batches, lengths, heads, windows, page sizes and types over the ranges between and around them.
"""
import math
import os
import sys

import torch

own = False

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
DT = {"f16": F16, "bf16": BF16, "f32": F32}
ES = {"f16": 2, "bf16": 2, "f32": 4}


def _ffi():
    path = os.path.join(os.getcwd(), "exllamav3-rs_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import exl3r.ffi as ffi
    return ffi


def _attn(name, bsz, seq, lo, hi, hq, hk, hd, dtype, window=0, sinks=0, page=256, shared=0, lse=False, kind="attn"):
    return dict(name=name, kind=kind, bsz=bsz, seq=seq, lo=lo, hi=hi, hq=hq, hk=hk, hd=hd, dtype=dtype, window=window,
                sinks=sinks, page=page, shared=shared, lse=lse)


def listed():
    return [
        # One token of one chat, with a window: the smallest call, nothing but latency.
        _attn("decode_1_window", 1, 1, 1237, 1237, 16, 8, 128, "f16", window=512, sinks=4),
        # Batched decode of the large model, ragged lengths, full attention: the cache is the traffic.
        _attn("decode_64", 64, 1, 700, 8100, 64, 8, 128, "f16"),
        # Two long documents, one token each: few rows, a long axis.
        _attn("decode_2_long", 2, 1, 98765, 131000, 32, 4, 128, "bf16", lse=True),
        # Prefill of one long prompt, full attention: the matrix cores are the bound.
        _attn("prefill_4096", 1, 4096, 0, 0, 64, 8, 128, "bf16"),
        # Prefill of a longer prompt with a sliding window and sinks.
        _attn("prefill_8111_window", 1, 8111, 0, 0, 32, 8, 128, "f16", window=1024, sinks=4),
        # A chunk of a chunked prefill on top of what is cached, the hybrid model's heads of 256, small pages.
        _attn("chunk_3x511_hd256", 3, 511, 1800, 5300, 16, 2, 256, "bf16", page=16),
        # Generation for 64 requests with one long system prompt: one token each.
        _attn("shared_decode_64", 64, 1, 8192 + 9, 8192 + 700, 64, 8, 128, "f16", shared=8192, kind="shared"),
        # Scoring 16 candidate answers to one prompt: the answers' tokens at once.
        _attn("shared_score_16x37", 16, 37, 2048, 2048, 16, 8, 128, "bf16", shared=2048, kind="shared", lse=True),
        # Log probabilities beside the draw, one sequence: latency.
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=151936, dtype="f32", top=20),
        # The same for a decode batch.
        dict(name="logprobs_64", kind="logprobs", rows=64, vocab=151936, dtype="f32", top=20),
        # Scoring of a long prompt: every position's token, with the best five.
        dict(name="logprobs_4096", kind="logprobs", rows=4096, vocab=151936, dtype="bf16", top=5),
        # Perplexity over a ragged chunk, a vocabulary of odd size, no alternatives.
        dict(name="logprobs_511_odd", kind="logprobs", rows=511, vocab=32003, dtype="f16", top=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "chunk", "shared", "shared", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = rng.choice([151936, 128256, rng.randint(32000, 152000)])
        dtype = rng.choice(["f32", "f16", "bf16"])
        return dict(kind=kind, rows=_log(rng, 1, 4096 // ES[dtype] * 2), vocab=vocab, dtype=dtype,
                    top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]))
    hq, hk, hd = rng.choice([(16, 8, 128), (32, 8, 128), (64, 8, 128), (32, 4, 128), (40, 8, 128), (16, 2, 256),
                             (16, 16, 64), (28, 4, 64)])
    dtype, page, lse = rng.choice(["f16", "bf16"]), rng.choice([256, 256, 64, 16]), rng.random() < 0.3
    window, sinks = rng.choice([(0, 0), (_log(rng, 64, 4096), rng.choice([0, 1, 4, 37]))])
    key_bytes = 4 * hk * hd                                 # K and V of one position
    pairs = 4096 * 4096 * 64 * 128 // 2 // (hq * hd)        # tokens x keys of the largest listed prefill
    if kind == "decode":
        bsz = _log(rng, 1, 64)
        hi = _log(rng, 16, min(131072, (1 << 30) // (key_bytes * bsz)))
        return _unnamed(bsz, rng.choice([1, 1, 1, 2, 4]), rng.randint(0, hi), hi, hq, hk, hd, dtype, window, sinks, page,
                        lse=lse)
    if kind == "prefill":
        seq = _log(rng, 33, int(math.sqrt(4096 * 4096 * 64 * 128 / (hq * hd))) * 9 // 10)
        return _unnamed(1, seq, 0, 0, hq, hk, hd, dtype, window, sinks, page, lse=lse)
    if kind == "chunk":
        bsz, seq = rng.randint(1, 4), _log(rng, 5, 700)
        hi = _log(rng, 100, min(9000, pairs // (bsz * seq) - seq))
        return _unnamed(bsz, seq, rng.randint(0, hi), hi, hq, hk, hd, dtype, window, sinks, page, lse=lse)
    bsz, seq = _log(rng, 2, 64), rng.choice([1, 1, 1, 4, rng.randint(5, 40)])
    shared = 256 * _log(rng, 1, max(1, min(64, (pairs // (bsz * seq) - 1500) // 256)))
    hi = shared + _log(rng, 1, max(2, min(1500, (1 << 29) // (key_bytes * bsz))))
    return _unnamed(bsz, seq, rng.randint(shared, hi), hi, hq, hk, hd, dtype, window, sinks, page, shared, lse, "shared")


def _unnamed(*args, **kw):
    case = _attn(None, *args, **kw)
    del case["name"]
    return case


def _lens(case):
    """Tokens in the cache before the call, per sequence: spread over [lo, hi], the same in every run."""
    return [case["lo"] + int((case["hi"] - case["lo"]) * ((0.37 + 0.6180339887 * b) % 1.0)) for b in range(case["bsz"])]


def _visible(p, window, sinks):
    return p + 1 if window <= 0 else min(p + 1, window) + min(sinks, max(0, p + 1 - window))


def work(case):
    if case["kind"] == "logprobs":
        rows, n, k = case["rows"], case["vocab"], case["top"]
        # per logit: a subtraction, an exponential, two sums and a product
        return dict(bytes=rows * (n * ES[case["dtype"]] + 8 + 8 + 12 * k), flops=5 * rows * n)
    seq, hd, w, sk, shared = case["seq"], case["hd"], case["window"], case["sinks"], case["shared"]
    pairs, keys, low = 0, 0, shared
    for n in _lens(case):
        pairs += sum(_visible(n + s, w, sk) for s in range(seq))
        first = max(0, n - w + 1) if w > 0 else 0           # the first key that the first token's window holds
        low = min(low, first)
        keys += n + seq - max(first, shared) + max(0, min(sk, first) - shared)
    if shared:
        keys += shared - low + min(sk, low)                 # the prefix once, as far as some token sees it
    io = 2 * case["bsz"] * seq * case["hq"] * hd * 2 + (4 * case["bsz"] * seq * case["hq"] if case["lse"] else 0)
    return dict(bytes=keys * 2 * case["hk"] * hd * 2 + io, flops=4 * pairs * case["hq"] * hd)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "logprobs":
        rows, n = case["rows"], case["vocab"]
        x = torch.empty((rows, n), device="cuda", dtype=DT[case["dtype"]])
        for r in range(0, rows, 512):                       # a broad bulk and some tokens that stand out
            part = torch.randn((min(512, rows - r), n), generator=g, device="cuda") * 2.2 - 3.0
            at = torch.randint(0, n, (part.shape[0], 40), generator=g, device="cuda")
            part.scatter_add_(1, at, torch.rand(at.shape, generator=g, device="cuda") * 16.0)
            x[r:r + 512] = part.to(x.dtype)
        tokens = torch.randint(0, n, (rows,), generator=g, device="cuda")
        best = torch.cat([x[r:r + 512].argmax(dim=1) for r in range(0, rows, 512)])
        tokens = torch.where(torch.rand((rows,), generator=g, device="cuda") < 0.6, best, tokens)
        st = dict(case=case, x=x, tokens=tokens)
        if own:
            ffi = _ffi()
            k = case["top"]
            st["logprobs"] = torch.empty(rows, device="cuda", dtype=F32)
            st["entropy"] = torch.empty(rows, device="cuda", dtype=F32)
            st["top_ids"] = torch.empty((rows, k), device="cuda", dtype=torch.int64) if k else None
            st["top_logprobs"] = torch.empty((rows, k), device="cuda", dtype=F32) if k else None
            st["ws"] = torch.empty(ffi.token_logprobs_workspace_bytes(rows, n), device="cuda", dtype=torch.uint8)
        return st
    dt, bsz, seq, page, hk, hd = DT[case["dtype"]], case["bsz"], case["seq"], case["page"], case["hk"], case["hd"]
    lens = _lens(case)
    common = case["shared"] // page
    need = [(n + seq + page - 1) // page for n in lens]
    pages = common + sum(k - common for k in need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros((bsz, max(need) + 2), dtype=torch.int32)
    table[:, :common] = order[:common]
    at = common
    for b, k in enumerate(need):
        table[b, common:k] = order[at:at + k - common]
        at += k - common
    kc = torch.empty((pages, page, hk, hd), device="cuda", dtype=dt)
    vc = torch.empty_like(kc)
    step = max(1, (1 << 26) // (page * hk * hd))
    for c, std in ((kc, 1.0), (vc, 0.7)):
        for i in range(0, pages, step):
            c[i:i + step] = (torch.randn(c[i:i + step].shape, generator=g, device="cuda") * std).to(dt)
    q = (torch.randn((bsz, seq, case["hq"], hd), generator=g, device="cuda") * 1.2).to(dt)
    st = dict(case=case, q=q, kc=kc, vc=vc, table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              host_lens=lens)
    if own:
        ffi = _ffi()
        st["out"] = torch.empty_like(q)
        st["lse"] = torch.empty((bsz, seq, case["hq"]), device="cuda", dtype=F32) if case["lse"] else None
        st["ws"] = torch.empty(ffi.paged_attn_workspace_bytes(q, kc, st["table"], case["shared"]), device="cuda",
                               dtype=torch.uint8)
    return st


def run(st):
    case = st["case"]
    if case["kind"] == "logprobs":
        if own:
            ffi = _ffi()
            ffi.token_logprobs(st["x"], st["tokens"], st["logprobs"], st["entropy"], st["top_ids"], st["top_logprobs"],
                               workspace=st["ws"])
            return dict(logprobs=st["logprobs"], entropy=st["entropy"]) | (
                dict(top_ids=st["top_ids"], top_logprobs=st["top_logprobs"]) if case["top"] else {})
        return _plain_logprobs(st["x"], st["tokens"], case["top"])
    if own:
        ffi = _ffi()
        if case["kind"] == "shared":
            ffi.paged_attn_shared(st["q"], st["kc"], st["vc"], st["table"], st["lens"], st["out"], case["shared"],
                                  window=case["window"], sinks=case["sinks"], lse=st["lse"], workspace=st["ws"])
        else:
            ffi.paged_attn(st["q"], st["kc"], st["vc"], st["table"], st["lens"], st["out"], window=case["window"],
                           sinks=case["sinks"], lse=st["lse"], workspace=st["ws"])
        return dict(out=st["out"]) | (dict(lse=st["lse"]) if case["lse"] else {})
    return _plain_attn(st, case)


def _plain_logprobs(x, tokens, k):
    outs = []
    step = max(1, (1 << 27) // x.shape[1])
    for r in range(0, x.shape[0], step):
        f = x[r:r + step].float()
        t = f - f.max(dim=1, keepdim=True).values
        e = torch.exp(t)
        total = e.sum(dim=1)
        norm = torch.log(total)
        part = [t.gather(1, tokens[r:r + step, None])[:, 0] - norm, norm - (e * t).sum(dim=1) / total]
        if k:
            # the value's order in the high word, the earlier index first among equals
            bits = (f + 0.0).view(torch.int32)
            key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64)
            idx = torch.arange(f.shape[1], device=f.device)
            top = ((key << 32) + (0xffffffff - idx)).topk(k, dim=1).values
            ids = 0xffffffff - (top & 0xffffffff)
            part += [ids, t.gather(1, ids) - norm[:, None]]
        outs.append(part)
    cat = [torch.cat(p) for p in zip(*outs)]
    return dict(zip(("logprobs", "entropy", "top_ids", "top_logprobs"), cat))


def _plain_attn(st, case):
    q, hk, hd, seq = st["q"], case["hk"], case["hd"], case["seq"]
    g = case["hq"] // hk
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:3], device="cuda", dtype=F32)
    for b, n in enumerate(st["host_lens"]):
        rows = st["table"][b, :(n + seq + case["page"] - 1) // case["page"]].long()
        total = n + seq
        pos = n + torch.arange(seq, device="cuda")
        # a block of query tokens at a time, against the keys from the first that it sees; the sinks beside them
        step = max(1, min(seq, (1 << 28) // (g * total)))
        k_all = st["kc"][rows].reshape(-1, hk, hd)[:total]
        v_all = st["vc"][rows].reshape(-1, hk, hd)[:total]
        for h in range(hk):
            k, v = k_all[:, h].float(), v_all[:, h].float()
            for s in range(0, seq, step):
                p = pos[s:s + step]
                qs = q[b, s:s + step, h * g:(h + 1) * g].float().reshape(-1, hd)
                sc = torch.matmul(qs, k.t().contiguous()).view(p.shape[0], g, total) * (1.0 / math.sqrt(hd))
                j = torch.arange(total, device="cuda")
                see = j[None, :] <= p[:, None]
                if case["window"] > 0:
                    see &= (p[:, None] - j[None, :] < case["window"]) | (j[None, :] < case["sinks"])
                sc = torch.where(see[:, None, :], sc, float("-inf"))
                m = sc.max(dim=2, keepdim=True).values
                e = torch.exp(sc - m)
                l = e.sum(dim=2)
                o = torch.matmul(e.view(-1, total), v).view(p.shape[0], g, hd) / l[..., None]
                out[b, s:s + step, h * g:(h + 1) * g] = o.to(out.dtype)
                lse[b, s:s + step, h * g:(h + 1) * g] = m[..., 0] + torch.log(l)
    return dict(out=out) | (dict(lse=lse) if case["lse"] else {})


def exact(case, seed):
    """From the definitions, in 64 bits."""
    global own
    if case["kind"] != "logprobs" and work(case)["flops"] > 4e11:
        return None
    saved, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = saved
    if case["kind"] == "logprobs":
        names = ["logprobs", "entropy"] + (["top_ids", "top_logprobs"] if case["top"] else [])
        parts = {n: [] for n in names}
        for r in range(0, case["rows"], 64):
            x = st["x"][r:r + 64].double()
            z = torch.logsumexp(x, dim=1, keepdim=True)
            lp = x - z
            parts["logprobs"].append(torch.take_along_dim(lp, st["tokens"][r:r + 64, None], 1)[:, 0])
            parts["entropy"].append(-(lp.exp() * lp).sum(1))
            if case["top"]:
                v, i = torch.sort(x, dim=1, descending=True, stable=True)
                parts["top_ids"].append(i[:, :case["top"]].clone())
                parts["top_logprobs"].append(v[:, :case["top"]] - z)
        return {n: torch.cat(p) for n, p in parts.items()}
    q, hq, hk, hd, page = st["q"], case["hq"], case["hk"], case["hd"], case["page"]
    out = torch.empty(q.shape, device="cuda", dtype=F64)
    lse = torch.empty(q.shape[:3], device="cuda", dtype=F64)
    for b, n in enumerate(st["host_lens"]):
        at = torch.arange(n + case["seq"], device="cuda")
        page_of = st["table"][b].long()[at // page]
        for h in range(hk):
            keys, values = (c[page_of, at % page, h].double() for c in (st["kc"], st["vc"]))
            for head in range(h * (hq // hk), (h + 1) * (hq // hk)):
                for s in range(0, case["seq"], 1024):
                    here = n + s + torch.arange(min(1024, case["seq"] - s), device="cuda")
                    score = (q[b, s:s + 1024, head].double() / math.sqrt(hd)) @ keys.transpose(0, 1).contiguous()
                    back = here[:, None] - at[None, :]
                    hidden = back < 0
                    if case["window"] > 0:
                        hidden = hidden | ((back >= case["window"]) & (at[None, :] >= case["sinks"]))
                    score.masked_fill_(hidden, -math.inf)
                    z = torch.logsumexp(score, dim=1)
                    out[b, s:s + 1024, head] = torch.exp(score - z[:, None]) @ values
                    lse[b, s:s + 1024, head] = z
    return dict(out=out) | (dict(lse=lse) if case["lse"] else {})
