"""Operators of packed prompts, drafted tokens and scored tokens: their cases.

listed() holds the cases, draw(rng) more of the same ranges; prepare(case,
seed) makes what a program has in hand before the call, run(state) is one
pass, work(case) the bytes and operations no implementation can do without,
exact(case, seed) the result in 64 bits.  With `own` false, run() computes
the operators in plain torch operations; with `own` true it calls the
framework's kernels.

Operators:
  packed    causal attention over packed prompts of different lengths, with
            grouped heads: the forward pass of a prefill, or a training step's
            forward and backward pass
  tree      attention of a tree of drafted tokens over a key/value cache (one
            token is the tree of one)
  logprob   log probabilities of given tokens, the entropy and the top
            alternatives: scoring, or a training step's forward and backward
            pass through log probability and entropy
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # three short prompts of a small decoder (8 heads of 64): latency
        dict(name="packed_short", op="packed", lens="17,1,40", heads=8, kv_heads=8, d=64, dtype="float32",
             train=False),
        # a ragged batch of prompts through a decoder with grouped heads and an
        # fp32 cache
        dict(name="packed_ragged", op="packed", lens="1031,5,517,2047,130,366", heads=32, kv_heads=4, d=64,
             dtype="float32", train=False),
        # one long document, bf16: the largest prompt
        dict(name="packed_long", op="packed", lens="8192", heads=32, kv_heads=8, d=128, dtype="bfloat16", train=False),
        # a training step over packed documents, bf16
        dict(name="packed_train", op="packed", lens="4096,1500,33,900,663,1000", heads=32, kv_heads=8, d=128,
             dtype="bfloat16", train=True),
        # a training step in fp32, a head size and lengths that fit no tile
        dict(name="packed_train_odd", op="packed", lens="777,1,1250,63", heads=12, kv_heads=4, d=80, dtype="float32",
             train=True),
        # a plain decode step: one token over a middling cache
        dict(name="tree_token", op="tree", batch=1, tokens=1, cap=1024, length=515, heads=8, kv_heads=8, d=64,
             dtype="float32"),
        # two dozen drafted tokens over an almost full cache, grouped heads
        dict(name="tree_draft", op="tree", batch=1, tokens=24, cap=2048, length=2019, heads=32, kv_heads=4, d=64,
             dtype="float32"),
        # a serving batch with large trees over long bf16 caches
        dict(name="tree_batch", op="tree", batch=16, tokens=64, cap=8192, length=8001, heads=32, kv_heads=8, d=128,
             dtype="bfloat16"),
        # a few sampled tokens with their top alternatives
        dict(name="logprob_step", op="logprob", rows=4, vocab=32000, top=20, dtype="float32", train=False),
        # a prompt scored over a large vocabulary, bf16 logits
        dict(name="logprob_score", op="logprob", rows=2048, vocab=128000, top=5, dtype="bfloat16", train=False),
        # a training step through the loss, bf16 logits
        dict(name="logprob_train", op="logprob", rows=4096, vocab=32000, top=0, dtype="bfloat16", train=True),
        # the same in fp32 with a vocabulary that no vector width divides
        dict(name="logprob_train_odd", op="logprob", rows=1001, vocab=50001, top=0, dtype="float32", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 8), (8, 2), (32, 4), (32, 8), (12, 4), (12, 12), (16, 1)]


def draw(rng):
    op = rng.choice(["packed", "packed", "tree", "logprob"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    if op == "packed":
        total = _log(rng, 16, 8192)
        cuts = sorted(rng.random() for _ in range(rng.randint(0, 9)))
        heads, kv = rng.choice(HEADS)
        case = dict(op=op, lens="", heads=heads, kv_heads=kv, d=rng.choice([32, 64, 80, 96, 128]), dtype=dtype,
                    train=rng.random() < 0.5)
        while True:
            ends = [int(c * total) for c in cuts] + [total]
            case["lens"] = ",".join(str(b - a) for a, b in zip([0] + ends, ends))
            if work(case)["flops"] <= 5e11:      # no more than the largest of the listed
                return case
            total = total * 3 // 4
    if op == "tree":
        heads, kv = rng.choice(HEADS)
        tokens = _log(rng, 1, 64)
        length = _log(rng, 8, 8100)
        return dict(op=op, batch=_log(rng, 1, 16), tokens=tokens, cap=length + tokens + rng.randint(0, 100),
                    length=length, heads=heads, kv_heads=kv, d=rng.choice([32, 64, 80, 128]), dtype=dtype)
    rows, vocab = _log(rng, 1, 4096), _log(rng, 1000, 128000)
    rows = min(rows, 2048 * 128000 // vocab // (4 if dtype == "float32" else 2))
    train = rng.random() < 0.5
    return dict(op=op, rows=rows, vocab=vocab, top=0 if train else rng.choice([0, 1, 5, 20]), dtype=dtype, train=train)


# ── inputs ───────────────────────────────────────────────────────────────

def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=gen)

    s = dict(case)
    if case["op"] == "packed":
        lens = _lens(case)
        total, H, G, d = sum(lens), case["heads"], case["kv_heads"], case["d"]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, device=DEV, dtype=torch.int32)
        # what a projection of normed states gives: values near 1, keys and
        # queries with a few strong directions
        s["q"] = (randn(total, H, d) * 1.5).to(dt)
        s["k"] = (randn(total, G, d) + 0.5 * randn(1, G, d)).to(dt)
        s["v"] = randn(total, G, d).to(dt)
        if case["train"]:
            s["grad"] = randn(total, H, d).to(dt)
            for n in "qkv":
                s[n].requires_grad_()
    elif case["op"] == "tree":
        B, T, H, G, d = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "d"))
        s["k"] = randn(B, G, case["cap"], d).to(dt)
        s["v"] = randn(B, G, case["cap"], d).to(dt)
        s["q"] = (randn(B, T, H, d) * 1.5).to(dt)
        # caches of a batch differ in length; the first is the longest
        cut = torch.randint(0, case["length"] // 2 + 1, (B,), device=DEV, generator=gen)
        cut[0] = 0
        s["len"] = (case["length"] - cut).to(torch.int32)
        # each drafted token continues an earlier one or the cache itself (-1)
        u = torch.rand((B, T), device=DEV, generator=gen)
        t = torch.arange(T, device=DEV)
        s["parents"] = ((u * (t + 1)).floor().clamp(max=t) - 1).to(torch.int32)
    else:
        N, V = case["rows"], case["vocab"]
        x = torch.empty((N, V), device=DEV, dtype=dt)
        for i in range(0, N, 256):
            n = min(256, N - i)
            # a broad bulk with a few likely tokens and a few forbidden ones
            c = randn(n, V) * 2.0
            hot = torch.randint(0, V, (n, 8), device=DEV, generator=gen)
            c.scatter_add_(1, hot, 6.0 + 2.0 * randn(n, 8))
            c.scatter_(1, torch.randint(0, V, (n, 16), device=DEV, generator=gen), -math.inf)
            x[i:i + n] = c.to(dt)
        tok = torch.randint(0, V, (N,), device=DEV, generator=gen)
        # half of the tokens are the likeliest ones, as sampled text has them
        tok = torch.where(torch.rand(N, device=DEV, generator=gen) < 0.5, x.argmax(-1), tok)
        # a forbidden token is never the given one
        x.scatter_(1, tok[:, None], x.gather(1, tok[:, None]).clamp(min=-30.0))
        s["x"], s["tok"] = x, tok
        if case["train"]:
            s["g_lp"] = randn(N)
            s["g_ent"] = 0.1 * randn(N)
            x.requires_grad_()
    return s


# ── plain forms ──────────────────────────────────────────────────────────

def _plain_packed(s):
    H, G, d = s["heads"], s["kv_heads"], s["d"]
    rep, scale, dt = H // G, 1.0 / math.sqrt(d), DTYPES[s["dtype"]]
    q, k, v = (s[n].detach() for n in "qkv")
    out = torch.empty_like(q)
    if s["train"]:
        dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    a = 0
    for n in _lens(s):
        b = a + n
        if n == 0:
            continue
        # one group of heads at a time: [rep, n, d] queries over [n, d] keys
        future = torch.ones((n, n), device=q.device, dtype=torch.bool).triu(1)
        for g in range(G):
            hs = slice(g * rep, (g + 1) * rep)
            qg = q[a:b, hs].float().transpose(0, 1).contiguous()
            kg, vg = k[a:b, g].float().contiguous(), v[a:b, g].float().contiguous()
            sc = torch.matmul(qg, kg.t().contiguous()).mul_(scale).masked_fill_(future, -math.inf)
            p = torch.exp(sc - sc.amax(-1, keepdim=True))
            p /= p.sum(-1, keepdim=True)
            og = torch.matmul(p, vg)
            out[a:b, hs] = og.transpose(0, 1).to(dt)
            if s["train"]:
                go = s["grad"][a:b, hs].float().transpose(0, 1).contiguous()
                dp = torch.matmul(go, vg.t().contiguous())
                ds = p * (dp - (go * og).sum(-1, keepdim=True)) * scale
                dq[a:b, hs] = torch.matmul(ds, kg).transpose(0, 1).to(dt)
                dk[a:b, g] = torch.matmul(ds.reshape(rep * n, n).t().contiguous(), qg.reshape(rep * n, d)).to(dt)
                dv[a:b, g] = torch.matmul(p.reshape(rep * n, n).t().contiguous(), go.reshape(rep * n, d)).to(dt)
        a = b
    return (out, dq, dk, dv) if s["train"] else out


def _plain_tree(s):
    B, T, H, G, d = (s[n] for n in ("batch", "tokens", "heads", "kv_heads", "d"))
    rep, scale = H // G, 1.0 / math.sqrt(d)
    L = s["cap"]
    # seen[b, t, u]: drafted token u is t or one of its ancestors
    seen = torch.zeros((B, T, T), device=DEV, dtype=torch.bool)
    par = s["parents"].long()
    for t in range(T):
        up = seen.gather(1, par[:, t].clamp(min=0)[:, None, None].expand(B, 1, T))[:, 0]
        seen[:, t] = up & (par[:, t] >= 0)[:, None]
        seen[:, t, t] = True
    pos = torch.arange(L, device=DEV)
    u = pos[None] - s["len"][:, None]                                 # [B, L] drafted index of a position
    draft = seen.gather(2, u.clamp(0, T - 1)[:, None, :].expand(B, T, L))
    ok = (u < 0)[:, None] | (draft & ((u >= 0) & (u < T))[:, None])   # [B, T, L]
    q = s["q"].float().view(B, T, G, rep, d).permute(0, 2, 3, 1, 4).reshape(B, G, rep * T, d).contiguous()
    sc = torch.matmul(q, s["k"].float().transpose(2, 3).contiguous()) * scale
    sc = sc.view(B, G, rep, T, L).masked_fill(~ok[:, None, None], -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, G, rep * T, L), s["v"].float()).view(B, G, rep, T, d)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, d).to(DTYPES[s["dtype"]])


def _plain_logprob(s):
    x = s["x"].detach()
    N = s["rows"]
    lp, ent = (torch.empty(N, device=DEV) for _ in range(2))
    top = s["top"]
    tv = torch.empty((N, top), device=DEV)
    ti = torch.empty((N, top), device=DEV, dtype=torch.int64)
    dx = torch.empty_like(x) if s["train"] else None
    for i in range(0, N, 512):
        r = slice(i, min(N, i + 512))
        xr = x[r].float()
        z = xr - xr.amax(-1, keepdim=True)
        e = torch.exp(z)
        tot = e.sum(-1, keepdim=True)
        logp = z - torch.log(tot)
        lp[r] = logp.gather(1, s["tok"][r, None])[:, 0]
        p = e / tot
        plogp = torch.where(e > 0, p * logp, torch.zeros_like(p))
        ent[r] = -plogp.sum(-1)
        if top:
            v, j = torch.sort(xr, dim=-1, descending=True, stable=True)   # equal values: the lowest token first
            ti[r] = j[:, :top]
            tv[r] = logp.gather(1, ti[r])
        if s["train"]:
            g = -s["g_lp"][r, None] * p - s["g_ent"][r, None] * (plogp + p * ent[r, None])
            g.scatter_add_(1, s["tok"][r, None], s["g_lp"][r, None])
            dx[r] = g.to(x.dtype)
    if s["train"]:
        return lp, ent, dx
    return (lp, ent, tv, ti) if top else (lp, ent)


def run(state):
    s = state
    if not own:
        return {"packed": _plain_packed, "tree": _plain_tree, "logprob": _plain_logprob}[s["op"]](s)
    from rac_amd import ext, rac_torch
    if s["op"] == "packed":
        if not s["train"]:
            return ext.packed_attention(s["q"], s["k"], s["v"], s["cu"])
        out = rac_torch.rac_packed_attention(s["q"], s["k"], s["v"], s["cu"])
        return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])
    if s["op"] == "tree":
        return ext.tree_attention(s["q"], s["k"], s["v"], s["len"], s["parents"])
    if not s["train"]:
        return ext.token_logprobs(s["x"], s["tok"], top=s["top"])
    lp, ent = rac_torch.rac_token_logprobs(s["x"], s["tok"])
    dx, = torch.autograd.grad((lp, ent), s["x"], (s["g_lp"], s["g_ent"]))
    return lp.detach(), ent.detach(), dx


# ── work and the result in 64 bits ───────────────────────────────────────

def work(case):
    es = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "packed":
        lens = _lens(case)
        total, H, G, d = sum(lens), case["heads"], case["kv_heads"], case["d"]
        pairs = H * sum(n * (n + 1) // 2 for n in lens)
        io = total * d * es
        if not case["train"]:
            return {"bytes": io * (2 * H + 2 * G), "flops": 4 * d * pairs}
        # forward and backward: q, k, v, grad read; out, dq, dk, dv written
        return {"bytes": io * (4 * H + 4 * G), "flops": 14 * d * pairs}
    if case["op"] == "tree":
        B, T, H, G, d = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "d"))
        # the batch's caches are 3/4 of the longest on average, but for the first
        keys = case["length"] + (B - 1) * case["length"] * 3 // 4 + B * T
        return {"bytes": es * d * (2 * G * keys + 2 * B * T * H), "flops": 4 * d * H * T * keys}
    n = case["rows"] * case["vocab"]
    if case["train"]:
        return {"bytes": 2 * n * es, "flops": 12 * n}
    return {"bytes": n * es, "flops": 6 * n}


def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "packed":
        H, G, d = case["heads"], case["kv_heads"], case["d"]
        q, k, v = (s[n].detach().to(f8) for n in "qkv")
        out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
        start = 0
        for n in _lens(case):
            rows = slice(start, start + n)
            start += n
            for h in range(H if n else 0):
                g = h // (H // G)
                Q, K, V = q[rows, h].contiguous(), k[rows, g].contiguous(), v[rows, g].contiguous()
                S = (Q @ K.T.contiguous()) / math.sqrt(d)
                S = torch.tril(S) + torch.triu(torch.full_like(S, -math.inf), 1)
                P = torch.softmax(S, -1)
                O = P @ V
                out[rows, h] = O
                if case["train"]:
                    gO = s["grad"][rows, h].to(f8).contiguous()
                    dv[rows, g] += P.T.contiguous() @ gO
                    D = (gO * O).sum(-1, keepdim=True)
                    dS = P * (gO @ V.T.contiguous() - D) / math.sqrt(d)
                    dq[rows, h] = dS @ K
                    dk[rows, g] += dS.T.contiguous() @ Q
        return (out, dq, dk, dv) if case["train"] else out
    if case["op"] == "tree":
        B, T, H, G = (case[n] for n in ("batch", "tokens", "heads", "kv_heads"))
        lens, par = s["len"].tolist(), s["parents"].tolist()
        out = torch.empty(s["q"].shape, device=DEV, dtype=f8)
        for b in range(B):
            # the positions token t sees: the cache, its ancestors, itself
            seen = torch.zeros((T, lens[b] + T), device=DEV, dtype=torch.bool)
            seen[:, :lens[b]] = True
            for t in range(T):
                u = t
                while u >= 0:
                    seen[t, lens[b] + u] = True
                    u = par[b][u]
            for g in range(G):
                K, V = (s[n][b, g, :lens[b] + T].to(f8) for n in "kv")
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    S = s["q"][b, :, h].to(f8).contiguous() @ K.T.contiguous() / math.sqrt(case["d"])
                    out[b, :, h] = torch.softmax(torch.where(seen, S, -math.inf), -1) @ V
        return out
    N, top = case["rows"], case["top"]
    x, tok = s["x"].detach(), s["tok"]
    lp, ent = (torch.empty(N, device=DEV, dtype=f8) for _ in range(2))
    tv = torch.empty((N, top), device=DEV, dtype=f8)
    dx = torch.empty(x.shape, device=DEV, dtype=f8) if case["train"] else None
    for a in range(0, N, 128):
        rows = torch.arange(a, min(N, a + 128), device=DEV)
        L = torch.log_softmax(x[rows].to(f8), -1)
        P = L.exp()
        PL = torch.nan_to_num(P * L, nan=0.0)        # 0 * -inf of a forbidden token
        lp[rows] = L[torch.arange(len(rows), device=DEV), tok[rows]]
        ent[rows] = -PL.sum(-1)
        if top:
            tv[rows] = torch.topk(L, top, -1).values
        if case["train"]:
            gl, ge = s["g_lp"][rows, None].to(f8), s["g_ent"][rows, None].to(f8)
            hit = torch.zeros_like(P)
            hit[torch.arange(len(rows), device=DEV), tok[rows]] = 1.0
            dx[rows] = gl * (hit - P) - ge * (PL + P * ent[rows, None])
    if case["train"]:
        return lp, ent, dx
    return (lp, ent, tv, None) if top else (lp, ent)
