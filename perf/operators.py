"""Workloads of the serving operators for batches that share a prompt prefix and for drafted tokens.

``shared_prefix_attention``: paged attention of a decode batch whose sequences all begin with the same long prefix
(a system prompt held once in the prefix cache), one or several query tokens per sequence.  ``verify_drafts``:
acceptance of drafted tokens against the target's probabilities, and the draw of the token that follows them.

``run`` computes a case either with plain torch operations (``own`` false) or with the framework's entry points.
Head layouts and vocabularies are those of the model shapes that ``bench.py`` builds.
"""
import math

import torch

own = False

PAGE = 256  # the engine's default page size

# (query heads, key/value heads, head dim, sliding window) of the model shapes in bench.py; gemma3 has window layers
# and global layers
HEADS = {
    "qwen3": (32, 8, 128, 0),
    "lfm2": (32, 8, 64, 0),
    "gemma3": (4, 1, 256, 0),
    "gemma3-window": (4, 1, 256, 512),
}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    att = {"op": "attention", "softcap": 0.0}
    ver = {"op": "verify", "softcap": 0.0}
    return [
        # four chats on a short system prompt, right after their first token: the call's latency
        dict(att, name="attn few chats", heads="qwen3", batch=4, prefix=256, own_min=1, own_max=64, q_min=1, q_max=1),
        # a usual batch on a tool-use prompt; own parts of a short question and the reply so far
        dict(att, name="attn batch", heads="qwen3", batch=32, prefix=2048, own_min=32, own_max=512, q_min=1, q_max=1),
        # the benchmark's 128 requests, all on one long document
        dict(att, name="attn long document", heads="qwen3", batch=128, prefix=8192, own_min=64, own_max=1024, q_min=1,
             q_max=1),
        # the same kind of batch with up to four drafted tokens for each request
        dict(att, name="attn drafts", heads="qwen3", batch=64, prefix=4096, own_min=32, own_max=512, q_min=1, q_max=5),
        # sliding-window layers, a prefix that ends inside a page
        dict(att, name="attn window", heads="gemma3-window", batch=64, prefix=1001, own_min=1, own_max=700, q_min=1,
             q_max=1),
        # narrow heads, short drafts, a very long shared prefix
        dict(att, name="attn narrow heads", heads="lfm2", batch=96, prefix=16000, own_min=16, own_max=300, q_min=1,
             q_max=3),
        # one chat whose drafts are looked up in its own text (no draft distribution): latency
        dict(ver, name="verify one chat", batch=1, vocab=151936, drafts_min=4, drafts_max=4, draft="lookup",
             temp=0.6, top_k=0, top_p=0.95, wide=False),
        # a usual batch with a draft model, the sampling defaults
        dict(ver, name="verify batch", batch=32, vocab=151936, drafts_min=0, drafts_max=4, draft="model", temp=0.6,
             top_k=0, top_p=0.95, wide=False),
        # the largest batch, plain temperature sampling
        dict(ver, name="verify large", batch=128, vocab=151936, drafts_min=3, drafts_max=5, draft="model", temp=1.0,
             top_k=0, top_p=1.0, wide=False),
        # greedy requests on a small vocabulary
        dict(ver, name="verify greedy", batch=48, vocab=65536, drafts_min=0, drafts_max=7, draft="lookup", temp=1.0,
             top_k=1, top_p=1.0, wide=False),
        # a large vocabulary, soft-capped 32-bit logits, top-k and top-p together
        dict(ver, name="verify capped top-k", batch=24, vocab=262144, drafts_min=1, drafts_max=3, draft="model",
             temp=0.7, top_k=64, top_p=0.9, wide=True, softcap=30.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        q_max = rng.choice([1, 1, 2, 3, 5, 8])
        heads = rng.choice(sorted(HEADS))
        batch = _log_int(rng, 1, 128)
        prefix = _log_int(rng, 64, 16384)
        # keep the score work at most that of the largest listed case
        while batch * q_max * prefix * HEADS[heads][0] > 128 * 8192 * 32:
            prefix = prefix // 2 + rng.randrange(7)
        own_min = _log_int(rng, 1, 64)
        return {"op": "attention", "heads": heads, "batch": batch, "prefix": prefix, "own_min": own_min,
                "own_max": own_min + _log_int(rng, 1, 900), "q_min": 1, "q_max": q_max,
                "softcap": rng.choice([0.0, 0.0, 0.0, 50.0])}
    drafts_max = rng.choice([1, 2, 3, 4, 5, 7])
    vocab = rng.choice([65536, 151936, 262144, _log_int(rng, 2000, 262144)])
    batch = _log_int(rng, 1, 128)
    while batch * (drafts_max + 1) * vocab > 128 * 5 * 151936:
        batch = batch // 2 + 1
    return {"op": "verify", "batch": batch, "vocab": vocab, "drafts_min": rng.randrange(drafts_max + 1),
            "drafts_max": drafts_max, "draft": rng.choice(["model", "lookup"]),
            "temp": round(rng.uniform(0.3, 1.2), 2), "top_k": rng.choice([0, 0, 1, 20, 64]),
            "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]), "wide": rng.random() < 0.3,
            "softcap": rng.choice([0.0, 0.0, 30.0])}


def _lengths(case):
    """Query tokens and own keys of each sequence: plain functions of the case, so that work() knows them too.
    They run evenly from the smallest to the largest, in a mixed order."""
    n = case["batch"]

    def spread(lo, hi, step):
        return [lo + (hi - lo) * ((i * step) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]

    step = next(s for s in (37, 41, 43, 47) if math.gcd(s, n) == 1)
    if case["op"] == "verify":
        return [d + 1 for d in spread(case["drafts_min"], case["drafts_max"], step)], None
    qs = spread(case["q_min"], case["q_max"], 1 if n < 3 else step)
    owns = [max(o, q) for o, q in zip(spread(case["own_min"], case["own_max"], step), qs)]
    return qs, owns


# ------------------------------------------------------------------------------------------------ inputs
def _prepare_attention(case, g):
    nq, nkv, hd, window = HEADS[case["heads"]]
    qs, owns = _lengths(case)
    B, P = case["batch"], case["prefix"]
    np_ = -(-P // PAGE)
    shared = P // PAGE  # pages that a sequence's own keys do not reach into
    need = [-(-(P + o) // PAGE) - shared for o in owns]
    NB = np_ + sum(need)
    dev = "cuda"
    kc = torch.randn(NB, nkv, PAGE, hd, device=dev, generator=g).bfloat16()
    vc = torch.randn(NB, nkv, PAGE, hd, device=dev, generator=g).bfloat16()
    perm = torch.randperm(NB, device=dev, generator=g).int().cpu()
    prefix_blocks = perm[:np_]
    bt = torch.zeros(B, shared + max(need), dtype=torch.int32)
    bt[:, :shared] = prefix_blocks[:shared]
    at = np_
    for b in range(B):
        bt[b, shared:shared + need[b]] = perm[at:at + need[b]]
        at += need[b]
    T = sum(qs)
    q = (1.5 * torch.randn(T, nq, hd, device=dev, generator=g)).bfloat16()
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(qs).cumsum(0)
    ctx = torch.tensor([P + o for o in owns], dtype=torch.int32)
    return {"op": "attention", "q": q, "kc": kc, "vc": vc, "prefix_blocks": prefix_blocks.to(dev), "prefix": P,
            "bt": bt.to(dev), "ctx": ctx.to(dev), "cu": cu.to(dev) if case["q_max"] > 1 else None,
            "max_q": max(qs), "max_len": P + max(owns), "scale": hd ** -0.5, "softcap": case["softcap"],
            "window": window}


def _prepare_verify(case, g):
    ns, _ = _lengths(case)
    B, V, R, dev = case["batch"], case["vocab"], sum(ns), "cuda"
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(ns).cumsum(0)
    # a wide bell of unlikely tokens and a few dozen likely ones, as a language model's logits are
    x = 2.0 * torch.randn(R, V, device=dev, generator=g)
    likely = torch.randint(0, V, (R, 40), device=dev, generator=g)
    lift = 9.0 + 2.5 * torch.randn(R, 40, device=dev, generator=g).abs() + 2.0 * torch.randn(R, 1, device=dev, generator=g)
    x.scatter_(1, likely, lift)
    logits = x if case["wide"] else x.bfloat16()
    last = torch.zeros(R, dtype=torch.bool)
    last[(cu[1:] - 1).long()] = True
    rows = (~last).nonzero().flatten().to(dev)  # rows that a drafted token is held against
    ids = torch.randint(0, V, (R,), device=dev, generator=g)
    probs = None
    if case["draft"] == "model":
        # the drafter's own distribution: near the target's, drawn from at the request's temperature
        d = logits[rows].float()
        for lo in range(0, d.shape[0], 64):
            part = d[lo:lo + 64]
            part += 0.7 * torch.randn(part.shape, device=dev, generator=g)
            part.copy_(torch.softmax(part / case["temp"], dim=1))
        probs = d
        race = torch.empty(64, V, device=dev)
        drafts = torch.cat([(probs[lo:lo + 64] / race[:min(64, probs.shape[0] - lo)].exponential_(generator=g))
                            .argmax(1) for lo in range(0, probs.shape[0], 64)]) if probs.shape[0] else ids[:0]
    else:
        best = logits[rows].float().argmax(1) if rows.numel() else ids[:0]
        other = torch.randint(0, V, best.shape, device=dev, generator=g)
        drafts = torch.where(torch.rand(best.shape, device=dev, generator=g) < 0.75, best, other)
    ids[rows + 1] = drafts
    full = lambda v, t: torch.full((B,), v, dtype=t, device=dev)  # noqa: E731
    return {"op": "verify", "logits": logits, "ids": ids, "cu": cu.to(dev), "max_q": max(ns),
            "temps": full(case["temp"], torch.float32), "top_ks": full(case["top_k"], torch.int32),
            "top_ps": full(case["top_p"], torch.float32),
            "uniforms": torch.rand(R, device=dev, generator=g), "probs": probs, "softcap": case["softcap"],
            "cut": case["top_k"] > 0 or case["top_p"] < 1.0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_attention(case, g) if case["op"] == "attention" else _prepare_verify(case, g)


# ------------------------------------------------------------------------------------------------ plain forms
def _attention_plain(s):
    q, kc, vc, P, window = s["q"].float(), s["kc"], s["vc"], s["prefix"], s["window"]
    T, nq, hd = q.shape
    nkv = kc.shape[1]
    G = nq // nkv
    dev, ctx, B = q.device, s["ctx"].long(), s["ctx"].numel()
    cu = torch.arange(B + 1, device=dev) if s["cu"] is None else s["cu"].long()
    n, Q, L = cu[1:] - cu[:-1], s["max_q"], s["max_len"] - P
    # query tokens in a padded grid [B, Q]; a padded place holds token 0 and is dropped at the end
    j = torch.arange(Q, device=dev)
    real = j[None] < n[:, None]
    tok = torch.where(real, cu[:-1, None] + j[None], 0)
    pos = ctx[:, None] - n[:, None] + j[None]
    qp = q[tok].view(B, Q, nkv, G, hd)
    kp = kc[s["prefix_blocks"].long()].permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :P].float()
    vp = vc[s["prefix_blocks"].long()].permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :P].float()
    key = P + torch.arange(L, device=dev)
    page = s["bt"].long()[:, (key // PAGE).clamp(max=s["bt"].shape[1] - 1)]
    ks = kc[page, :, (key % PAGE)[None]].float()  # [B, L, nkv, hd]
    vs = vc[page, :, (key % PAGE)[None]].float()
    s1 = torch.einsum("bqkgd,kpd->bqkgp", qp, kp) * s["scale"]
    s2 = torch.einsum("bqkgd,blkd->bqkgl", qp, ks) * s["scale"]
    if s["softcap"] > 0:
        s1, s2 = s["softcap"] * torch.tanh(s1 / s["softcap"]), s["softcap"] * torch.tanh(s2 / s["softcap"])

    def seen(keys):
        m = keys[None, None] <= pos[:, :, None]
        return m & (keys[None, None] > pos[:, :, None] - window) if window > 0 else m

    s1.masked_fill_(~seen(torch.arange(P, device=dev))[:, :, None, None], -math.inf)
    s2.masked_fill_(~seen(key)[:, :, None, None], -math.inf)
    m = torch.maximum(s1.amax(-1), s2.amax(-1)).unsqueeze(-1)
    e1, e2 = torch.exp(s1 - m), torch.exp(s2 - m)
    z = e1.sum(-1, keepdim=True) + e2.sum(-1, keepdim=True)
    o = (torch.einsum("bqkgp,kpd->bqkgd", e1, vp) + torch.einsum("bqkgl,blkd->bqkgd", e2, vs)) / z
    return o.reshape(B, Q, nq, hd)[real].to(s["q"].dtype)


def _target_probs(s, rows, seq):
    """Probabilities [len(rows), V] in 64 bits of the target's rows after temperature, top-k and top-p."""
    raw = s["logits"][rows]
    V = raw.shape[1]
    x = raw.double()
    if s["softcap"] > 0:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    p = torch.exp((x - x.amax(1, keepdim=True)) / s["temps"][seq].double()[:, None])
    del x
    k, top = s["top_ks"][seq].long(), s["top_ps"][seq].double()
    if not s["cut"]:
        return p / p.sum(1, keepdim=True)
    order = torch.sort(raw, dim=1, descending=True, stable=True).indices  # equal logits: lowest token first
    ps = p.gather(1, order)
    k = torch.where((k <= 0) | (k > V), V, k)
    ps *= torch.arange(V, device=p.device)[None] < k[:, None]
    before = torch.cumsum(ps, 1) - ps
    keep = (before < (top * ps.sum(1))[:, None]) | (top >= 1.0)[:, None]
    keep[:, 0] = True
    ps *= keep
    p.scatter_(1, order, ps)
    return p / p.sum(1, keepdim=True)


def _verify_plain(s):
    cu, B, Q = s["cu"].long(), s["temps"].numel(), s["max_q"]
    dev, n = cu.device, cu[1:] - cu[:-1]
    R, V = s["logits"].shape
    row = torch.arange(R, device=dev)
    seq = torch.bucketize(row, cu[1:], right=True)
    p = _target_probs(s, row, seq)
    u = s["uniforms"].double()
    # acceptance of the drafts, row by row
    last = row + 1 == cu[seq + 1]
    draft = s["ids"][(row + 1).clamp(max=R - 1)]
    drow = row - seq  # one draft row fewer than rows for each sequence before
    pd = p.gather(1, draft[:, None])[:, 0]
    if s["probs"] is None:
        qd = torch.ones_like(pd)
    else:
        qd = s["probs"][drow.clamp(max=max(0, s["probs"].shape[0] - 1)), draft].double() if s["probs"].shape[0] else pd
    ok = (u * qd < pd) & ~last
    j = torch.arange(Q, device=dev)
    grid = (cu[:-1, None] + j[None]).clamp(max=R - 1)
    run_ok = torch.cumprod((ok[grid] & (j[None] < n[:, None] - 1)).long(), 1)
    acc = run_ok.sum(1)  # accepted drafts of each sequence
    at = cu[:-1] + acc  # the row that the next token is drawn from
    pr = p[at]
    res = pr.clone()
    rejected = acc < n - 1
    if s["probs"] is None:
        d = draft[at][:, None]
        res.scatter_(1, d, torch.where(rejected[:, None], 0.0, res.gather(1, d)))
    elif s["probs"].shape[0]:
        qrow = s["probs"][(at - torch.arange(B, device=dev)).clamp(max=s["probs"].shape[0] - 1)].double()
        res = torch.where(rejected[:, None], (pr - qrow).clamp(min=0.0), pr)
    tot = res.sum(1, keepdim=True)
    res = torch.where(tot > 0, res, pr)
    cum = torch.cumsum(res, 1)
    want = u[cu[1:] - 1][:, None] * cum[:, -1:]
    tok = (cum > want).int().argmax(1)
    out = torch.where(j[None] < acc[:, None], s["ids"][(grid + 1).clamp(max=R - 1)], -1)
    out = torch.where(j[None] == acc[:, None], tok[:, None], out)
    return {"tokens": out, "counts": (acc + 1).int()}


def run(state):
    s = state
    if own:
        from nanovllm_b200 import ops
        if s["op"] == "attention":
            return ops.shared_prefix_attention(s["q"], s["kc"], s["vc"], s["prefix_blocks"], s["prefix"], s["bt"],
                                               s["ctx"], s["scale"], softcap=s["softcap"], window=s["window"],
                                               cu_q=s["cu"], max_q=s["max_q"], max_len=s["max_len"])
        tokens, counts = ops.verify_drafts(s["logits"], s["ids"], s["cu"], s["max_q"], s["temps"], s["top_ks"],
                                           s["top_ps"], s["uniforms"], draft_probs=s["probs"], softcap=s["softcap"])
        return {"tokens": tokens, "counts": counts}
    return _attention_plain(s) if s["op"] == "attention" else _verify_plain(s)


# ------------------------------------------------------------------------------------------------ work, exact values
def work(case):
    qs, owns = _lengths(case)
    if case["op"] == "attention":
        nq, nkv, hd, window = HEADS[case["heads"]]
        P, T = case["prefix"], sum(qs)
        pairs, keys, first = 0, 0, P
        for n, o in zip(qs, owns):
            lo = max(0, P + o - n + 1 - window) if window else 0  # first key that the sequence's first token sees
            first = min(first, lo)
            keys += P + o - max(P, lo)
            for i in range(n):
                end = P + o - n + i + 1
                pairs += end - (max(0, end - window) if window else 0)
        keys += P - first
        return {"bytes": 2 * (2 * keys * nkv * hd + 2 * T * nq * hd), "flops": 4 * pairs * nq * hd}
    # the target's rows once; of the draft's rows the one that the residual is taken from
    V, R = case["vocab"], sum(qs)
    b = R * V * (4 if case["wide"] else 2)
    if case["draft"] == "model":
        b += 4 * V * sum(1 for n in qs if n > 1)
    return {"bytes": b + 24 * R, "flops": 4 * R * V}


def _exact_attention(s):
    q, out = s["q"].double(), []
    nkv, nq, hd = s["kc"].shape[1], q.shape[1], q.shape[2]
    ctx, B = s["ctx"].tolist(), s["ctx"].numel()
    cu = list(range(B + 1)) if s["cu"] is None else s["cu"].tolist()
    head = torch.arange(nq, device=q.device) // (nq // nkv)
    for b in range(B):
        at = torch.arange(ctx[b], device=q.device)
        page = torch.where(at < s["prefix"], s["prefix_blocks"][(at // PAGE).clamp(max=s["prefix_blocks"].numel() - 1)],
                           s["bt"][b, at // PAGE]).long()
        k, v = (c[page, :, at % PAGE].double()[:, head] for c in (s["kc"], s["vc"]))
        for t in range(cu[b], cu[b + 1]):
            end = ctx[b] - (cu[b + 1] - 1 - t)
            lo = max(0, end - s["window"]) if s["window"] else 0
            x = (k[lo:end] * q[t]).sum(-1) * s["scale"]
            if s["softcap"]:
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            w = torch.softmax(x, 0)
            out.append((w[:, :, None] * v[lo:end]).sum(0))
    return torch.stack(out)


def _exact_verify(s):
    cu, u, ids = s["cu"].tolist(), s["uniforms"].double().tolist(), s["ids"].tolist()
    B, V = len(cu) - 1, s["logits"].shape[1]
    T, K, TP = s["temps"].tolist(), s["top_ks"].tolist(), s["top_ps"].tolist()
    tokens, counts, drow = torch.full((B, s["max_q"]), -1), [], 0
    for b in range(B):
        n, got = cu[b + 1] - cu[b], 0
        while True:
            r = cu[b] + got
            raw = s["logits"][r]
            x = raw.double()
            if s["softcap"]:
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            p = torch.softmax(x / T[b], 0)
            if 0 < K[b] < V or TP[b] < 1:
                idx = torch.sort(raw, descending=True, stable=True).indices
                idx = idx[:K[b]] if 0 < K[b] < V else idx
                c = torch.cumsum(p[idx], 0)
                m = max(1, int((c - p[idx] < TP[b] * c[-1]).sum())) if TP[b] < 1 else idx.numel()
                p = torch.zeros_like(p).index_copy(0, idx[:m], p[idx[:m]])
                p = p / p.sum()
            if got == n - 1:
                break
            d = ids[r + 1]
            qrow = None if s["probs"] is None else s["probs"][drow + got].double()
            if u[r] * (1.0 if qrow is None else float(qrow[d])) < float(p[d]):
                tokens[b, got] = d
                got += 1
                continue
            left = p.clone()
            if qrow is None:
                left[d] = 0
            else:
                left = torch.clamp(p - qrow, min=0)
            p = left if float(left.sum()) > 0 else p
            break
        c = torch.cumsum(p, 0)
        tokens[b, got] = int(torch.searchsorted(c, u[cu[b + 1] - 1] * c[-1], right=True))
        counts.append(got + 1)
        drow += max(0, n - 1)
    return {"tokens": tokens, "counts": torch.tensor(counts, dtype=torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attention(s) if s["op"] == "attention" else _exact_verify(s)
