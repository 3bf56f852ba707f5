"""Verification of drafted tokens (ops.verify_drafts) against a 64-bit oracle, and its distribution."""
import math

import pytest
import torch

from nanovllm_b200 import ops
from nanovllm_b200.exceptions import DeviceWaitTimeout

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def probs_of(row, temp, k, top, cap):
    """Target probabilities by a sort of (logit, token) pairs, in 64 bits."""
    x = [float(v) for v in row.double()]
    x = [-math.inf if math.isnan(v) else v for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    m = x[order[0]]
    if m == -math.inf:
        return [0.0] * len(x)
    capped = (lambda v: cap * math.tanh(v / cap)) if cap else (lambda v: v)
    w = [1.0 if v == m else 0.0 if v == -math.inf else math.exp(max(-1e4, (capped(v) - capped(m)) / temp)) for v in x]
    kept = order if k <= 0 or k > len(x) else order[:k]
    if top < 1.0:
        total, mass, n = math.fsum(w[i] for i in kept), 0.0, 0
        while n < len(kept) and (n == 0 or mass < top * total):
            mass += w[kept[n]]
            n += 1
        kept = kept[:n]
    z = math.fsum(w[i] for i in kept)
    p = [0.0] * len(x)
    for i in kept:
        p[i] = w[i] / z
    return p


def oracle(s):
    cu, u, ids = s["cu_q"].tolist(), s["uniforms"].double().tolist(), s["ids"].tolist()
    V, drow, tokens, counts = s["logits"].shape[1], 0, [], []
    for b in range(len(cu) - 1):
        r0, n, out = cu[b], cu[b + 1] - cu[b], []
        if n:
            left = None
            for j in range(n):
                p = probs_of(s["logits"][r0 + j], float(s["temps"][b]), int(s["top_ks"][b]), float(s["top_ps"][b]),
                             s.get("softcap", 0.0))
                if j == n - 1:
                    left = p
                    break
                d = ids[r0 + j + 1]
                q = None if s.get("draft_probs") is None else s["draft_probs"][drow + j].double().tolist()
                if 0 <= d < V and u[r0 + j] * (1.0 if q is None else q[d]) < p[d]:
                    out.append(d)
                    continue
                left = [max(0.0, a - c) for a, c in zip(p, q)] if q else [0.0 if i == d else a for i, a in enumerate(p)]
                left = left if sum(left) > 0 else p
                break
            total, c, tok = math.fsum(left), 0.0, 0
            for i, v in enumerate(left):
                c += v
                if v > 0:
                    tok = i
                    if c > u[r0 + n - 1] * total:
                        break
            out.append(tok)
            drow += n - 1
        counts.append(len(out))
        tokens.append(out + [-1] * (s["max_q"] - len(out)))
    return tokens, counts


def make(ns, V, seed, temps=1.0, top_ks=0, top_ps=1.0, model=False, dtype=torch.float32, spread=2.0, good=0.6, ties=False):
    g = torch.Generator().manual_seed(seed)
    B, R = len(ns), sum(ns)
    x = spread * torch.randn(R, V, generator=g)
    if ties:
        x = torch.round(x)
    x = x.to(dtype)
    cu = torch.tensor([0] + ns, dtype=torch.int32).cumsum(0).int()
    ids = torch.randint(0, V, (R,), generator=g)
    vec = lambda v, t: (torch.tensor(v, dtype=t) if isinstance(v, list) else torch.full((B,), v, dtype=t))  # noqa: E731
    q = []
    for b in range(B):
        for r in range(int(cu[b]), int(cu[b + 1]) - 1):
            if model:
                q.append(torch.softmax(x[r].float() + 0.5 * torch.randn(V, generator=g), 0))
                ids[r + 1] = torch.multinomial(q[-1], 1, generator=g)
            elif torch.rand(1, generator=g) < good:
                ids[r + 1] = x[r].argmax()
    return dict(logits=x, ids=ids, cu_q=cu, max_q=max(ns + [1]), temps=vec(temps, torch.float32),
                top_ks=vec(top_ks, torch.int32), top_ps=vec(top_ps, torch.float32),
                uniforms=torch.rand(R, generator=g),
                draft_probs=(torch.stack(q) if q else torch.zeros(0, V)) if model else None)


def call(s, dev):
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    tokens, counts = ops.verify_drafts(**d)
    if dev == "cuda":
        torch.cuda.synchronize()
        ops.check_device_errors()
    return tokens.cpu().tolist(), counts.cpu().tolist()


KNOBS = [(1.0, 0, 1.0), (0.6, 0, 0.95), (1.3, 5, 1.0), (0.8, 20, 0.7), (1.0, 1, 1.0), (0.7, 0, 0.3), (2.0, 10 ** 6, 0.999)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("temp,k,top", KNOBS)
@pytest.mark.parametrize("model", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_equal_the_oracle(temp, k, top, model, dtype, dev):
    for V, seed in ((1, 0), (2, 1), (333, 2), (1000, 3)):
        s = make([1, 4, 0, 2, 7, 1, 3], V, seed, temp, k, top, model, dtype)
        assert call(s, dev) == tuple(oracle(s)), (V, seed)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mixed_requests_and_ties(dtype, dev):
    """Each sequence with its own knobs; whole-number logits, so that every cut falls among equal values."""
    n = len(KNOBS)
    s = make([3] * n, 700, 5, [t for t, _, _ in KNOBS], [k for _, k, _ in KNOBS], [p for _, _, p in KNOBS], True, dtype,
             ties=True)
    assert call(s, dev) == tuple(oracle(s))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("k,top", [(0, 1.0), (8, 0.8)])
def test_softcap(k, top, dev):
    s = dict(make([3, 1, 5], 400, 7, 0.9, k, top, True, spread=12.0), softcap=10.0)
    assert call(s, dev) == tuple(oracle(s))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("k,top", [(0, 1.0), (5, 0.8)])
def test_masks_under_a_softcap(k, top, dev):
    s = dict(make([3, 1, 4], 300, 43, 0.9, k, top, True, spread=12.0), softcap=10.0)
    s["logits"][:, ::2] = -math.inf
    s["logits"][:, 5::4] = math.nan
    s["logits"][2] = -math.inf
    assert call(s, dev) == tuple(oracle(s))


@gpu
@pytest.mark.parametrize("V", [9001, 70000, 151936])
@pytest.mark.parametrize("k,top", [(0, 0.95), (0, 0.5), (2000, 1.0), (3000, 0.9), (30, 0.9), (0, 1.0), (10 ** 5, 0.9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_and_steep_rows(V, k, top, dtype):
    """Cuts among few tokens (sorted) and among many thousand (radix select), with many equal logits, against the CPU
    restatement in 64 bits; rows with one far token, rows of few values, rows of one value."""
    s = make([3, 3, 2, 4], V, V + k, 1.0, k, top, True, dtype, spread=1.0)
    x = s["logits"]
    x[1] = x[1] * 4
    x[3, 17] = 40.0
    x[4] = torch.round(x[4])
    x[6] = 1.5
    x[8, 100:] = -50.0
    x[9] = torch.linspace(-9, 9, V).to(dtype)
    assert call(s, "cuda") == call(s, "cpu")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [40000, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_vocabulary(V, dtype, dev):
    s = make([2, 3], V, 13, [0.7, 1.0], [0, 50], [0.9, 1.0], True, dtype)
    assert call(s, dev) == tuple(oracle(s))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("knobs", [(1.0, 0, 1.0), (0.5, 3, 0.9), (1.0, 0, 0.9), (1.0, 1, 1.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_and_special_logits(knobs, dtype, dev):
    """Masks of -inf and of the type's lowest value, NaN, +inf, rows with nothing left, rows of one value."""
    ninf, low = -math.inf, torch.finfo(dtype).min
    s = make([2, 2, 2, 3, 2, 2, 1, 2], 60, 17, *knobs, model=True, dtype=dtype)
    x = s["logits"]
    x[0, 5:] = ninf
    x[1, :59] = low
    x[2] = ninf          # nothing left: the draft is refused, token 0
    x[4] = low           # all equal
    x[6, ::2] = math.nan
    x[7, 10] = math.inf
    x[8, 3] = x[8, 40] = math.inf
    x[9] = math.nan
    x[11] = 0.0
    x[11, ::3] = -0.0    # equal to 0.0
    x[13, 1:] = ninf
    assert call(s, dev) == tuple(oracle(s))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("model", [False, True])
def test_drafts_outside_the_vocabulary_are_refused(model, dev):
    s = make([4, 4, 4], 100, 19, model=model)
    s["ids"][1], s["ids"][6], s["ids"][9] = -1, 100, 2 ** 40
    got = call(s, dev)
    assert got == tuple(oracle(s)) and got[1][0] == 1


@pytest.mark.parametrize("dev", DEVICES)
def test_edges_of_the_uniforms(dev):
    """0 accepts whatever p gives, the largest uniform draws the last token with weight; also as 64-bit numbers."""
    s = make([3, 3, 1, 1], 50, 23, model=True)
    s["uniforms"][:] = torch.tensor([0.0, 0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0, 1 - 2.0 ** -24])
    s["logits"][6, :7] = -math.inf
    s["logits"][7, 44:] = -math.inf
    got = call(s, dev)
    assert got == tuple(oracle(s)) and got[1][0] == 3 and got[0][2][0] == 7 and got[0][3][0] == 43
    s["uniforms"] = s["uniforms"].double() * (1 - 2.0 ** -40)
    assert call(s, dev) == tuple(oracle(s))


@pytest.mark.parametrize("dev", DEVICES)
def test_draft_equal_to_target_is_always_accepted(dev):
    """p = q up to the rounding of q: with 32-bit q below p nothing is refused; a refusal with nothing left draws p."""
    s = make([5, 1], 64, 29, model=True)
    p = torch.softmax(s["logits"].double(), 1)
    s["draft_probs"] = (p[:4] * (1 - 1e-6)).float()
    got = call(s, dev)
    assert got[1] == [5, 1] and got == tuple(oracle(s))
    s["draft_probs"] = torch.ones(4, 64)  # every token's q is above p: nothing is left of p - q
    s["uniforms"][0] = 0.999
    got = call(s, dev)
    assert got == tuple(oracle(s)) and got[1] == [1, 1]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("model", [False, True])
def test_first_token_is_distributed_as_the_target(model, dev):
    """Over a fine grid of uniforms and all drafts weighted by q, the first emitted token has the target's
    probabilities: q(d) weighs draft d, na acceptance numbers by nd draw numbers per draft.  A grid of n midpoints
    misses an interval's length by at most 1 / n, and the two grids together by 1 / na + 1 / nd."""
    V, (na, nd) = 6, (97, 101) if dev == "cuda" else (23, 25)
    g = torch.Generator().manual_seed(31)
    x, q = torch.randn(V, generator=g), torch.softmax(1.5 * torch.randn(V, generator=g), 0)
    if not model:
        q = torch.zeros(V)
        q[2] = 1.0
    want = torch.tensor(probs_of(x, 0.8, 5, 0.97, 0.0))
    ua, ud = (torch.arange(na) + 0.5) / na, (torch.arange(nd) + 0.5) / nd
    seen = torch.zeros(V, dtype=torch.double)
    for d in [i for i in range(V) if q[i] > 0]:
        n = na * nd
        ids = torch.zeros(2 * n, dtype=torch.long)
        ids[1::2] = d
        u = torch.stack([ua.repeat_interleave(nd), ud.repeat(na)], 1).flatten()
        s = dict(logits=x.expand(2 * n, V).contiguous(), ids=ids, cu_q=torch.arange(0, 2 * n + 1, 2).int(), max_q=2,
                 temps=torch.full((n,), 0.8), top_ks=torch.full((n,), 5, dtype=torch.int32),
                 top_ps=torch.full((n,), 0.97), uniforms=u.contiguous(),
                 draft_probs=q.expand(n, V).contiguous() if model else None)
        first = torch.tensor(call(s, dev)[0])[:, 0]
        seen += float(q[d]) * torch.bincount(first, minlength=V).double() / n
    assert float((seen - want).abs().max()) <= 1 / na + 1 / nd


BAD = {
    "ids type": lambda s: dict(s, ids=s["ids"].int()),
    "ids length": lambda s: dict(s, ids=s["ids"][:-1]),
    "cu_q type": lambda s: dict(s, cu_q=s["cu_q"].long()),
    "temps": lambda s: dict(s, temps=s["temps"][:1]),
    "top_ks": lambda s: dict(s, top_ks=s["top_ks"].long()),
    "top_ps": lambda s: dict(s, top_ps=s["top_ps"].double()),
    "uniforms": lambda s: dict(s, uniforms=s["uniforms"].half()),
    "logits type": lambda s: dict(s, logits=s["logits"].half()),
    "probs type": lambda s: dict(s, draft_probs=s["draft_probs"].bfloat16()),
    "probs width": lambda s: dict(s, draft_probs=s["draft_probs"][:, :-1].contiguous()),
    "max_q": lambda s: dict(s, max_q=0),
    "softcap": lambda s: dict(s, softcap=-1.0),
    "vocabulary": lambda s: dict(s, logits=torch.zeros(s["logits"].shape[0], (1 << 20) + 1), draft_probs=None),
}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what", sorted(BAD))
def test_refusals(what, dev):
    with pytest.raises(RuntimeError):
        call(BAD[what](make([3, 2], 40, 1, model=True)), dev)


@gpu
def test_bad_values_on_the_device_are_reported():
    for change in (dict(max_q=2), dict(cu_q=torch.tensor([0, 3, 99], dtype=torch.int32)),
                   dict(draft_probs=torch.zeros(1, 40))):
        s = dict(make([3, 2], 40, 1, model=True), **change)
        d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        ops.error_word(torch.device("cuda")).zero_()
        ops.verify_drafts(**d)
        torch.cuda.synchronize()
        with pytest.raises(DeviceWaitTimeout):
            ops.check_device_errors()


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_logits_and_rows_behind_the_last_sequence(dev):
    s = make([2, 3, 1], 333, 37, 0.9, 0, 0.9, True, torch.bfloat16)
    wide = torch.full((9, 340), float("nan"), dtype=torch.bfloat16)
    wide[:6, 3:336] = s["logits"]
    probs = torch.full((5, 340), float("nan"))
    probs[:3, 1:334] = s["draft_probs"]
    t = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    t.update(logits=wide.to(dev)[:, 3:336], draft_probs=probs.to(dev)[:, 1:334])
    t["ids"] = torch.cat([t["ids"], t["ids"][:3]])
    t["uniforms"] = torch.cat([t["uniforms"], t["uniforms"][:3]])
    assert call(t, dev) == tuple(oracle(s))


@gpu
def test_streams_and_graphs():
    """Calls at once on two streams and captured graphs replayed together give the single call's tokens."""
    cases = [make([4] * 12, 30000, i, 0.8, 0, 0.95, True, torch.bfloat16) for i in range(2)]
    dev = [{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()} for s in cases]
    want = [ops.verify_drafts(**d) for d in dev]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in dev], [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.verify_drafts(**dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i][0]) and torch.equal(c, want[i][1]) for t, c in got[i])
    graphs, outs = [], []
    for d in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.verify_drafts(**d))
        graphs.append(g)
    for _ in range(5):
        for t, c in outs:
            t.fill_(7)
            c.fill_(7)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]) for o, w in zip(outs, want))
    ops.check_device_errors()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread,shift", [(1e-3, 0.0), (3.0, -40.0), (300.0, 0.0), (1e30, 0.0)])
def test_cuts_far_below_the_largest(spread, shift, dtype, dev):
    """Cuts beyond any list of the largest, at tiny, negative and huge logits, by count, by mass and by both."""
    for k, top in ((900, 1.0), (1999, 1.0), (0, 0.9), (0, 0.999999), (1200, 0.97)):
        s = make([2, 3, 1, 2], 2000, 71, 1.0, k, top, False, dtype, spread=spread)
        s["logits"] = (s["logits"].float() + shift).to(dtype)
        s["logits"][0, 17] = s["logits"][0].max() * 4  # one far above: the bins below it start there
        s["logits"][3] = s["logits"][3].abs().neg()
        assert call(s, dev) == tuple(oracle(s)), (k, top)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("top", [1.0, 0.9])
def test_drafts_beyond_32_bits_are_no_token(top, dev):
    """Such an id is refused, and no token of the vocabulary stands in for it in what is drawn from."""
    V = 40
    s = make([2] * 60, V, 73, 1.0, 0, top, spread=0.5)
    s["ids"][1::2] = s["logits"][::2].argmax(1) + 2 ** 32
    got = call(s, dev)
    assert got == tuple(oracle(s)) and all(c == 1 for c in got[1])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("model", [False, True])
def test_draws_from_short_lists(model, dev):
    """One to a few hundred kept tokens, refused drafts inside and outside the kept set, nothing left of p - q."""
    for k, seed in ((1, 81), (2, 82), (31, 83), (64, 84)):
        s = make([3, 1, 2, 5, 2], 1500, seed, 0.8, k, 0.9, model, torch.bfloat16, good=0.3)
        assert call(s, dev) == tuple(oracle(s)), k
    if model:
        s = make([2, 2, 2], 600, 85, 1.0, 40, 1.0, True, torch.bfloat16)
        s["draft_probs"][:] = 1.0  # more than p everywhere: the probabilities themselves
        s["uniforms"][::2] = 0.999
        assert call(s, dev) == tuple(oracle(s))


@gpu
@pytest.mark.parametrize("cu", [[0, 10, 2, 12], [0, 3, 1, 12], [5, 3, 12, 12], [0, 2, 0, 2, 0, 2]])
def test_overlapping_sequences_are_reported(cu):
    """cu_q that falls: the call reports it; what it writes stays inside its outputs."""
    s = make([3, 4, 5], 900, 91, 0.8, 20, 0.9, True, torch.bfloat16)
    s["cu_q"], s["max_q"] = torch.tensor(cu, dtype=torch.int32), 12
    for k in ("temps", "top_ks", "top_ps"):
        s[k] = s[k][:1].expand(len(cu) - 1).contiguous()
    with pytest.raises(DeviceWaitTimeout):
        call(s, "cuda")
    s = make([3, 4, 5], 900, 91, 0.8, 20, 0.9, True, torch.bfloat16)
    assert call(s, "cuda") == tuple(oracle(s))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("equal,top", [(2, 0.5), (4, 0.25), (4, 0.75), (8, 0.5)])
@pytest.mark.parametrize("gap", [30.0, 24.0, 60.0])
def test_top_p_at_the_edge_of_equal_logits(gap, equal, top, dev):
    """Equal largest logits and next to nothing else: top_p falls on the sum of some of them but for that rest, which
    decides whether one more is kept (gap 60: 1e-23 of the mass, none in 64 bits either)."""
    g = torch.Generator().manual_seed(97)
    s = make([1] * 24, 4000, 97, 1.0, 0, top, dtype=torch.bfloat16)
    x = torch.full((24, 4000), -gap)
    x.scatter_(1, torch.stack([torch.randperm(4000, generator=g)[:equal] for _ in range(24)]), 0.0)
    s["logits"] = x.bfloat16()
    assert call(s, dev) == tuple(oracle(s))
