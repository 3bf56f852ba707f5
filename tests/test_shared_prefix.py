"""Attention of a decode batch on a shared prefix (ops.shared_prefix_attention) against a 64-bit oracle."""

import pytest
import torch

from nanovllm_b200 import ops
from nanovllm_b200.exceptions import DeviceWaitTimeout

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BS = 256


def make(prefix, owns, qs, nq, nkv, hd, seed=0, amp=1.0, bs=BS, spare=2, poison=True):
    """A cache with scattered pages.  ``owns[b]``: keys of sequence b behind the prefix (negative: a sequence that is
    shorter than the prefix).  With ``poison`` every cache slot that no sequence owns holds NaN or infinity."""
    g = torch.Generator().manual_seed(seed)
    B = len(owns)
    ctx = [prefix + o for o in owns]
    np_ = -(-prefix // bs)
    whole = prefix // bs
    need = [max(0, -(-n // bs) - whole) if n > prefix else 0 for n in ctx]
    NB = np_ + sum(need) + spare
    kc = torch.full((NB, nkv, bs, hd), float("nan")).bfloat16() if poison else torch.zeros(NB, nkv, bs, hd).bfloat16()
    vc = kc.clone()
    if poison:
        vc[:, :, ::2] = float("inf")
    perm = torch.randperm(NB, generator=g).tolist()
    pre = perm[:np_]
    bt = torch.full((B, max(1, whole + max(need))), 10 ** 9, dtype=torch.int32)  # entries that are not to be read
    at = np_

    def fill(page, lo, hi):
        for c in (kc, vc):
            c[page, :, lo:hi] = (torch.randn(nkv, hi - lo, hd, generator=g) * amp).bfloat16()

    for i, p in enumerate(pre):
        fill(p, 0, min(bs, prefix - i * bs))
    for b in range(B):
        for i in range(need[b]):
            page, first = perm[at], (whole + i) * bs
            bt[b, whole + i] = page
            lo, hi = max(0, prefix - first), min(bs, ctx[b] - first)
            if hi > lo:
                fill(page, lo, hi)
            at += 1
    T = sum(qs)
    q = (torch.randn(T, nq, hd, generator=g) * amp).bfloat16()
    cu = torch.tensor([0] + qs, dtype=torch.int32).cumsum(0).int()
    return dict(q=q, k_cache=kc, v_cache=vc, prefix_blocks=torch.tensor(pre, dtype=torch.int32), prefix_len=prefix,
                block_tables=bt, ctx_lens=torch.tensor(ctx, dtype=torch.int32), cu_q=cu, max_q=max(qs + [1]))


def oracle(s, scale, softcap=0.0, window=0):
    """(o, sum p |v|) in 64 bits, key by key list of each sequence."""
    q, bs = s["q"].double(), s["k_cache"].shape[2]
    T, nq, hd = q.shape
    nkv = s["k_cache"].shape[1]
    o, a = torch.zeros(T, nq, hd, dtype=torch.double), torch.zeros(T, nq, hd, dtype=torch.double)
    for b, n in enumerate(s["ctx_lens"].tolist()):
        t0, t1 = int(s["cu_q"][b]), int(s["cu_q"][b + 1])
        if t1 == t0 or n <= 0:
            continue
        pages = [int(s["prefix_blocks"][j // bs]) if j < s["prefix_len"] else int(s["block_tables"][b, j // bs])
                 for j in range(n)]
        at = (torch.tensor(pages), slice(None), torch.arange(n) % bs)
        keys, values = (s[c][at].double().repeat_interleave(nq // nkv, 1) for c in ("k_cache", "v_cache"))
        for t in range(t0, t1):
            pos = n - (t1 - t0) + t - t0
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            k, v = keys[lo:pos + 1], values[lo:pos + 1]
            x = torch.einsum("hd,khd->hk", q[t], k) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            p = torch.softmax(x, 1)
            o[t], a[t] = torch.einsum("hk,khd->hd", p, v), torch.einsum("hk,khd->hd", p, v.abs())
    return o, a


def check(got, s, scale, softcap=0.0, window=0):
    """The output is rounded to bf16 once (2^-8 |o|) and each weight may be (2^-8 of sum p |v|); scores and sums in 32
    bits add far less than 2^-10 of sum p |v| at these sizes (|score| < 64, at most 2^-14 off)."""
    o, a = oracle(s, scale, softcap, window)
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10) * a
    err = (got.double().cpu() - o).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol + 1e-30).all()), f"max error over tolerance: {(err / (tol + 1e-30)).max().item():.3g}"


def call(s, dev, scale, **kw):
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    d.update(kw)
    out = ops.shared_prefix_attention(scale=scale, **d)
    if dev == "cuda":
        torch.cuda.synchronize()
        ops.check_device_errors()
    return out


LAYOUTS = [(32, 8, 128), (8, 8, 64), (4, 1, 256), (6, 2, 128), (24, 1, 64), (16, 8, 64), (4, 2, 512), (5, 5, 96)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,hd", LAYOUTS)
def test_one_token_per_sequence(nq, nkv, hd, dev):
    owns = [1, 2, 63, 64, 65, 200, 257, 5]
    s = make(320, owns, [1] * len(owns), nq, nkv, hd, seed=hd + nq)
    got = call(s, dev, hd ** -0.5, cu_q=None)
    check(got, s, hd ** -0.5)
    assert torch.equal(got, call(s, dev, hd ** -0.5))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 256, 511, 1030])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 1, 256), (4, 4, 64), (2, 1, 512)])
def test_prefix_lengths_with_several_tokens(prefix, nq, nkv, hd, dev):
    """Prefixes that end anywhere in a page or tile; sequences of 0 to 9 query tokens."""
    qs = [1, 4, 0, 9, 2]
    s = make(prefix, [1, 70, 30, 9, 129], qs, nq, nkv, hd, seed=prefix + hd)
    check(call(s, dev, hd ** -0.5), s, hd ** -0.5)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (100, 0.0), (400, 0.0), (0, 20.0), (300, 5.0)])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 1, 256), (8, 4, 64), (3, 1, 48)])
def test_window_and_softcap(window, softcap, nq, nkv, hd, dev):
    s = make(500, [1, 3, 200, 600, 40], [1, 3, 1, 5, 2], nq, nkv, hd, seed=window, amp=2.0)
    check(call(s, dev, hd ** -0.5, window=window, softcap=softcap), s, hd ** -0.5, softcap, window)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 1, 256), (4, 4, 64), (2, 1, 512)])
def test_sequences_shorter_than_the_prefix(nq, nkv, hd, dev):
    """Contexts inside the prefix, of one key, of none (zeros), and with fewer keys than query tokens."""
    s = make(300, [-1, -299, -300, 20, -298, -150], [1, 1, 1, 2, 4, 3], nq, nkv, hd, seed=5)
    got = call(s, dev, hd ** -0.5)
    check(got, s, hd ** -0.5)
    assert bool((got[2] == 0).all()) and bool((got[5:7] == 0).all())


@gpu
@pytest.mark.parametrize("rows", [17, 32, 33, 64, 65, 150])
@pytest.mark.parametrize("prefix", [1, 127, 128, 129, 700, 1536])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 1, 64), (4, 1, 256)])
def test_many_rows(rows, prefix, nq, nkv, hd):
    """Batches that fill one or several tiles of query rows against the prefix; uneven numbers of query tokens."""
    qs, n = [], 0
    while n < rows:
        qs.append(min(rows - n, (0, 1, 3, 2, 1, 5)[len(qs) % 6]))
        n += qs[-1]
    owns = [q + (0, 7, 64, 130)[i % 4] for i, q in enumerate(qs)]
    s = make(prefix, owns, qs, nq, nkv, hd, seed=rows + prefix)
    check(call(s, "cuda", hd ** -0.5), s, hd ** -0.5)


@gpu
@pytest.mark.parametrize("window,softcap,amp,scale", [(90, 0.0, 1.0, 0.1), (600, 0.0, 1.0, 0.1), (0, 15.0, 3.0, 0.1),
                                                      (0, 0.0, 3.0, 0.1), (0, 0.0, 1.0, -0.1), (0, 0.0, 1.0, 0.0)])
@pytest.mark.parametrize("batch", [30, 80])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (8, 2, 64), (4, 1, 256)])
def test_many_rows_masks_and_scales(window, softcap, amp, scale, batch, nq, nkv, hd):
    """Windows that leave rows without a key of the prefix, contexts inside it, soft-caps, moving maxima, any scale."""
    owns = [(1, 5, 700, 64, -300, -899, -900)[i % 7] for i in range(batch)]
    s = make(900, owns, [1] * batch, nq, nkv, hd, seed=batch, amp=amp)
    check(call(s, "cuda", scale, window=window, softcap=softcap), s, scale, softcap, window)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("step", [3, 7, 32, 45, 128])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 2, 64), (4, 1, 256)])
def test_rising_scores(step, nq, nkv, hd, dev):
    """Scores that grow by 6.5 (9.4 powers of two) every few keys while the values shrink as much, so that every key keeps
    its share of the output through each move of the maximum."""
    s = make(512, [40] * 40, [1, 3] * 20, nq, nkv, hd, seed=step, spare=0)
    s["q"].zero_()[..., 0] = 1.0
    s["q"][::3, :, 0] = 0.5
    level = (torch.arange(512) // step).clamp(max=9).float()
    for i, p in enumerate(s["prefix_blocks"].tolist()):
        own = level[i * BS:(i + 1) * BS]
        s["k_cache"][p] = 0.0
        s["k_cache"][p, :, :, 0] = (6.5 * own).bfloat16()
        s["v_cache"][p] = (s["v_cache"][p].float() * torch.exp(-6.5 * own)[None, :, None]).bfloat16()
    check(call(s, dev, 1.0), s, 1.0)


@pytest.mark.parametrize("dev", DEVICES)
def test_large_scores(dev):
    """Scores spread over tens of units: the running maximum moves from tile to tile."""
    s = make(700, [300, 10], [1, 3], 8, 2, 128, seed=9, amp=3.0)
    check(call(s, dev, 128 ** -0.5), s, 128 ** -0.5)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hd", [128, 512])
def test_strides_out_and_rows_behind_the_last_sequence(hd, dev):
    qs, nq, nkv = [2, 1, 3], 4, 2
    s = make(256, [3, 1, 70], qs, nq, nkv, hd, seed=11)
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    wide = torch.zeros(9, nq + 2, 2 * hd, dtype=torch.bfloat16, device=dev)
    wide[:6, 1:nq + 1, :hd] = d["q"]
    wide[6:] = float("nan")
    table = torch.full((3, 40), 10 ** 9, dtype=torch.int32, device=dev)
    table[:, 3:3 + d["block_tables"].shape[1]] = d["block_tables"]
    d["q"], d["block_tables"] = wide[:, 1:nq + 1, :hd], table[:, 3:3 + d["block_tables"].shape[1]]
    big = torch.full((9, nq + 1, hd + 8), 7.0, dtype=torch.bfloat16, device=dev)
    out = big[:, :nq, :hd]
    back = ops.shared_prefix_attention(scale=hd ** -0.5, out=out, **d)
    assert back.data_ptr() == out.data_ptr()
    check(out[:6], s, hd ** -0.5)
    assert bool((big[6:] == 7.0).all()) and bool((big[:, nq:] == 7.0).all()) and bool((big[:, :, hd:] == 7.0).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_equals_attention_without_sharing(hd, dev):
    """The same keys through whole tables and ops.prefill_attention / ops.paged_decode."""
    nq, nkv, owns = 8, 2, [5, 300, 64]
    s = make(512, owns, [1, 1, 1], nq, nkv, hd, seed=3, poison=False)
    bt = s["block_tables"].clone()
    bt[:, :2] = s["prefix_blocks"]
    bt[bt == 10 ** 9] = 0
    a = call(s, dev, hd ** -0.5)
    b = ops.paged_decode(s["q"].to(dev), s["k_cache"].to(dev), s["v_cache"].to(dev), bt.to(dev),
                         s["ctx_lens"].to(dev), hd ** -0.5)
    err = (a.double() - b.double()).abs().cpu()
    o, v = oracle(s, hd ** -0.5)
    assert bool((err <= 2 * (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10) * v)).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_prefix_length_on_the_device(dev):
    s = make(290, [1, 40], [1, 2], 8, 2, 128, seed=21)
    got = call(s, dev, 128 ** -0.5, prefix_len=torch.tensor([290], dtype=torch.int32, device=dev))
    check(got, s, 128 ** -0.5)


@pytest.mark.parametrize("dev", DEVICES)
def test_no_sequences_and_no_rows(dev):
    s = make(64, [1], [1], 4, 2, 64)
    e = dict(s, q=s["q"][:0], block_tables=s["block_tables"][:0], ctx_lens=s["ctx_lens"][:0], cu_q=s["cu_q"][:1])
    assert call(e, dev, 0.125).shape == (0, 4, 64)
    s = make(64, [3, 2], [0, 0], 4, 2, 64)
    assert call(s, dev, 0.125).shape == (0, 4, 64)


BAD = {
    "block size": lambda s: dict(s, k_cache=s["k_cache"][:, :, :32].contiguous(),
                                 v_cache=s["v_cache"][:, :, :32].contiguous()),
    "heads": lambda s: dict(s, q=s["q"][:, :3].contiguous()),
    "cache shapes": lambda s: dict(s, v_cache=s["v_cache"][:1].contiguous()),
    "head dim": lambda s: dict(s, q=s["q"][..., :64].contiguous()),
    "long tables": lambda s: dict(s, block_tables=s["block_tables"].long()),
    "long lengths": lambda s: dict(s, ctx_lens=s["ctx_lens"].long()),
    "prefix beyond its pages": lambda s: dict(s, prefix_len=513),
    "negative prefix": lambda s: dict(s, prefix_len=-1),
    "rows of tables": lambda s: dict(s, block_tables=s["block_tables"][:1]),
    "cu_q length": lambda s: dict(s, cu_q=s["cu_q"][:2]),
    "tokens without cu_q": lambda s: dict(s, cu_q=None),
    "max_q": lambda s: dict(s, max_q=0),
    "window": lambda s: dict(s, window=-1),
    "softcap": lambda s: dict(s, softcap=-1.0),
    "out shape": lambda s: dict(s, out=torch.empty_like(s["q"])[:1]),
}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what", sorted(BAD))
def test_refusals(what, dev):
    s = BAD[what](make(300, [3, 2], [2, 1], 8, 2, 128))
    with pytest.raises(RuntimeError):
        call(s, dev, 0.1)


@gpu
@pytest.mark.parametrize("what", ["float32 q", "strided cache", "odd rows", "cpu table", "head dim 520"])
def test_refusals_of_device_layouts(what):
    s = make(300, [3, 2], [2, 1], 8, 2, 520 if what == "head dim 520" else 128)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    if what == "float32 q":
        d["q"] = d["q"].float()
    if what == "strided cache":
        d["k_cache"] = torch.cat([d["k_cache"]] * 2, 3)[..., :128]
    if what == "odd rows":
        d["q"] = torch.zeros(3, 8, 132, dtype=torch.bfloat16, device="cuda")[..., :128]
    if what == "cpu table":
        d["block_tables"] = d["block_tables"].cpu()
    with pytest.raises(RuntimeError):
        ops.shared_prefix_attention(scale=0.1, **d)


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("what", ["page", "prefix page", "context", "max_len", "max_q", "device prefix"])
def test_bad_values_on_the_device_are_reported(what, hd):
    """The kernels' own bounds checks turn these into an error code; other sequences keep their results."""
    s = make(256, [3, 400, 2], [2, 1, 1], 8, 2, hd, seed=2)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    if what == "page":
        d["block_tables"][1, 2] = d["k_cache"].shape[0]
    if what == "prefix page":
        d["prefix_blocks"][0] = -1
    if what == "context":
        d["ctx_lens"][1] = d["block_tables"].shape[1] * BS + 1
    if what == "max_len":
        d["max_len"] = 400
    if what == "max_q":
        d["max_q"] = 1
    if what == "device prefix":
        d["prefix_len"] = torch.tensor([257], dtype=torch.int32, device="cuda")
    ops.error_word(torch.device("cuda")).zero_()
    out = ops.shared_prefix_attention(scale=hd ** -0.5, **d)
    torch.cuda.synchronize()
    with pytest.raises(DeviceWaitTimeout):
        ops.check_device_errors()
    ops.check_device_errors()  # read once, then clear
    if what in ("page", "context", "max_len"):
        keep = torch.tensor([0, 1, 3])
        o, a = oracle({**s, "q": s["q"][keep], "ctx_lens": s["ctx_lens"][[0, 2]],
                       "block_tables": s["block_tables"][[0, 2]],
                       "cu_q": torch.tensor([0, 2, 3], dtype=torch.int32)}, hd ** -0.5)
        err = (out[keep.cuda()].double().cpu() - o).abs()
        assert bool((err <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10) * a).all())


@gpu
def test_long_offsets():
    """Pages whose elements lie beyond 2^31 of the cache's start."""
    nq, nkv, hd, NB = 16, 8, 128, 8400
    assert NB * nkv * BS * hd > 2 ** 31
    s = make(700, [300, 60], [1, 2], nq, nkv, hd, seed=8)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    n = s["k_cache"].shape[0]
    for name in ("k_cache", "v_cache"):
        big = torch.empty(NB, nkv, BS, hd, dtype=torch.bfloat16, device="cuda")
        big[-n:] = d[name]
        d[name] = big
    d["prefix_blocks"] += NB - n
    d["block_tables"] += NB - n
    got = ops.shared_prefix_attention(scale=hd ** -0.5, **d)
    torch.cuda.synchronize()
    ops.check_device_errors()
    check(got, s, hd ** -0.5)


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_streams_and_graphs(hd):
    """Two calls on two streams at once, and two captured graphs replayed together, give the single call's bits."""
    cases = [make(1200, [300, 60, 9] * 8, [1, 2, 3] * 8, 8, 2, hd, seed=i) for i in range(2)]
    dev = [{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()} for s in cases]
    f = lambda d: ops.shared_prefix_attention(scale=hd ** -0.5, **d)  # noqa: E731
    want = [f(d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(f(dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for d in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f(d))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("many", [3, 30])
def test_graph_follows_lengths_on_the_device(many):
    """A captured call replayed with another prefix length, contexts and pages."""
    a = make(900, [30, 200], [1, many - 1], 8, 2, 128, seed=1, spare=3)
    b = make(640, [290, 40], [many - 2, 2], 8, 2, 128, seed=2, spare=4)
    buf = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    buf["k_cache"] = torch.zeros(12, 2, BS, 128, dtype=torch.bfloat16, device="cuda")
    buf["v_cache"] = torch.zeros_like(buf["k_cache"])
    buf["prefix_blocks"] = torch.zeros(8, dtype=torch.int32, device="cuda")
    buf["block_tables"] = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    buf["prefix_len"] = torch.zeros(1, dtype=torch.int32, device="cuda")

    def load(s):
        for k in ("q", "ctx_lens", "cu_q"):
            buf[k].copy_(s[k])
        for k in ("k_cache", "v_cache", "prefix_blocks"):
            buf[k][:s[k].shape[0]] = s[k].cuda()
        buf["block_tables"][:, :s["block_tables"].shape[1]] = s["block_tables"].cuda()
        buf["prefix_len"].fill_(s["prefix_len"])

    load(a)
    buf["max_q"] = many
    f = lambda: ops.shared_prefix_attention(scale=128 ** -0.5, max_len=2048, **buf)  # noqa: E731
    f()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    for s in (a, b, a):
        load(s)
        g.replay()
        torch.cuda.synchronize()
        ops.check_device_errors()
        check(out, s, 128 ** -0.5)
