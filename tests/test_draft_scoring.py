"""The operators of one scoring step together: keys and values of drafted tokens stored, attention on the shared prefix,
logits, verification; several steps on one paged cache, each stage held against 64 bits."""
import math

import pytest
import torch

from nanovllm_b200 import ops
from test_shared_prefix import oracle as attention_oracle
from test_verify_drafts import oracle as verify_oracle

gpu = pytest.mark.gpu
BS, V, D, NQ, NKV = 256, 520, 256, 4, 2


class Toy:
    """One attention layer whose logits favour the token ``succ`` of the current one; text on a paged cache."""

    def __init__(self, dev, hd, prefix, texts, max_q, seed):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.hd, self.max_q, self.g, self.P = dev, hd, max_q, g, prefix
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.E = r(V, D)
        self.succ = torch.randperm(V, generator=g)
        self.w_qkv = (r((NQ + 2 * NKV) * hd, D) / math.sqrt(D)).bfloat16().to(dev)
        self.w_o = (r(D, NQ * hd) / math.sqrt(NQ * hd)).bfloat16().to(dev)
        head = torch.empty(V, D)
        head[self.succ] = 12.0 * self.E / D
        self.w_lm = head.bfloat16().to(dev)
        self.E = self.E.bfloat16().to(dev)
        self.qw, self.kw = (torch.rand(hd, generator=g).add(0.5).bfloat16().to(dev) for _ in range(2))
        self.rope = ops.ref.rope_cos_sin(hd, prefix + 1024, 10000.0).to(dev)
        B, whole = len(texts), prefix // BS
        own_pages = -(-(prefix % BS + max(texts) + 8 * max_q) // BS)
        pages = torch.randperm(-(-prefix // BS) + B * own_pages, generator=g).int()
        self.prefix_blocks = pages[:-(-prefix // BS)]
        self.bt = torch.cat([self.prefix_blocks[:whole].expand(B, whole), pages[-(-prefix // BS):].view(B, own_pages)], 1)
        self.kc, self.vc = (torch.full((pages.numel(), NKV, BS, hd), math.nan).bfloat16().to(dev) for _ in range(2))
        shared = torch.randint(0, V, (prefix,), generator=g).tolist()
        self.text = [shared + torch.randint(0, V, (n,), generator=g).tolist() for n in texts]
        pos = torch.arange(prefix)
        self.store(shared, pos, self.prefix_blocks[pos // BS].long() * BS + pos % BS)
        for b, t in enumerate(self.text):  # the last token of a text is stored by the step that it begins
            self.store(t[prefix:-1], torch.arange(prefix, len(t) - 1), self.slots(b, prefix, len(t) - 1))

    def slots(self, b, lo, hi):
        pos = torch.arange(lo, hi)
        return self.bt[b, pos // BS].long() * BS + pos % BS

    def qkv_store(self, ids, pos, slots):
        x = self.E[ids]
        q = ops.qk_norm_rope_store(ops.linear(x, self.w_qkv), pos, self.rope, self.qw, self.kw, 0, False, 1e-6, self.kc,
                                   self.vc, slots, NQ, NKV, self.hd)
        return x, q

    def store(self, ids, pos, slots):
        if len(ids):
            d = self.dev
            self.qkv_store(torch.tensor(ids, device=d), pos.to(d), slots.to(torch.int32).to(d))

    def batch(self):
        """Each text's last token and 0 .. max_q - 1 drafts behind it, padded to one size with rows of no sequence."""
        B, T = len(self.text), len(self.text) * self.max_q
        ids, pos, slots, cu, ctx = [], [], [], [0], []
        for b, t in enumerate(self.text):
            row, n = [t[-1]], int(torch.randint(0, self.max_q, (1,), generator=self.g))
            for _ in range(n):
                good = torch.rand(1, generator=self.g) < 0.8
                row.append(int(self.succ[row[-1]]) if good else int(torch.randint(0, V, (1,), generator=self.g)))
            ids += row
            pos += range(len(t) - 1, len(t) + n)
            slots.append(self.slots(b, len(t) - 1, len(t) + n))
            cu.append(cu[-1] + n + 1)
            ctx.append(len(t) + n)
        pad = T - len(ids)
        i32 = dict(dtype=torch.int32)
        return dict(ids=torch.tensor(ids + [0] * pad), pos=torch.tensor(pos + [0] * pad),
                    slots=torch.cat(slots + [torch.full((pad,), -1)]).int(), cu=torch.tensor(cu, **i32),
                    ctx=torch.tensor(ctx, **i32), uniforms=torch.rand(T, generator=self.g))

    def step(self, s, knobs, prefix_len):
        """What a scoring step calls, all of it on the device and at fixed sizes."""
        x, q = self.qkv_store(s["ids"], s["pos"], s["slots"])
        o = ops.shared_prefix_attention(q, self.kc, self.vc, s["prefix_blocks"], prefix_len, s["bt"], s["ctx"],
                                        self.hd ** -0.5, cu_q=s["cu"], max_q=self.max_q)
        h = x + ops.linear(o.reshape(o.shape[0], -1), self.w_o)
        logits = ops.linear(h, self.w_lm)
        tokens, counts = ops.verify_drafts(logits, s["ids"], s["cu"], self.max_q, *knobs, s["uniforms"])
        return q, o, h, logits, tokens, counts


def check_step(m, s, knobs, got):
    q, o, h, logits, tokens, counts = (t.cpu() for t in got)
    n = int(s["cu"][-1])
    kc, vc = m.kc.cpu(), m.vc.cpu()
    # attention: as its own test holds it, from the keys and values that are stored
    want, a = attention_oracle(dict(q=q, k_cache=kc, v_cache=vc, prefix_blocks=m.prefix_blocks, prefix_len=m.P,
                                    block_tables=m.bt, ctx_lens=s["ctx"], cu_q=s["cu"]), m.hd ** -0.5)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * a
    assert bool(((o[:n].double() - want[:n]).abs() <= tol[:n] + 1e-30).all())
    # logits: one rounding to bf16, and sums of D products in 32 bits (D 2^-24 of the sum of absolute products)
    w = m.w_lm.cpu().double()
    want, a = h[:n].double() @ w.T, h[:n].double().abs() @ w.T.abs()
    assert bool(((logits[:n].double() - want).abs() <= 2.0 ** -8 * want.abs() + (D * 2.0 ** -24 + 2.0 ** -16) * a).all())
    # tokens: exactly those of a 64-bit verification of these logits
    temps, top_ks, top_ps = knobs
    want = verify_oracle(dict(logits=logits, ids=s["ids"], cu_q=s["cu"], max_q=m.max_q, temps=temps.cpu(),
                              top_ks=top_ks.cpu(), top_ps=top_ps.cpu(), uniforms=s["uniforms"]))
    assert (tokens.tolist(), counts.tolist()) == tuple(want)
    if m.P % BS == 0:  # one token at a time: every query token as a sequence of its own (whole shared pages: one table)
        rows = torch.repeat_interleave(torch.arange(len(m.text)), s["cu"].diff().long())
        caches = (c.nan_to_num(0.0) for c in (m.kc, m.vc))  # paged_decode wants finite values at unused keys too
        single = ops.paged_decode(q[:n].to(m.dev), *caches, m.bt[rows].to(m.dev), (s["pos"][:n] + 1).int().to(m.dev),
                                  m.hd ** -0.5).cpu()
        assert bool(((single.double() - o[:n].double()).abs() <= 2 * tol[:n] + 1e-30).all())


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu), pytest.param("graph", marks=gpu)])
@pytest.mark.parametrize("hd,prefix,texts,max_q", [(64, 512, [1, 40, 7], 4), (128, 300, [3, 1, 260, 90], 5),
                                                   (128, 1024, [5] * 20, 3), (256, 256, [2, 30], 1)])
def test_scoring_steps_on_one_cache(dev, hd, prefix, texts, max_q):
    graph, dev = dev == "graph", "cuda" if dev == "graph" else dev
    m = Toy(dev, hd, prefix, texts, max_q, seed=hd + prefix)
    B = len(texts)
    knobs = (torch.linspace(0.5, 1.0, B).to(dev), torch.tensor([(0, 1, 8, 40)[b % 4] for b in range(B)],
             dtype=torch.int32, device=dev), torch.tensor([(1.0, 0.9)[b % 2] for b in range(B)]).to(dev))
    fixed = dict(bt=m.bt.to(dev), prefix_blocks=m.prefix_blocks.to(dev))
    prefix_len = torch.tensor([prefix], dtype=torch.int32, device=dev) if graph else prefix
    static, replay, out, accepted = None, None, None, 0
    for _ in range(4):
        s = m.batch()
        put = {k: v.to(dev) for k, v in s.items()}
        if not graph:
            out = m.step(dict(put, **fixed), knobs, prefix_len)
        elif static is None:
            static = put
            out = m.step(dict(static, **fixed), knobs, prefix_len)  # first calls outside the capture
            torch.cuda.synchronize()
            replay = torch.cuda.CUDAGraph()
            with torch.cuda.graph(replay):
                out = m.step(dict(static, **fixed), knobs, prefix_len)
            replay.replay()
        else:
            for k, v in put.items():
                static[k].copy_(v)
            replay.replay()
        if dev == "cuda":
            torch.cuda.synchronize()
            ops.check_device_errors()
        check_step(m, s, knobs, out)
        for b, (row, c) in enumerate(zip(out[4].cpu().tolist(), out[5].cpu().tolist())):
            m.text[b] += row[:c]
            accepted += c - 1
    assert max_q == 1 or accepted > 0
    # the cache holds the accepted text, whatever refused drafts were stored in between: one pass over each text gives
    # the same keys and values but for two roundings to bf16 on either side and the norm's share of the first
    kept = m.kc.clone(), m.vc.clone()
    for b, t in enumerate(m.text):
        at = m.slots(b, prefix, len(t) - 1)
        m.store(t[prefix:-1], torch.arange(prefix, len(t) - 1), at)
        for was, now in zip(kept, (m.kc, m.vc)):
            x, y = (c.cpu().double()[at // BS, :, at % BS] for c in (was, now))
            size = x.abs().amax(-1, keepdim=True)  # a rotation mixes two values of a head
            assert bool(((x - y).abs() <= 6 * 2.0 ** -8 * size).all())
