"""latent_prefill_attention and the layer seam latent_attention against float64 (bounds: latent_reference)."""
from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu


def make(dev, seqs, heads, r, dr, dn, page, seed, *, before=0, behind=0, gain=1.0):
    """seqs: (new, total) tokens.  Cache rows that no sequence owns are NaN; `before` and `behind` rows of q belong to
    no sequence."""
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    need = [-(-t // page) for _, t in seqs]
    nb = sum(need) + 2
    perm = torch.randperm(nb, generator=gen)
    table = torch.full((len(seqs), max(need + [1])), -1, dtype=torch.int32)
    cache = torch.full((nb, page, r + dr), float("nan"))
    rows, at = [], 0
    for b, ((_, t), k) in enumerate(zip(seqs, need)):
        ids = perm[at:at + k]
        at += k
        table[b, :k] = ids.to(torch.int32)
        x = rnd(t, r + dr).to(torch.bfloat16)
        rows.append(x.to(dev))
        flat = torch.full((k * page, r + dr), float("nan"))
        flat[:t] = x.float()
        cache[ids] = flat.view(k, page, r + dr)
    tokens = before + sum(n for n, _ in seqs) + behind
    cum = lambda v, o: torch.tensor([o] + v).cumsum(0).to(torch.int32).to(dev)  # noqa: E731
    return dict(q=(rnd(tokens, heads, dn + dr) * gain).to(torch.bfloat16).to(dev),
                w=(rnd(heads * 2 * dn, r) * r ** -0.5).to(torch.bfloat16).to(dev),
                cache=cache.to(torch.bfloat16).to(dev), table=table.to(dev), rows=rows, seqs=seqs,
                cu_q=cum([n for n, _ in seqs], before), cu_k=cum([t for _, t in seqs], 0), before=before,
                lens=torch.tensor([t for _, t in seqs], dtype=torch.int32, device=dev))


def run(pkg, c, heads, dn, scale, lengths="cu_k", **kw):
    weights = pkg.LatentWeights(c["w"], num_heads=heads, nope_dim=dn, v_dim=dn)
    kw.setdefault("max_seqlen_q", max([n for n, _ in c["seqs"]] + [1]))
    kw.setdefault("total_kv_tokens", sum(t for _, t in c["seqs"]))
    by = dict(cu_k=dict(cu_seqlens_k=c["cu_k"]), lens=dict(kv_lens=c["lens"]), fresh={})[lengths]
    return pkg.latent_prefill_attention(c["q"][..., :dn], c["q"][..., dn:], c["cache"], weights, c["table"],
                                        c["cu_q"], scale=scale, **by, **kw)


def form(pkg, c, heads, r, dr, dn, page):
    lib = pkg._lib.load()
    code = lib.pa_latent_prefill_route(len(c["seqs"]), c["q"].shape[0], max(n for n, _ in c["seqs"]),
                                       sum(t for _, t in c["seqs"]), c["table"].shape[1], page, heads, r, dr, dn)
    return {0: "expanded", 1: "absorbed"}[code]


def check(pkg, c, got, heads, r, dr, dn, page, scale, *, some_heads=None, some_rows=None):
    which = form(pkg, c, heads, r, dr, dn, page)
    w = c["w"].view(heads, 2, dn, r)
    at = c["before"]
    assert not got[:at].any()
    for b, ((n, t), rows) in enumerate(zip(c["seqs"], c["rows"])):
        idx = list(range(n)) if some_rows is None or n <= some_rows else sorted(
            set(torch.randperm(n, generator=torch.Generator().manual_seed(b))[:some_rows].tolist()) |
            {0, n - 1, min(n - 1, 255), min(n - 1, 256)})
        for h in some_heads or range(heads):
            if not idx:
                continue
            q = c["q"][at:at + n, h][idx]
            o, s = ref.attend(q[:, :dn], q[:, dn:], rows, w[h, 0], w[h, 1], [t - n + i + 1 for i in idx], scale, which)
            ref.check(got[at:at + n, h][idx], o, s, f"{which} sequence {b} head {h}")
        at += n
    assert not got[at:].any()


@pytest.mark.parametrize("want,heads,r,dr,dn,page,seqs", [
    ("expanded", 1, 512, 64, 128, 16, [(1, 1)]),
    ("expanded", 3, 512, 64, 128, 16, [(5, 5), (70, 70), (1, 1)]),
    ("expanded", 2, 512, 64, 128, 64, [(257, 257)]),
    ("expanded", 2, 256, 32, 64, 7, [(63, 64), (64, 64), (65, 65), (0, 0), (128, 130)]),
    ("expanded", 2, 512, 32, 128, 256, [(300, 301)]),
    ("expanded", 2, 256, 64, 64, 1, [(40, 45), (33, 33)]),
    ("expanded", 2, 512, 64, 64, 48, [(200, 520)]),
    ("expanded", 1, 256, 64, 128, 32, [(600, 1000)]),
    ("absorbed", 3, 512, 64, 128, 16, [(2, 300), (1, 64), (3, 33)]),
    ("absorbed", 16, 512, 64, 128, 64, [(7, 500), (0, 10), (1, 1)]),
    ("absorbed", 65, 256, 32, 64, 5, [(2, 70)]),
    ("absorbed", 5, 512, 32, 128, 256, [(30, 900), (14, 700)]),
    ("absorbed", 33, 256, 64, 64, 17, [(4, 200), (5, 31)]),
])
def test_prefill(pkg, dev, want, heads, r, dr, dn, page, seqs):
    print(f"{want}: heads {heads} latent {r}+{dr} head {dn} page {page} {seqs}", flush=True)
    c = make(dev, seqs, heads, r, dr, dn, page, seed=heads + r + len(seqs), before=2, behind=3)
    assert form(pkg, c, heads, r, dr, dn, page) == want
    scale = (dn + dr) ** -0.5
    got = run(pkg, c, heads, dn, scale)
    check(pkg, c, got, heads, r, dr, dn, page, scale, some_rows=24)
    assert torch.equal(got, run(pkg, c, heads, dn, scale, lengths="lens")), "kv_lens and cu_seqlens_k agree"
    # a given out keeps the rows outside the sequences
    out = torch.full((got.shape[0], heads + 1, dn + 8), 3.0, dtype=torch.bfloat16, device=dev)
    run(pkg, c, heads, dn, scale, out=out[:, 1:, 8:])
    inside = torch.zeros(got.shape[0], dtype=torch.bool, device=dev)
    inside[c["before"]:c["before"] + sum(n for n, _ in seqs)] = True
    assert torch.equal(out[inside][:, 1:, 8:], got[inside])
    assert (out[~inside] == 3).all() and (out[:, 0] == 3).all() and (out[..., :8] == 3).all()


@pytest.mark.parametrize("heads,seqs", [(2, [(300, 100), (5, 2), (3, 0)]), (16, [(4, 2), (6, 0), (2, 300)])])
def test_prefill_rows_that_see_nothing(pkg, dev, heads, seqs):
    """kv lengths below the new tokens': the first rows see no key and are zero."""
    c = make(dev, seqs, heads, 512, 64, 128, 16, seed=5)
    got = run(pkg, c, heads, 128, 0.1)
    at = 0
    w = c["w"].view(heads, 2, 128, 512)
    for b, (n, t) in enumerate(seqs):
        none = max(0, n - t)
        assert not got[at:at + none].any()
        o, s = ref.attend(c["q"][at:at + n, 0, :128], c["q"][at:at + n, 0, 128:], c["rows"][b], w[0, 0], w[0, 1],
                          [t - n + i + 1 for i in range(n)], 0.1, form(pkg, c, heads, 512, 64, 128, 16))
        ref.check(got[at:at + n, 0], o, s, f"sequence {b}")
        at += n


@pytest.mark.parametrize("heads,seqs", [(2, [(400, 500), (130, 130)]), (16, [(5, 600)])])
def test_prefill_large_scores(pkg, dev, heads, seqs):
    c = make(dev, seqs, heads, 512, 64, 128, 32, seed=6, gain=40.0)
    check(pkg, c, run(pkg, c, heads, 128, 0.2), heads, 512, 64, 128, 32, 0.2, some_heads=[0, heads - 1], some_rows=40)


def test_prefill_fresh_and_max_seqlen_q(pkg, dev):
    """No kv lengths: those of the new tokens.  Rows past max_seqlen_q are zero in a new output."""
    c = make(dev, [(70, 70), (300, 300)], 2, 512, 64, 128, 16, seed=7)
    full = run(pkg, c, 2, 128, 0.1)
    assert torch.equal(full, run(pkg, c, 2, 128, 0.1, lengths="fresh", total_kv_tokens=None))
    # 200 of 370 rows wanted: the rule takes the absorbed form, which rounds elsewhere
    cut = run(pkg, c, 2, 128, 0.1, max_seqlen_q=100)
    assert not cut[170:].any()
    w = c["w"].view(2, 2, 128, 512)
    for h in range(2):
        o, s = ref.attend(c["q"][70:170, h, :128], c["q"][70:170, h, 128:], c["rows"][1], w[h, 0], w[h, 1],
                          list(range(1, 101)), 0.1, "absorbed")
        ref.check(cut[70:170, h], o, s, f"cut head {h}")


def test_prefill_head_groups(pkg, dev):
    """More K and V than are expanded at a time: the groups' launches give what one launch gives."""
    heads, total = 24, 70000
    lib = pkg._lib.load()
    size = lambda t: lib.pa_latent_prefill_workspace_size(1, 600, 600, t, 300, 256, heads, 512, 64, 128)  # noqa: E731
    assert size(total * 4) < 24 * total * 4 * 512 * 0.75, "the bound takes several groups"
    c = make(dev, [(600, 900)], heads, 512, 64, 128, 256, seed=3, behind=5)
    one = run(pkg, c, heads, 128, 0.1)
    several = run(pkg, c, heads, 128, 0.1, total_kv_tokens=total * 4)
    assert torch.equal(one, several)
    check(pkg, c, one, heads, 512, 64, 128, 256, 0.1, some_heads=[0, 7, 8, 23], some_rows=6)


def test_prefill_bounds_too_small_stay_in_bounds(pkg, dev):
    """A total_kv_tokens below the real sum drops rows but reads and writes nothing outside."""
    c = make(dev, [(300, 400), (200, 300)], 2, 512, 64, 128, 16, seed=8)
    got = run(pkg, c, 2, 128, 0.1, total_kv_tokens=500)
    full = run(pkg, c, 2, 128, 0.1)
    assert torch.isfinite(got).all() and torch.equal(got[:300], full[:300])
    c["table"][0, 0], c["table"][1, 1] = 1 << 30, -5
    c["cache"].nan_to_num_(nan=0.25)
    for cu in ([0, -7, 90], [50, 20, 800], [0, 1 << 30, 5], [0, 0, 0]):
        c["cu_k"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        assert torch.isfinite(run(pkg, c, 2, 128, 0.1)).all()
    for cu in ([0, -7, 90], [50, 20, 800], [0, 1 << 30, 5], [600, 700, 800], [-9, 3, 3]):
        c["cu_q"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        assert torch.isfinite(run(pkg, c, 2, 128, 0.1)).all()


def test_prefill_nothing(pkg, dev):
    c = make(dev, [(4, 4)], 2, 512, 64, 128, 16, seed=1, behind=2)
    none = dict(c, seqs=[], table=c["table"][:0], cu_q=c["cu_q"][:1], lens=c["lens"][:0])
    out = run(pkg, none, 2, 128, 0.1, lengths="lens", total_kv_tokens=0)
    assert tuple(out.shape) == (6, 2, 128) and not out.any()
    none = dict(c, table=c["table"][:, :0])
    assert not run(pkg, none, 2, 128, 0.1).any()


@pytest.mark.parametrize("heads,seqs", [(4, [(300, 300), (17, 40)]), (16, [(3, 200), (1, 77)])])
def test_prefill_graph_replays(pkg, dev, heads, seqs):
    """Captured once per form, replayed with new lengths and inputs, eager work of the same shape in between."""
    c = make(dev, seqs, heads, 512, 64, 128, 16, seed=11)
    c["cache"].nan_to_num_(nan=0.0)
    out = torch.zeros((c["q"].shape[0], heads, 128), dtype=torch.bfloat16, device=dev)
    run(pkg, c, heads, 128, 0.1, lengths="lens", out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(pkg, c, heads, 128, 0.1, lengths="lens", out=out)
    gen = torch.Generator().manual_seed(1)
    for i in range(4):
        c["q"].copy_(torch.randn(c["q"].shape, generator=gen).to(torch.bfloat16))
        c["lens"].copy_(torch.tensor([t - 5 * i for _, t in seqs], dtype=torch.int32))
        out.fill_(2.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(pkg, c, heads, 128, 0.1, lengths="lens")), f"replay {i}"


# ---------------------------------------------------------------------------
# the layer seam: store, decode, prefill and mixed steps over one pool
# ---------------------------------------------------------------------------
class Layer:
    """A layer's weights and pool, and a float64 twin of the pool's rows per sequence."""

    def __init__(self, pkg, dev, heads=16, r=512, dr=64, dn=128, page=16, pages=60, seed=0):
        self.pkg, self.dev, self.heads, self.r, self.dr, self.dn, self.page = pkg, dev, heads, r, dr, dn, page
        self.gen = torch.Generator().manual_seed(seed)
        self.w = (self.rnd(heads * 2 * dn, r) * r ** -0.5).to(torch.bfloat16).to(dev)
        self.weights = pkg.LatentWeights(self.w, num_heads=heads, nope_dim=dn, v_dim=dn)
        self.norm = (1 + 0.1 * self.rnd(r)).to(torch.bfloat16).to(dev)
        self.freqs = pkg.rotary_frequencies(dr, 1e4, device=dev)
        self.cache = torch.full((pages, page, r + dr), float("nan"), dtype=torch.bfloat16, device=dev)
        self.table = torch.randperm(pages, generator=self.gen).to(torch.int32).view(4, pages // 4).to(dev)
        self.lens = [0] * 4

    def rnd(self, *s):
        return torch.randn(s, generator=self.gen)

    def step(self, new, decodes):
        """new[b] tokens of sequences b (the first `decodes` of them one each); checks the output."""
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)  # noqa: E731
        ids = [b for b, n in enumerate(new) if n]
        pos, slots, tab = [], [], self.table.cpu()
        for b in ids:
            for j in range(self.lens[b], self.lens[b] + new[b]):
                pos.append(j)
                slots.append(int(tab[b, j // self.page]) * self.page + j % self.page)
            self.lens[b] += new[b]
        t = len(pos)
        q = self.rnd(t, self.heads, self.dn + self.dr).to(torch.bfloat16).to(self.dev)
        x = (2 * self.rnd(t, self.r + self.dr)).to(torch.bfloat16).to(self.dev)
        table, lens = self.table[ids], i32([self.lens[b] for b in ids])
        cu = i32([0] + [new[b] for b in ids]).cumsum(0).to(torch.int32)
        cu_k = i32([0] + [self.lens[b] for b in ids]).cumsum(0).to(torch.int32)
        if decodes is None:
            meta = self.pkg.DecodeAttentionMetadata(i32(pos), i32(slots), table, lens)
        elif decodes == 0:
            meta = self.pkg.PrefillAttentionMetadata(i32(pos), i32(slots), table, cu, cu_k, None, None, max(new))
        else:
            meta = self.pkg.MixedAttentionMetadata(i32(pos), i32(slots), table, cu, lens, decodes, max(new))
        scale = (self.dn + self.dr) ** -0.5
        before = q.clone()
        cache, out = self.pkg.latent_attention(self.cache, q, x[:, :self.r], x[:, self.r:], self.norm, self.weights,
                                               self.freqs, meta, scale=scale, eps=1e-6)
        assert cache is self.cache and torch.equal(q, before)
        # the store's own rows (checked by the store's tests) are the attention's input
        q_rope, _ = ref.rotate(q[..., self.dn:], i32(pos), self.freqs.inv_freq, 1.0, True)
        q_rope = q_rope.to(torch.bfloat16)
        w = self.w.view(self.heads, 2, self.dn, self.r)
        at = 0
        for b in ids:
            k = -(-self.lens[b] // self.page)
            rows = self.cache[self.table[b, :k].long()].flatten(0, 1)[:self.lens[b]]
            assert torch.isfinite(rows).all()
            n = new[b]
            for h in (0, self.heads - 1):
                args = (q[at:at + n, h, :self.dn], q_rope[at:at + n, h], rows, w[h, 0], w[h, 1],
                        [self.lens[b] - n + i + 1 for i in range(n)], scale)
                o, s1 = ref.attend(*args, "absorbed")
                _, s2 = ref.attend(*args, "expanded")
                ref.check(out[at:at + n, h], o, torch.maximum(s1, s2), f"sequence {b} head {h}")
            at += n
        return out


def test_layer_run_of_steps(pkg, dev):
    """Prompts, decode steps, a next turn beside running sequences, over one pool."""
    layer = Layer(pkg, dev)
    layer.step([40, 1, 17, 0], 0)
    layer.step([1, 1, 1, 0], None)
    layer.step([1, 1, 1, 100], 3)      # a new prompt beside three running sequences
    layer.step([1, 1, 9, 30], 2)       # next turns beside two
    layer.step([1, 1, 1, 1], None)
    layer.step([1, 1, 0, 0], 2)        # a mixed step of decodes alone
    layer.step([0, 0, 60, 0], 0)


def test_layer_small_latent_half_layout_step(pkg, dev):
    layer = Layer(pkg, dev, heads=5, r=256, dr=32, dn=64, page=7, pages=80, seed=3)
    layer.step([33, 70, 2, 5], 0)
    layer.step([1, 1, 4, 9], 2)
    layer.step([1, 1, 1, 1], None)
