"""The layer seam latent_attention against a float64 model of its own: the pool's rows are worked out from the inputs of
every step (norm, rotation, one rounding to bf16) and compared with the cache, and only then used as the attention's
keys and values.  The attention's bounds are latent_reference's for the form that ran; a row's are those of the store's
tests: half a bf16 step, and a few units of 2^-24 for the float32 in between."""
from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -8


class Model:
    """A layer, its pool, and what every sequence has put into it."""

    def __init__(self, pkg, dev, *, heads=16, r=512, dr=64, dn=128, page=16, pages=60, width=None, seed=0,
                 interleaved=True, eps=0.25, norm=True, scaling=None, oracle=()):
        self.pkg, self.dev, self.heads, self.r, self.dr, self.dn, self.page = pkg, dev, heads, r, dr, dn, page
        self.interleaved, self.eps, self.oracle = interleaved, eps, dict(oracle)
        self.gen = torch.Generator().manual_seed(seed)
        self.w = (self.rnd(heads * 2 * dn, r) * r ** -0.5).to(torch.bfloat16).to(dev)
        self.weights = pkg.LatentWeights(self.w, num_heads=heads, nope_dim=dn, v_dim=dn)
        self.norm = (1 + 0.3 * self.rnd(r)).to(torch.bfloat16).to(dev) if norm else None
        self.freqs = pkg.rotary_frequencies(dr, 1e4, scaling=scaling, device=dev)
        self.cache = torch.full((pages, page, r + dr), float("nan"), dtype=torch.bfloat16, device=dev)
        own = torch.randperm(pages, generator=self.gen).to(torch.int32).view(4, pages // 4)
        self.table = torch.full((4, width or pages // 4), -1, dtype=torch.int32)
        self.table[:, :pages // 4] = own
        self.rows = [torch.empty((0, r + dr), dtype=torch.bfloat16, device=dev) for _ in range(4)]

    def rnd(self, *s):
        return torch.randn(s, generator=self.gen)

    def check_rows(self, x, pos, got):
        """New rows of the pool against the inputs they come from."""
        c = x[:, :self.r].double()
        units = 0
        if self.norm is not None and self.oracle.get("norm", True):
            c = c / torch.sqrt(c.square().mean(-1, keepdim=True) + self.oracle.get("eps", self.eps)) * self.norm.double()
            units = 8
        kr, size = ref.rotate(x[:, None, self.r:], pos, self.freqs.inv_freq, self.oracle.get("amplitude",
                              self.freqs.amplitude), self.oracle.get("interleaved", self.interleaved))
        assert ((got[:, :self.r].double() - c).abs() <= (STEP * (units > 0) + units * 2.0 ** -24) * c.abs()).all(), \
            "latent rows"
        assert ((got[:, self.r:].double() - kr[:, 0]).abs() <= STEP * kr[:, 0].abs() + 6 * 2.0 ** -24 * size[:, 0]).all(), \
            "key parts"

    def step(self, new, decodes, *, longest=None, total_kv_tokens=None):
        """new[b] tokens of sequences b (decodes None: a decode step; 0: a prefill step; else a mixed one whose first
        `decodes` sequences have one each); longest: the metadata's max_seqlen_k."""
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)  # noqa: E731
        ids = [b for b, n in enumerate(new) if n]
        before = [len(r) for r in self.rows]
        total = [before[b] + new[b] for b in range(4)]
        pos = [j for b in ids for j in range(before[b], total[b])]
        slots = [int(self.table[b, j // self.page]) * self.page + j % self.page
                 for b in ids for j in range(before[b], total[b])]
        t = len(pos)
        q = self.rnd(t, self.heads, self.dn + self.dr).to(torch.bfloat16).to(self.dev)
        x = (2 * self.rnd(t, self.r + self.dr)).to(torch.bfloat16).to(self.dev)
        table, lens = self.table[ids].to(self.dev), i32([total[b] for b in ids])
        cu = i32([0] + [new[b] for b in ids]).cumsum(0).to(torch.int32)
        cu_k = i32([0] + [total[b] for b in ids]).cumsum(0).to(torch.int32)
        if decodes is None:
            meta = self.pkg.DecodeAttentionMetadata(i32(pos), i32(slots), table, lens)
        elif decodes == 0:
            meta = self.pkg.PrefillAttentionMetadata(i32(pos), i32(slots), table, cu, cu_k, None, longest,
                                                     max(new))
        else:
            meta = self.pkg.MixedAttentionMetadata(i32(pos), i32(slots), table, cu, lens, decodes, max(new),
                                                   max_seqlen_k=longest)
        scale = (self.dn + self.dr) ** -0.5
        q_in, x_in = q.clone(), x.clone()
        cache, out = self.pkg.latent_attention(self.cache, q, x[:, :self.r], x[:, self.r:], self.norm, self.weights,
                                               self.freqs, meta, scale=scale, eps=self.eps,
                                               interleaved=self.interleaved, total_kv_tokens=total_kv_tokens)
        assert cache is self.cache and torch.equal(q, q_in) and torch.equal(x, x_in)
        # ---- the pool: new rows from their inputs, old ones untouched, nothing elsewhere
        flat = self.cache.view(-1, self.r + self.dr)
        self.check_rows(x, i32(pos), flat[i32(slots).long()])
        at = 0
        for b in ids:
            self.rows[b] = torch.cat([self.rows[b], flat[i32(slots[at:at + new[b]]).long()]])
            at += new[b]
        used = torch.zeros(flat.shape[0], dtype=torch.bool, device=self.dev)
        for b in range(4):
            at_b = i32([int(self.table[b, j // self.page]) * self.page + j % self.page for j in range(total[b])]).long()
            assert torch.equal(flat[at_b], self.rows[b]), f"rows of sequence {b}"
            used[at_b] = True
        assert torch.isnan(flat[~used]).all(), "slots that nobody wrote"
        # ---- the attention
        q_rope, _ = ref.rotate(q[..., self.dn:], i32(pos), self.freqs.inv_freq, self.freqs.amplitude, self.interleaved)
        q_rope = q_rope.to(torch.bfloat16)
        w = self.w.view(self.heads, 2, self.dn, self.r)
        at = 0
        for i, b in enumerate(ids):
            n = new[b]
            one = decodes is None or i < decodes
            form = "absorbed" if one else self.form(meta, decodes, len(ids), t, total_kv_tokens)
            rows = list(range(n)) if n <= 12 else sorted({0, 1, n // 2, n - 2, n - 1})
            for h in (0, self.heads - 1):
                o, s = ref.attend(q[at:at + n, h, :self.dn][rows], q_rope[at:at + n, h][rows], self.rows[b], w[h, 0],
                                  w[h, 1], [total[b] - n + j + 1 for j in rows], scale, form)
                ref.check(out[at:at + n, h][rows], o, s, f"{form} sequence {b} head {h}")
            at += n
        return out

    def form(self, meta, decodes, sequences, tokens, bound):
        """The form of a step's prefill, from the bounds that it gives."""
        batch, width = sequences - (decodes or 0), self.table.shape[1] * self.page
        if bound is None:
            bound = min(batch * min(width, width if meta.max_seqlen_k is None else int(meta.max_seqlen_k)), 0x7fffffff)
        max_q = meta.max_seqlen_q if decodes else meta.max_seqlen_bucket
        code = self.pkg._lib.load().pa_latent_prefill_route(batch, tokens, max_q, bound, self.table.shape[1], self.page,
                                                            self.heads, self.r, self.dr, self.dn)
        return {0: "expanded", 1: "absorbed"}[code]


RUN = [([40, 1, 17, 0], 0), ([1, 1, 1, 0], None), ([1, 1, 1, 100], 3), ([1, 1, 9, 30], 2), ([1, 1, 1, 1], None),
       ([1, 1, 0, 0], 2), ([0, 0, 60, 0], 0)]


@pytest.mark.parametrize("kw", [
    dict(), dict(interleaved=False), dict(norm=False, interleaved=False, seed=1),
    dict(heads=5, r=256, dr=32, dn=64, page=7, pages=160, seed=3, interleaved=False),
    dict(heads=5, r=256, dr=32, dn=64, page=7, pages=160, seed=4),
    dict(heads=33, dr=32, page=64, pages=16, seed=5, interleaved=False,
         scaling=dict(type="yarn", factor=8, original_max_position=64))],
    ids=["interleaved", "half", "half-no-norm", "small-half", "small-interleaved", "yarn-half"])
def test_run_of_steps(pkg, dev, kw):
    """Prompts, decode steps, next turns beside running sequences, a mixed step of decodes alone."""
    model = Model(pkg, dev, **kw)
    for new, decodes in RUN:
        model.step(new, decodes)


@pytest.mark.parametrize("oracle", [dict(eps=0.0), dict(norm=False), dict(interleaved=False), dict(amplitude=1.25)],
                         ids=lambda o: next(iter(o)))
def test_model_notices(pkg, dev, oracle):
    """A model that lacks a part of the step does not agree with the pool."""
    model = Model(pkg, dev, oracle=oracle)
    with pytest.raises(AssertionError, match="latent rows|key parts"):
        model.step([5, 3, 0, 0], 0)


@pytest.mark.parametrize("bounds", [dict(), dict(longest=150), dict(total_kv_tokens=300),
                                    dict(longest=torch.tensor(150))], ids=["none", "each", "sum", "cpu-tensor"])
def test_bounds_of_a_step(pkg, dev, bounds):
    """What the host knows of the kv lengths chooses a step's plan, not its result."""
    model = Model(pkg, dev, heads=8, pages=40, seed=6)
    model.step([70, 33, 90, 5], 0, **bounds)
    model.step([1, 1, 40, 9], 2, **bounds)


def test_steps_over_tables_wider_than_any_bound(pkg, dev):
    """Tables of 2^30 tokens a sequence and no bound at all: the step runs, in little memory."""
    model = Model(pkg, dev, heads=8, r=256, dr=32, dn=64, page=1 << 16, pages=4, width=1 << 14, seed=7)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    at = torch.cuda.memory_allocated()
    model.step([20, 3, 1, 0], 0)
    model.step([1, 5, 7, 30], 1)
    model.step([1, 1, 1, 1], None)
    # (the model's own copies of the pool's masks and rows are a few pools)
    assert torch.cuda.max_memory_allocated() - at < 8 * model.cache.numel() * 2 + (64 << 20)
