"""Performance cases of the latent-attention path and of the rotation: the calls an engine makes per layer and step
where the cache holds one latent vector a token instead of K and V rows per head.

``listed()`` names the cases, ``draw()`` makes further ones over the same ranges.  ``run()`` computes a case through
the package's public entry points where ``own`` is true, else in plain torch operations in 32 bits.

A case is a dict of plain values; ``op`` says which operator it calls:

  "rotary"    rotary_embedding: [tokens, heads, dim] rows of ``dtype``, ``rotary_dim`` elements from ``start`` on
              rotated (``interleaved`` pairs or halves), frequencies of ``base`` and ``scaling``, positions < max_pos
  "store"     latent_store: RMSNorm of the latent rows, rotation of the shared key part and of q's, paged write
  "decode"    latent_decode_attention: one new token a sequence over the paged latent cache
  "prefill"   latent_prefill_attention: ragged new tokens behind cached ones

  heads, latent (R), rope (Dr), nope (Dn, and the value size), page
  seqs, new_lo .. new_hi, prefix_lo .. prefix_hi    new and cached tokens a sequence (decode: cached only, the new
                                                    token included)
  lens        seeds the lengths, which are part of the case; values and page placement come from the seed
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    """``vllm-jax_amd/`` under its module name (the folder's hyphen needs an import by path)."""
    import __graft_entry__
    return __graft_entry__.load_package()


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _rotary(tokens, heads, dim, rotary_dim, *, start=0, interleaved=False, dtype="bf16", base=1e6, scaling="",
            factor=1.0, max_pos=32768, name=None):
    c = dict(op="rotary", tokens=tokens, heads=heads, dim=dim, rotary_dim=rotary_dim, start=start,
             interleaved=interleaved, dtype=dtype, base=float(base), scaling=scaling, factor=float(factor),
             max_pos=max_pos)
    if name:
        c["name"] = name
    return c


def _latent(op, heads, page, *, latent=512, rope=64, nope=128, seqs=1, new=(1, 1), prefix=(0, 0), interleaved=True,
            lens=0, name=None):
    c = dict(op=op, heads=heads, latent=latent, rope=rope, nope=nope, page=page, seqs=seqs, new_lo=new[0],
             new_hi=new[1], prefix_lo=prefix[0], prefix_hi=prefix[1], interleaved=interleaved, lens=lens)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # A decode step's q rows, whole heads in halves (Qwen3-8B heads): latency.
        _rotary(64, 32, 128, 128, name="rotary_step"),
        # An odd prompt in float32 with part of an odd head size rotated, frequencies stretched by a larger base.
        _rotary(1999, 16, 80, 40, dtype="fp32", scaling="ntk", factor=4, name="rotary_part_fp32"),
        # Long prompts: the last 64 of 192 elements, interleaved, yarn, positions up to 128k.
        _rotary(16384, 64, 192, 64, start=128, interleaved=True, scaling="yarn", factor=32, max_pos=131072,
                name="rotary_long"),
        # The store of the engine's smallest decode step: four tokens, 16-token pages.
        _latent("store", 16, 16, seqs=4, new=(1, 1), prefix=(16, 127), lens=1, name="store_step"),
        # The store of a batch of prompts, 64 heads.
        _latent("store", 64, 256, seqs=8, new=(1024, 3000), lens=2, interleaved=False, name="store_prompts"),
        # The smallest decode: four short chats over 16-token pages, the smaller latent.
        _latent("decode", 16, 16, latent=256, rope=32, nope=64, seqs=4, prefix=(17, 128), lens=3, name="decode_tiny"),
        # One user's long conversation: a single 32k-token context.
        _latent("decode", 64, 64, seqs=1, prefix=(32768, 32768), lens=4, name="decode_one_long"),
        # The serving batch on a device that holds 16 of a model's heads: bound by the cache's reads.
        _latent("decode", 16, 256, seqs=256, prefix=(512, 8192), lens=5, name="decode_batch_16"),
        # The serving batch with all 128 heads on one device: bound by the matrix cores.
        _latent("decode", 128, 64, seqs=64, prefix=(512, 8192), lens=6, name="decode_batch_128"),
        # A few short prompts at once.
        _latent("prefill", 16, 256, seqs=4, new=(17, 511), lens=7, name="prefill_tiny"),
        # The next turns of eight long conversations, short ones behind their own cached contexts.
        _latent("prefill", 32, 64, seqs=8, new=(20, 200), prefix=(2000, 12000), lens=8, name="prefill_turn"),
        # The largest: long documents.
        _latent("prefill", 64, 256, seqs=2, new=(8192, 16384), lens=9, name="prefill_long"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: any operator, the listed head counts, latent sizes and page sizes, lengths over the logarithm of
    their range."""
    op = rng.choice(["rotary", "store", "decode", "decode", "prefill", "prefill"])
    heads = rng.choice([8, 16, 20, 32, 64, 128])
    page = rng.choice([16, 32, 64, 256])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        r = min(dim, rng.choice([32, 40, 64, 96, 128, dim]))
        scaling = rng.choice(["", "linear", "ntk", "yarn"])
        return _rotary(_log_int(rng, 1, 16384), rng.choice([1, 8, 16, 20, 32, 64]), dim, r,
                       start=rng.choice([0, dim - r]), interleaved=rng.random() < 0.5,
                       dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), base=rng.choice([1e4, 1e6]),
                       scaling=scaling, factor=rng.choice([2, 4, 32]) if scaling else 1,
                       max_pos=_log_int(rng, 1024, 131072))
    size = rng.choice([dict(latent=512, rope=64, nope=128)] * 3 + [dict(latent=256, rope=32, nope=64)])
    lens = rng.randrange(1 << 20)
    inter = rng.random() < 0.5
    if op == "store":
        n = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 24000 // n))
        return _latent("store", heads, page, **size, seqs=n, new=(max(1, hi // 3), hi), prefix=(0, 4096),
                       interleaved=inter, lens=lens)
    if op == "decode":
        n = _log_int(rng, 1, 256)
        hi = _log_int(rng, 16, max(64, min(32768, 500_000 // n)))
        return _latent("decode", heads, page, **size, seqs=n, prefix=(max(1, hi // rng.choice([1, 2, 16])), hi),
                       lens=lens)
    n = _log_int(rng, 1, 32)
    hi = _log_int(rng, 1, max(32, min(12000, 32768 // n)))
    p = _log_int(rng, 16, max(64, min(16384, 100_000 // n))) if rng.random() < 0.6 else 0
    c = _latent("prefill", heads, page, **size, seqs=n, new=(max(1, hi // rng.choice([1, 2, 8])), hi),
                prefix=(p // rng.choice([1, 4]), p), lens=lens)
    while work(c)["flops"] > 6e12:  # below the largest listed case
        c.update(new_lo=max(1, c["new_lo"] // 2), new_hi=max(1, c["new_hi"] // 2), prefix_lo=c["prefix_lo"] // 2,
                 prefix_hi=c["prefix_hi"] // 2)
    return c


def _lengths(case):
    """New tokens and all tokens of each sequence."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    pre = [rng.randint(case["prefix_lo"], case["prefix_hi"]) for _ in range(case["seqs"])]
    if case["op"] == "decode":
        return new, pre
    return new, [n + p for n, p in zip(new, pre)]


def work(case):
    if case["op"] == "rotary":
        size = DTYPES[case["dtype"]].itemsize
        rows = case["tokens"] * case["heads"]
        return {"bytes": 2 * rows * case["dim"] * size + 4 * case["tokens"], "flops": 3 * rows * case["rotary_dim"]}
    new, total = _lengths(case)
    h, r, dr, dn = case["heads"], case["latent"], case["rope"], case["nope"]
    tokens, row = sum(new), 2 * (r + dr)
    if case["op"] == "store":
        return {"bytes": tokens * (2 * row + 4 * h * dr + 8), "flops": tokens * (4 * r + 3 * (h + 1) * dr)}
    table = 4 * sum(-(-n // case["page"]) for n in total)
    weights = 2 * h * 2 * dn * r
    io = 2 * tokens * h * (2 * dn + dr)
    flops = 0
    for n, t in zip(new, total):
        pairs = n * (t - n) + n * (n + 1) // 2
        absorbed = 2 * h * (pairs * (2 * r + dr) + n * r * 2 * dn)
        expanded = 2 * h * (pairs * (2 * dn + dr) + t * r * 2 * dn)
        flops += min(absorbed, expanded)
    return {"bytes": sum(total) * row + weights + io + table, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(shape, gen, dev, dtype=torch.bfloat16, scale=1.0):
    t = torch.empty(shape, dtype=dtype, device=dev)
    flat = t.view(-1)
    step = 1 << 28
    for s in range(0, flat.numel(), step):
        n = min(step, flat.numel() - s)
        flat[s:s + n] = torch.randn(n, generator=gen, device=dev, dtype=torch.float32) * scale
    return t


def _scaling(case):
    if not case["scaling"]:
        return None
    s = dict(type=case["scaling"], factor=case["factor"])
    if case["scaling"] == "yarn":
        s.update(original_max_position=4096)
    return s


def _frequencies(r, base, scaling, factor):
    """Angle a position of each of the r / 2 pairs, in 64 bits, and the factor on cos and sin."""
    i = np.arange(r // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (r / (r - 2))
    f = base ** (-2 * i / r)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        def pair(turns):  # the pair that makes `turns` turns over the original 4096 positions
            return r * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), r - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0


def _layout(case, gen, dev):
    """Block tables (-1 padded), slots and positions as a scheduler lays them out: sequences' pages in a random order
    over the pool."""
    new, total = _lengths(case)
    bs = case["page"]
    own_pages = [-(-n // bs) for n in total]
    num_pages = sum(own_pages)
    num_pages += num_pages // 8 + 1               # a pool is never quite full
    perm = torch.randperm(num_pages, generator=gen, device=dev).to(torch.int32).cpu().numpy()
    table = np.full((len(total), max(own_pages)), -1, np.int32)
    at, slots, positions = 0, [], []
    for i, (n, t, o) in enumerate(zip(new, total, own_pages)):
        table[i, :o] = perm[at:at + o]
        at += o
        pos = np.arange(t - n, t)
        positions.append(pos)
        slots.append(table[i, pos // bs].astype(np.int64) * bs + pos % bs)
    i32 = lambda a: torch.as_tensor(np.ascontiguousarray(a, dtype=np.int32), device=dev)  # noqa: E731
    cu = lambda n: i32(np.concatenate([[0], np.cumsum(n)]))  # noqa: E731
    return dict(num_pages=num_pages, new=new, total=total, table=i32(table), slots=i32(np.concatenate(slots)),
                positions=i32(np.concatenate(positions)), cu_q=cu(new), cu_k=cu(total), lens=i32(total))


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "rotary":
        s["x"] = _randn((case["tokens"], case["heads"], case["dim"]), gen, dev, DTYPES[case["dtype"]])
        s["positions"] = torch.randint(0, case["max_pos"], (case["tokens"],), generator=gen, device=dev,
                                       dtype=torch.int32)
        if own:
            s["pa"] = _package()
            s["freqs"] = s["pa"].rotary_frequencies(case["rotary_dim"], case["base"], scaling=_scaling(case),
                                                    device=dev)
        return s
    s.update(_layout(case, gen, dev))
    h, r, dr, dn = case["heads"], case["latent"], case["rope"], case["nope"]
    tokens = sum(s["new"])
    # rows as the store leaves them: a normalised latent, a rotated key part of about unit size
    s["cache"] = _randn((s["num_pages"], case["page"], r + dr), gen, dev)
    if own:
        s["pa"] = _package()
    if case["op"] == "store":
        projected = _randn((tokens, r + dr), gen, dev, scale=2.0)  # the down projection's output, split by its user
        s["latent"], s["k_rope"] = projected[:, :r], projected[:, r:]
        s["q"] = _randn((tokens, h, dn + dr), gen, dev)
        s["norm"] = (1 + 0.1 * torch.randn(r, generator=gen, device=dev)).to(torch.bfloat16)
        if own:
            s["freqs"] = s["pa"].rotary_frequencies(dr, 1e4, device=dev)
        return s
    s["q"] = _randn((tokens, h, dn + dr), gen, dev)
    s["w"] = _randn((h * 2 * dn, r), gen, dev, scale=r ** -0.5)   # the up projection: K rows then V rows of each head
    if own:
        s["weights"] = s["pa"].LatentWeights(s["w"], num_heads=h, nope_dim=dn, v_dim=dn)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)(s, case)


def _run_own(s, case):
    pa = s["pa"]
    if case["op"] == "rotary":
        return pa.rotary_embedding(s["x"], s["positions"], s["freqs"], start=case["start"],
                                   interleaved=case["interleaved"])
    dn = case["nope"]
    if case["op"] == "store":
        cache, q_rope = pa.latent_store(s["latent"], s["k_rope"], s["norm"], s["positions"], s["slots"], s["cache"],
                                        s["freqs"], eps=EPS, interleaved=case["interleaved"], q_rope=s["q"][..., dn:])
        return {"cache": cache, "q_rope": q_rope}
    scale = (dn + case["rope"]) ** -0.5
    if case["op"] == "decode":
        return pa.latent_decode_attention(s["q"][..., :dn], s["q"][..., dn:], s["cache"], s["weights"], s["table"],
                                          s["lens"], scale=scale)
    return pa.latent_prefill_attention(s["q"][..., :dn], s["q"][..., dn:], s["cache"], s["weights"], s["table"],
                                       s["cu_q"], s["cu_k"], max_seqlen_q=max(s["new"]), max_seqlen_k=max(s["total"]),
                                       total_kv_tokens=sum(s["total"]), scale=scale)


def _rotate(x, positions, r, start, interleaved, base, scaling, factor):
    """The plain rotation of x [T, H, d]: angles in 64 bits, the rest in 32."""
    f, amp = _frequencies(r, base, scaling, factor)
    angle = positions.double()[:, None] * torch.as_tensor(f, device=x.device)
    cos, sin = (torch.cos(angle) * amp).float()[:, None], (torch.sin(angle) * amp).float()[:, None]
    y = x.float()
    part = y[..., start:start + r]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :r // 2], part[..., r // 2:])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    part = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([y[..., :start], part, y[..., start + r:]], -1).to(x.dtype)


def _rows(cache, table, page, total):
    """Cache rows of one sequence, [total, R + Dr]."""
    return cache[table[:-(-total // page)].long()].flatten(0, 1)[:total]


def _attend(q, k, v, first, scale):
    """q [H, n, dk] at kv positions first .. first + n - 1, k [H, L, dk], v [H, L, dv], 32 bits, causal."""
    h, n, _ = q.shape
    out = torch.empty((h, n, v.shape[2]), dtype=q.dtype, device=q.device)
    step = max(1, (1 << 28) // (h * k.shape[1]))
    kt = k.transpose(1, 2).contiguous()
    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        hi = first + r1
        x = torch.matmul(q[:, r0:r1], kt[:, :, :hi].contiguous()) * scale
        hidden = torch.arange(hi, device=q.device) > torch.arange(first + r0, first + r1, device=q.device)[:, None]
        x = x.masked_fill_(hidden, float("-inf"))
        x = torch.exp(x - x.amax(-1, keepdim=True))
        out[:, r0:r1] = torch.matmul(x, v[:, :hi]) / x.sum(-1, keepdim=True)
    return out


def _run_plain(s, case):
    if case["op"] == "rotary":
        return _rotate(s["x"], s["positions"], case["rotary_dim"], case["start"], case["interleaved"], case["base"],
                       case["scaling"], case["factor"])
    h, r, dr, dn, page = case["heads"], case["latent"], case["rope"], case["nope"], case["page"]
    if case["op"] == "store":
        rot = lambda x: _rotate(x, s["positions"], dr, 0, case["interleaved"], 1e4, "", 1.0)  # noqa: E731
        c = s["latent"].float()
        c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()
        row = torch.cat([c.to(torch.bfloat16), rot(s["k_rope"][:, None])[:, 0]], -1)
        s["cache"].view(-1, r + dr)[s["slots"].long()] = row
        return {"cache": s["cache"], "q_rope": rot(s["q"][..., dn:])}
    scale = (dn + dr) ** -0.5
    w = s["w"].float().view(h, 2 * dn, r)
    wk, wv = w[:, :dn].contiguous(), w[:, dn:].transpose(1, 2).contiguous()
    q = s["q"].float().transpose(0, 1).contiguous()                # [H, T, Dn + Dr]
    if case["op"] == "decode":
        q = torch.cat([torch.matmul(q[..., :dn].contiguous(), wk), q[..., dn:]], -1)    # [H, B, R + Dr]
        o = torch.empty((h, case["seqs"], r), dtype=torch.float32, device=q.device)
        for b, t in enumerate(s["total"]):
            c = _rows(s["cache"], s["table"][b], page, t).float()
            x = torch.matmul(q[:, b], c.t()) * scale
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o[:, b] = torch.matmul(x, c[:, :r]) / x.sum(-1, keepdim=True)
        return torch.matmul(o, wv).transpose(0, 1).to(torch.bfloat16)
    out = torch.empty((q.shape[1], h, dn), dtype=torch.bfloat16, device=q.device)
    at = 0
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        c = _rows(s["cache"], s["table"][b], page, t).float()
        g = max(1, min(h, (1 << 28) // (t * 2 * dn)))              # heads at a time
        for h0 in range(0, h, g):
            h1 = min(h, h0 + g)
            k = torch.matmul(c[:, :r], wk[h0:h1].transpose(1, 2).contiguous())
            k = torch.cat([k, c[None, :, r:].expand(h1 - h0, t, dr)], -1)
            v = torch.matmul(c[:, :r], wv[h0:h1])
            out[at:at + n, h0:h1] = _attend(q[h0:h1, at:at + n], k, v, t - n, scale).transpose(0, 1).to(torch.bfloat16)
        at += n
    return out


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def _turned(x, positions, f, amp, interleaved):
    """x as complex numbers times amp e^(i angle); x [..., T, r]."""
    r = x.shape[-1]
    z = torch.complex(x[..., 0::2], x[..., 1::2]) if interleaved else torch.complex(x[..., :r // 2], x[..., r // 2:])
    angle = positions.double()[:, None] * torch.as_tensor(f, device=x.device, dtype=torch.float64)
    z = z * torch.polar(torch.full_like(angle, amp), angle)
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        f, amp = _frequencies(case["rotary_dim"], case["base"], case["scaling"], case["factor"])
        y = s["x"].double()
        a, b = case["start"], case["start"] + case["rotary_dim"]
        y[..., a:b] = _turned(y[..., a:b].transpose(0, 1), s["positions"], f, amp, case["interleaved"]).transpose(0, 1)
        return y
    h, r, dr, dn, page = case["heads"], case["latent"], case["rope"], case["nope"], case["page"]
    if case["op"] == "store":
        f, amp = _frequencies(dr, 1e4, "", 1.0)
        c = s["latent"].double()
        c = c / torch.sqrt(torch.sum(c * c, -1, keepdim=True) / r + EPS) * s["norm"].double()
        k = _turned(s["k_rope"].double(), s["positions"], f, amp, case["interleaved"])
        pool = s["cache"].double()
        pool.view(-1, r + dr).index_copy_(0, s["slots"].long(), torch.cat([c, k], -1))
        q = _turned(s["q"][..., dn:].double().transpose(0, 1), s["positions"], f, amp, case["interleaved"])
        return {"cache": pool, "q_rope": q.transpose(0, 1)}
    scale = 1 / math.sqrt(dn + dr)
    w = s["w"].double().view(h, 2, dn, r)
    out = torch.empty((sum(s["new"]), h, dn), dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        c = _rows(s["cache"], s["table"][b], page, t).double()
        ct = c[:, :r].t().contiguous()
        for i in range(h):
            q = s["q"][at:at + n, i].double()
            k = torch.matmul(w[i, 0], ct)                          # [Dn, t]
            v = torch.matmul(w[i, 1], ct)
            for r0 in range(0, n, 2048):
                r1 = min(n, r0 + 2048)
                hi = t - n + r1
                x = (torch.matmul(q[r0:r1, :dn], k[:, :hi]) + torch.matmul(q[r0:r1, dn:], c[:hi, r:].t())) * scale
                past = torch.arange(hi, device=q.device)[None, :] - (t - n + torch.arange(r0, r1, device=q.device))[:, None]
                x = torch.softmax(torch.where(past > 0, -math.inf, x), -1)
                out[at + r0:at + r1, i] = torch.matmul(x, v[:, :hi].t())
        at += n
    return out
