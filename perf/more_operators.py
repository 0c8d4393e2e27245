"""Performance cases of decode over long cached contexts that reads less than all of them: attention of a batch whose
sequences share a prefix, and attention over the blocks of a context that a cheap score selects for each query.

``listed()`` names the cases, ``draw()`` makes further ones over the same ranges.  ``run()`` computes a case through
the package's public entry points where ``own`` is true, else in plain torch operations in 32 bits.

A case is a dict of plain values; ``op`` says which operator it calls:

  "bounds"    update_block_bounds: the elementwise minimum and maximum of the keys of every block that got new tokens
  "scores"    block_scores: for each sequence, kv head and block the largest bound of the logits of its q heads
  "select"    select_blocks: the first and the last blocks and those of the largest scores, ascending
  "sparse"    block_sparse_decode_attention: one new token a sequence over the selected blocks of its context
  "shared"    shared_prefix_attention: new tokens of sequences that share their first pages in groups

  heads, kv_heads, dim, page, block   block: tokens of a block, a part of a page
  seqs, ctx_lo .. ctx_hi              sequences and their tokens (shared: own tokens behind the prefix, new included)
  new_lo .. new_hi                    new tokens a sequence
  picks, first, recent                blocks selected, of which the first and the last always
  groups, prefix_lo .. prefix_hi      groups of sequences (seqs in all) and their prefixes, in whole pages
  lens        seeds the lengths, which are part of the case; values and page placement come from the seed
"""
import math
import random

import numpy as np
import torch

own = False


def _package():
    """``vllm-jax_amd/`` under its module name (the folder's hyphen needs an import by path)."""
    import __graft_entry__
    return __graft_entry__.load_package()


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _case(op, heads, kv_heads, page, *, dim=128, block=0, seqs=1, ctx=(1, 1), new=(1, 1), picks=0, first=1, recent=2,
          groups=0, prefix=(0, 0), ties=False, lens=0, name=None):
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, block=block, seqs=seqs, ctx_lo=ctx[0],
             ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1], picks=picks, first=first, recent=recent, groups=groups,
             prefix_lo=prefix[0], prefix_hi=prefix[1], ties=ties, lens=lens)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # A decode step's new tokens of the serving batch, 256-token pages in blocks of 32.
        _case("bounds", 32, 8, 256, block=32, seqs=256, ctx=(512, 8192), lens=1, name="bounds_step"),
        # A batch of prompts of odd lengths, 64-token pages in blocks of 16.
        _case("bounds", 32, 8, 64, block=16, seqs=8, ctx=(4000, 9000), new=(1000, 4000), lens=2,
              name="bounds_prompts"),
        # Scores of a small step: eight chats over 16-token pages, a block a page.
        _case("scores", 16, 8, 16, block=16, seqs=8, ctx=(500, 4000), lens=3, name="scores_step"),
        # Scores of a batch of long contexts: bound by the reads of the block bounds.
        _case("scores", 32, 8, 256, block=32, seqs=64, ctx=(16384, 65536), lens=4, name="scores_batch"),
        # The selection of a small step: few blocks, few kv heads.
        _case("select", 16, 8, 16, block=16, seqs=4, ctx=(1000, 4000), picks=64, lens=5, name="select_step"),
        # The selection of a batch of long contexts.
        _case("select", 32, 8, 256, block=32, seqs=64, ctx=(32768, 131072), picks=128, lens=6, name="select_batch"),
        # One user's 128k-token conversation, 2048 tokens of it read.
        _case("sparse", 32, 8, 64, block=32, seqs=1, ctx=(131072, 131072), picks=64, lens=7, name="sparse_one_long"),
        # The serving batch at long contexts, 2048 tokens a sequence read.
        _case("sparse", 32, 8, 256, block=32, seqs=128, ctx=(8192, 32768), picks=64, lens=8, name="sparse_batch"),
        # Four chats behind one system prompt: latency.
        _case("shared", 32, 8, 256, seqs=4, ctx=(17, 300), groups=1, prefix=(2048, 2048), lens=9, name="shared_few"),
        # A serving batch behind one long prompt.
        _case("shared", 32, 8, 256, seqs=128, ctx=(64, 1024), groups=1, prefix=(8192, 8192), lens=10,
              name="shared_batch"),
        # Drafted tokens to verify, five a sequence, behind four prefixes.
        _case("shared", 64, 8, 64, seqs=32, ctx=(100, 700), new=(5, 5), groups=4, prefix=(4096, 16384), lens=11,
              name="shared_drafts"),
        # The largest: many questions about one long document.
        _case("shared", 32, 8, 256, seqs=64, ctx=(20, 100), new=(20, 100), groups=1, prefix=(32768, 32768), lens=12,
              name="shared_questions"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: any operator, the heads of the engine's models, its page sizes, lengths over the logarithm of
    their range."""
    op = rng.choice(["bounds", "scores", "select", "sparse", "sparse", "shared", "shared", "shared"])
    heads, kv_heads = rng.choice([(8, 1), (16, 8), (32, 8), (32, 8), (64, 8), (32, 32), (24, 4)])
    page = rng.choice([16, 32, 64, 256])
    lens = rng.randrange(1 << 20)
    if op == "shared":
        n = _log_int(rng, 1, 256)
        new_hi = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 128)])
        own_hi = max(new_hi, _log_int(rng, 1, 2048))
        p = _log_int(rng, 16, 32768)
        c = _case("shared", heads, kv_heads, page, seqs=n, ctx=(max(1, own_hi // rng.choice([1, 4, 16])), own_hi),
                  new=(max(1, new_hi // rng.choice([1, 3])), new_hi), groups=max(1, n // rng.choice([1, 4, 16, n])),
                  prefix=(p // rng.choice([1, 2]), p), lens=lens)
        while work(c)["flops"] > 2e12 or work(c)["bytes"] > 2e9:  # below the largest listed case
            c.update(seqs=max(1, c["seqs"] // 2), prefix_lo=c["prefix_lo"] // 2, prefix_hi=c["prefix_hi"] // 2)
            c["groups"] = min(c["groups"], c["seqs"])
        return c
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    dim = rng.choice([64, 128, 128, 256])
    n = _log_int(rng, 1, 256)
    hi = _log_int(rng, 1, max(64, min(131072, 2_000_000 // n)))
    ctx = (max(1, hi // rng.choice([1, 2, 16])), hi)
    if op == "bounds":
        new_hi = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, min(hi, 32768 // n)))
        return _case(op, heads, kv_heads, page, dim=dim, block=block, seqs=n, ctx=ctx,
                     new=(max(1, new_hi // 2), new_hi), lens=lens)
    first, recent = rng.choice([(1, 2), (0, 1), (4, 4), (0, 0)])
    return _case(op, heads, kv_heads, page, dim=dim, block=block, seqs=n, ctx=ctx,
                 picks=max(1, first + recent, _log_int(rng, 1, 256)), first=first, recent=recent,
                 ties=rng.random() < 0.5, lens=lens)


def _lengths(case):
    """Per sequence: new tokens, all tokens, tokens shared with its group."""
    rng = random.Random(case["lens"])
    n = case["seqs"]
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(n)]
    new = [min(c, rng.randint(case["new_lo"], case["new_hi"])) for c in ctx]
    if case["op"] != "shared":
        return new, ctx, [0] * n
    shared = []
    for s0, s1 in zip(*_groups(case)):
        p = rng.randint(case["prefix_lo"], case["prefix_hi"]) // case["page"] * case["page"]
        shared += [p] * (s1 - s0)
    return new, [c + p for c, p in zip(ctx, shared)], shared


def _groups(case):
    """First and last sequence of each group."""
    at = [case["seqs"] * g // case["groups"] for g in range(case["groups"] + 1)]
    return at[:-1], at[1:]


def _counts(case, lengths):
    """Blocks of each sequence, and how many of them are selected."""
    blocks = [-(-t // case["block"]) for t in lengths]
    return blocks, [min(b, case["picks"]) for b in blocks]


def work(case):
    new, total, shared = _lengths(case)
    h, kv, d, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    row = 2 * kv * d                                              # bytes of one token's keys
    seqs, tokens = case["seqs"], sum(new)
    if case["op"] == "bounds":
        touched = sum((t - 1) // block - (t - n) // block + 1 for n, t in zip(new, total))
        old = sum((t - n) % block != 0 for n, t in zip(new, total))
        return {"bytes": tokens * row + (touched + old) * 2 * row + 4 * sum(-(-t // page) for t in total),
                "flops": 2 * tokens * kv * d}
    q_bytes = 2 * tokens * h * d
    if case["op"] == "shared":
        flops = sum(4 * h * d * (n * (t - n) + n * (n + 1) // 2) for n, t in zip(new, total))
        cached = sum(t - p for t, p in zip(total, shared)) + sum(shared[s] for s in _groups(case)[0])
        return {"bytes": cached * 2 * row + 2 * q_bytes + 4 * cached // page, "flops": flops}
    blocks, picks = _counts(case, total)
    if case["op"] == "scores":
        return {"bytes": sum(blocks) * (2 * row + 4 * kv) + q_bytes, "flops": 4 * sum(blocks) * h * d}
    if case["op"] == "select":
        return {"bytes": 4 * kv * (sum(blocks) + seqs * case["picks"]), "flops": kv * sum(blocks)}
    read = sum(min(t, p * block) for t, p in zip(total, picks))
    return {"bytes": read * 2 * row + 2 * q_bytes + 4 * kv * seqs * case["picks"], "flops": 4 * read * h * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(shape, gen, dev, dtype=torch.bfloat16):
    t = torch.empty(shape, dtype=dtype, device=dev)
    flat = t.view(-1)
    step = 1 << 28
    for s in range(0, flat.numel(), step):
        n = min(step, flat.numel() - s)
        flat[s:s + n] = torch.randn(n, generator=gen, device=dev, dtype=torch.float32)
    return t


def _layout(case, gen, dev):
    """Block tables (-1 padded) as a scheduler lays them out: pages in a random order over the pool, a group's prefix
    pages in the table of each of its sequences."""
    new, total, shared = _lengths(case)
    bs = case["page"]
    pages = [-(-t // bs) for t in total]
    starts = set(_groups(case)[0]) if case["op"] == "shared" else set(range(len(total)))
    num_pages = sum(p - (0 if i in starts else s // bs) for i, (p, s) in enumerate(zip(pages, shared)))
    num_pages += num_pages // 8 + 1               # a pool is never quite full
    perm = torch.randperm(num_pages, generator=gen, device=dev).to(torch.int32).cpu().numpy()
    table = np.full((len(total), max(pages)), -1, np.int32)
    at = 0
    for i, (p, s) in enumerate(zip(pages, shared)):
        have = 0
        if i not in starts:
            have = s // bs
            table[i, :have] = table[i - 1, :have]
        table[i, have:p] = perm[at:at + p - have]
        at += p - have
    i32 = lambda a: torch.as_tensor(np.ascontiguousarray(a, dtype=np.int32), device=dev)  # noqa: E731
    return dict(num_pages=num_pages, new=new, total=total, shared=shared, table=i32(table), lens=i32(total),
                cu_q=i32(np.concatenate([[0], np.cumsum(new)])))


def _choice(case, total, gen, dev):
    """Blocks that a selection leaves: the first, the last and random ones between, ascending, -1 behind them."""
    s = torch.full((case["seqs"], case["kv_heads"], case["picks"]), -1, dtype=torch.int32, device=dev)
    for b, n in enumerate(_counts(case, total)[0]):
        k = min(n, case["picks"])
        r = torch.rand((case["kv_heads"], n), generator=gen, device=dev)
        if k == case["picks"]:
            r[:, :case["first"]] = 2
            r[:, n - case["recent"]:] = 2
        s[b, :, :k] = torch.sort(torch.argsort(r, -1, descending=True)[:, :k], -1).values.to(torch.int32)
    return s


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = dict(case=case)
    h, kv, d, bs, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    if own:
        s["pa"] = _package()
    if case["op"] == "select":
        total = _lengths(case)[1]
        width = -(-max(total) // bs) * (bs // block)
        x = torch.randn((case["seqs"], kv, width), generator=gen, device=dev) * 20
        s["scores"] = torch.round(x) if case["ties"] else x
        s["total"], s["lens"] = total, torch.as_tensor(total, dtype=torch.int32, device=dev)
        return s
    s.update(_layout(case, gen, dev))
    if case["op"] == "scores":
        # the bounds of keys of about unit size: a minimum below, a maximum above
        x = _randn((s["num_pages"], bs // block, kv, 2, d), gen, dev)
        s["bounds"] = torch.stack([x.amin(3), x.amax(3)], 3)
    else:
        s["cache"] = _randn((2, s["num_pages"], bs, kv, d), gen, dev)
    if case["op"] == "bounds":
        s["bounds"] = torch.zeros((s["num_pages"], bs // block, kv, 2, d), dtype=torch.bfloat16, device=dev)
        return s
    s["q"] = _randn((sum(s["new"]), h, d), gen, dev)
    if case["op"] == "sparse":
        s["selected"] = _choice(case, s["total"], gen, dev)
    if case["op"] == "shared":
        first, last = _groups(case)
        i32 = lambda a: torch.as_tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
        s["cu_groups"], s["shared_lens"] = i32(first + last[-1:]), i32([s["shared"][b] for b in first])
        if own:
            s["prefixes"] = s["pa"].SharedPrefixes(s["cu_groups"], s["shared_lens"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)(s, case)


def _run_own(s, case):
    pa = s["pa"]
    scale = case["dim"] ** -0.5
    if case["op"] == "bounds":
        return pa.update_block_bounds(s["bounds"], s["cache"], s["table"], s["lens"],
                                      None if case["new_hi"] == 1 else s["cu_q"], max_seqlen_q=max(s["new"]))
    if case["op"] == "scores":
        return pa.block_scores(s["q"], s["bounds"], s["table"], s["lens"], page_size=case["page"], scale=scale)
    if case["op"] == "select":
        return pa.select_blocks(s["scores"], s["lens"], case["picks"], block=case["block"], first=case["first"],
                                recent=case["recent"])
    if case["op"] == "sparse":
        return pa.block_sparse_decode_attention(s["q"], s["cache"], s["table"], s["lens"], s["selected"],
                                                block=case["block"], scale=scale)
    return pa.shared_prefix_attention(s["q"], s["cache"], s["table"], s["lens"], s["prefixes"],
                                      None if case["new_hi"] == 1 else s["cu_q"], max_seqlen_q=max(s["new"]),
                                      scale=scale)


def _rows(pool, table, t0, t1):
    """Rows [t0, t1) of one sequence of a pool half ``[NB, BS, Hkv, d]`` as ``[Hkv, t1 - t0, d]`` in 32 bits."""
    t = torch.arange(t0, t1, device=pool.device)
    page = table[t // pool.shape[1]].long()
    return pool[page, t % pool.shape[1]].transpose(0, 1).float()


def _part(q, k, v, scale, limit=None):
    """Unnormalised attention of q [Hkv, n, d] to k, v [Hkv, L, d]: sums, maxima and weighted values.  ``limit`` [n]:
    the keys that each row sees."""
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
    if limit is not None:
        x.masked_fill_(torch.arange(k.shape[1], device=q.device) >= limit[:, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - m)
    return m, x.sum(-1, keepdim=True), torch.matmul(x, v)


def _run_plain(s, case):
    h, kv, d, bs, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    g, scale = h // kv, d ** -0.5
    if case["op"] == "bounds":
        keys = s["cache"][0].view(-1, block, kv, d)               # blocks of the pool
        out = s["bounds"].view(-1, kv, 2, d)
        per = bs // block
        for b, (n, t) in enumerate(zip(s["new"], s["total"])):
            j = torch.arange((t - n) // block, -(-t // block), device=keys.device)
            at = s["table"][b][j // per].long() * per + j % per
            k = keys[at].float()                                  # [blocks, block, Hkv, d]
            past = (j[:, None] * block + torch.arange(block, device=keys.device) >= t)[:, :, None, None]
            lo = k.masked_fill(past, float("inf")).amin(1)
            hi = k.masked_fill(past, float("-inf")).amax(1)
            out[at] = torch.stack([lo, hi], 2).to(torch.bfloat16)
        return s["bounds"]
    if case["op"] == "select":
        out = torch.full((case["seqs"], kv, case["picks"]), -1, dtype=torch.int32, device=s["scores"].device)
        for b, n in enumerate(_counts(case, s["total"])[0]):
            k = min(n, case["picks"])
            x = s["scores"][b, :, :n].clone()
            if k < n:
                x[:, :case["first"]] = float("inf")
                x[:, n - case["recent"]:] = float("inf")
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
            out[b, :, :k] = torch.sort(order, -1).values.to(torch.int32)
        return out
    q = s["q"].float().view(-1, kv, g, d)
    if case["op"] == "scores":
        per = bs // block
        out = torch.full((case["seqs"], kv, s["table"].shape[1] * per), float("-inf"), device=q.device)
        for b, n in enumerate(_counts(case, s["total"])[0]):
            j = torch.arange(n, device=q.device)
            x = s["bounds"][s["table"][b][j // per].long(), j % per].float()       # [n, Hkv, 2, d]
            x = x.permute(1, 2, 3, 0).contiguous()                                 # [Hkv, 2, d, n]
            up = torch.matmul(q[b].clamp(min=0), x[:, 1]) + torch.matmul(q[b].clamp(max=0), x[:, 0])
            out[b, :, :n] = up.amax(1) * scale
        return out
    if case["op"] == "sparse":
        out = torch.empty((case["seqs"], kv, g, d), dtype=torch.bfloat16, device=q.device)
        heads = torch.arange(kv, device=q.device)[:, None]
        for b, (n, t) in enumerate(zip(_counts(case, s["total"])[1], s["total"])):
            pos = s["selected"][b, :, :n].long()[:, :, None] * block + torch.arange(block, device=q.device)
            pos = pos.flatten(1)                                  # [Hkv, tokens]
            hidden = pos >= t
            pos = pos.clamp(max=t - 1)
            page = s["table"][b][pos // bs].long()
            k, v = (s["cache"][i][page, pos % bs, heads].float() for i in (0, 1))  # [Hkv, tokens, d]
            x = torch.matmul(q[b], k.transpose(1, 2).contiguous()) * scale
            x = x.masked_fill_(hidden[:, None], float("-inf"))
            x = torch.exp(x - x.amax(-1, keepdim=True))
            out[b] = (torch.matmul(x, v) / x.sum(-1, keepdim=True)).to(torch.bfloat16)
        return out.view(-1, h, d)
    out = torch.empty((q.shape[0], kv, g, d), dtype=torch.bfloat16, device=q.device)
    at = np.concatenate([[0], np.cumsum(s["new"])]).tolist()
    for s0, s1 in zip(*_groups(case)):
        p, t0 = s["shared"][s0], at[s0]
        rows = q[t0:at[s1]].transpose(0, 1).contiguous()          # [Hkv, tokens, G, d]
        prefix = None
        if p:
            k, v = _rows(s["cache"][0], s["table"][s0], 0, p), _rows(s["cache"][1], s["table"][s0], 0, p)
            flat = rows.view(kv, -1, d)
            step = max(1, (1 << 28) // (kv * p))
            parts = [_part(flat[:, r:r + step], k, v, scale) for r in range(0, flat.shape[1], step)]
            prefix = [torch.cat(x, 1).view(kv, rows.shape[1], g, -1) for x in zip(*parts)]
        for b in range(s0, s1):
            n, t, i = s["new"][b], s["total"][b], at[b] - t0
            k, v = _rows(s["cache"][0], s["table"][b], p, t), _rows(s["cache"][1], s["table"][b], p, t)
            limit = torch.arange(t - p - n + 1, t - p + 1, device=q.device).repeat_interleave(g)
            m, l, o = (x.view(kv, n, g, -1) for x in _part(rows[:, i:i + n].reshape(kv, n * g, d), k, v, scale, limit))
            if prefix is not None:
                pm, pl, po = (x[:, i:i + n] for x in prefix)
                top = torch.maximum(m, pm)
                a, c = torch.exp(m - top), torch.exp(pm - top)
                l, o = l * a + pl * c, o * a + po * c
            out[at[b]:at[b + 1]] = (o / l).transpose(0, 1).to(torch.bfloat16)
    return out.view(-1, h, d)


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    h, kv, d, bs, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    if case["op"] == "select":
        x = s["scores"].cpu().numpy()
        out = np.full((case["seqs"], kv, case["picks"]), -1, np.int32)
        for b, t in enumerate(s["total"]):
            n = (t + block - 1) // block
            for j in range(kv):
                keep = list(range(n))
                if n > case["picks"]:
                    last = n - case["recent"]
                    middle = np.arange(case["first"], last)
                    # by falling score, then by rising index
                    order = middle[np.lexsort((middle, -x[b, j, middle].astype(np.float64)))]
                    keep = sorted([*range(case["first"]), *order[:case["picks"] - case["first"] - case["recent"]],
                                   *range(last, n)])
                out[b, j, :len(keep)] = keep
        return torch.as_tensor(out)
    table = s["table"].cpu().numpy()
    dev = s["table"].device
    if case["op"] == "bounds":
        out = s["bounds"].double()
        for b, (n, t) in enumerate(zip(s["new"], s["total"])):
            for j in range((t - n) // block, (t - 1) // block + 1):
                page, at = int(table[b, j * block // bs]), j * block % bs
                x = s["cache"][0, page, at:at + min(block, t - j * block)].double()
                out[page, at // block, :, 0], out[page, at // block, :, 1] = x.min(0).values, x.max(0).values
        return out
    q = s["q"].double()
    if case["op"] == "scores":
        out = torch.full((case["seqs"], kv, table.shape[1] * (bs // block)), -math.inf, dtype=torch.float64, device=dev)
        for b, t in enumerate(s["total"]):
            n = -(-t // block)
            x = s["bounds"][s["table"][b, :-(-t // bs)].long()].flatten(0, 1)[:n].double()   # [n, Hkv, 2, d]
            for j in range(kv):
                best = None
                for i in range(h // kv):
                    row = q[b, j * (h // kv) + i]
                    up = torch.maximum(row * x[:, j, 0], row * x[:, j, 1]).sum(-1)
                    best = up if best is None else torch.maximum(best, up)
                out[b, j, :n] = best / math.sqrt(d)
        return out
    out = torch.empty((sum(s["new"]), h, d), dtype=torch.float64, device=dev)
    chosen = s["selected"].cpu().numpy() if case["op"] == "sparse" else None
    at = 0
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        pages = s["table"][b, :-(-t // bs)].long()
        if chosen is None:
            context = s["cache"][:, pages].flatten(1, 2)[:, :t]
        for j in range(kv):
            if chosen is None:
                k, v = context[0, :, j].double(), context[1, :, j].double()
                seen = t - n + 1 + torch.arange(n, device=dev)
            else:
                pos = np.concatenate([np.arange(c * block, min(t, (c + 1) * block)) for c in chosen[b, j] if c >= 0])
                pos = torch.as_tensor(pos, device=dev)
                k, v = (s["cache"][i, pages[pos // bs], pos % bs, j].double() for i in (0, 1))
                seen = torch.full((1,), k.shape[0], device=dev)
            rows = q[at:at + n, j * (h // kv):(j + 1) * (h // kv)].reshape(-1, d)
            seen = seen.repeat_interleave(h // kv)
            o = torch.empty_like(rows)
            step = max(1, (1 << 27) // k.shape[0])
            for r in range(0, rows.shape[0], step):
                x = torch.matmul(rows[r:r + step], k.t()) / math.sqrt(d)
                x[torch.arange(k.shape[0], device=dev)[None, :] >= seen[r:r + step, None]] = -math.inf
                o[r:r + step] = torch.matmul(torch.softmax(x, -1), v)
            out[at:at + n, j * (h // kv):(j + 1) * (h // kv)] = o.view(n, h // kv, d)
        at += n
    return out
