"""Latent attention: long shares, refused arguments on the device, calls beside each other."""
from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 12, 64])
def test_decode_shares_longer_than_64_tiles(pkg, dev, page):
    """Enough cached tokens that every workgroup walks more than 64 tiles (its rows' addresses are made for 64 at a
    time), over pages that hold whole groups of eight rows and pages that do not."""
    seqs, n, heads, r, dr, dn = 16, 41001, 3, 256, 32, 64
    gen = torch.Generator(device=dev).manual_seed(page)
    per = -(-n // page)
    cache = torch.randn((seqs * per, page, r + dr), generator=gen, device=dev).to(torch.bfloat16)
    table = torch.randperm(seqs * per, generator=gen, device=dev).to(torch.int32).view(seqs, per)
    lengths = [n - 1000 * i for i in range(seqs)]
    lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    assert sum(-(-m // 32) for m in lengths) > 64 * 256
    q = (3 * torch.randn((seqs, heads, dn + dr), generator=gen, device=dev)).to(torch.bfloat16)
    w = (torch.randn((heads * 2 * dn, r), generator=gen, device=dev) * r ** -0.5).to(torch.bfloat16)
    weights = pkg.LatentWeights(w, num_heads=heads, nope_dim=dn, v_dim=dn)
    got = pkg.latent_decode_attention(q[..., :dn], q[..., dn:], cache, weights, table, lens, scale=0.1)
    wr = w.view(heads, 2, dn, r)
    for b in (0, 7, 15):
        rows = cache[table[b].long()].flatten(0, 1)[:lengths[b]]
        for h in (0, 2):
            o, s = ref.attend(q[b:b + 1, h, :dn], q[b:b + 1, h, dn:], rows, wr[h, 0], wr[h, 1], [lengths[b]], 0.1,
                              "absorbed")
            ref.check(got[b:b + 1, h], o, s, f"page {page} sequence {b} head {h}")


def _operands(dev, heads=2, tokens=3, r=512, dr=64, dn=128):
    def bf(*s):
        return torch.zeros(s, dtype=torch.bfloat16, device=dev)

    def i32(*s):
        return torch.zeros(s, dtype=torch.int32, device=dev)

    return bf, i32, dict(qn=bf(tokens, heads, dn), qr=bf(tokens, heads, dr), cache=bf(4, 16, r + dr),
                         w=bf(heads * 2 * dn, r), table=i32(tokens, 1), lens=i32(tokens), cu=i32(tokens + 1))


def test_weights_refused(pkg, dev):
    bf, _, o = _operands(dev)
    ok = dict(num_heads=2, nope_dim=128, v_dim=128)
    pkg.LatentWeights(o["w"], **ok)
    for w, kw in ((o["w"].float(), ok), (o["w"], dict(ok, num_heads=3)), (o["w"], dict(ok, nope_dim=96)),
                  (o["w"], dict(ok, v_dim=64)), (bf(512, 384), ok), (o["w"][None], ok),
                  (o["w"], dict(ok, num_heads=0))):
        with pytest.raises(ValueError):
            pkg.LatentWeights(w, **kw)
    # a transposed parameter is copied into place
    t = torch.randn((512, 512), device=dev).to(torch.bfloat16)
    a, b = pkg.LatentWeights(t.t(), **ok), pkg.LatentWeights(t.t().contiguous(), **ok)
    assert torch.equal(a.w_kv, b.w_kv) and torch.equal(a.w_uk_t, b.w_uk_t)


def test_decode_refused(pkg, dev):
    bf, i32, o = _operands(dev)
    w = pkg.LatentWeights(o["w"], num_heads=2, nope_dim=128, v_dim=128)

    def call(**kw):
        a = {**o, "scale": 0.1, **kw}
        return pkg.latent_decode_attention(a["qn"], a["qr"], a["cache"], w, a["table"], a["lens"], scale=a["scale"],
                                           **{k: kw[k] for k in ("out", "workspace") if k in kw})

    assert not call().any()
    for bad in (dict(qn=bf(3, 2, 64)), dict(qn=bf(3, 3, 128)), dict(qn=bf(4, 2, 128)), dict(qr=bf(3, 2, 32)),
                dict(qn=o["qn"].float()), dict(qn=o["qn"].transpose(0, 2)), dict(cache=bf(4, 16, 600)),
                dict(cache=bf(4, 576)), dict(table=i32(2, 1)), dict(table=i32(3, 1).long()), dict(lens=i32(2)),
                dict(lens=i32(3).long()), dict(lens=torch.zeros(3, dtype=torch.int32)), dict(out=bf(3, 2, 64)),
                dict(out=torch.zeros((3, 2, 128), device=dev)), dict(workspace=torch.zeros(1 << 20))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(pkg._lib.PagedAttentionError, match="scale"):
        call(scale=-1.0)
    with pytest.raises(pkg._lib.PagedAttentionError, match="aligned"):
        call(qn=bf(3, 2, 132)[..., 4:])
    # a workspace that is too small or off its alignment is replaced
    assert not call(workspace=torch.zeros(5, dtype=torch.uint8, device=dev)).any()
    assert not call(workspace=torch.zeros((1 << 22) + 1, dtype=torch.uint8, device=dev)[1:]).any()


def test_prefill_and_store_refused(pkg, dev):
    bf, i32, o = _operands(dev)
    w = pkg.LatentWeights(o["w"], num_heads=2, nope_dim=128, v_dim=128)
    call = lambda **kw: pkg.latent_prefill_attention(
        o["qn"], o["qr"], o["cache"], w, o["table"], kw.pop("cu", o["cu"]), kw.pop("cu_k", None), max_seqlen_q=3,
        scale=0.1, **kw)
    call()
    for bad in (dict(cu=i32(3)), dict(cu=o["cu"].long()), dict(cu_k=i32(2)), dict(kv_lens=i32(2)),
                dict(cu_k=o["cu"], kv_lens=i32(3)), dict(total_kv_tokens=-1), dict(total_kv_tokens=1 << 31)):
        with pytest.raises(ValueError):
            call(**bad)
    freqs = pkg.rotary_frequencies(64, 1e4, device=dev)
    store = lambda **kw: pkg.latent_store(
        kw.pop("latent", bf(3, 512)), kw.pop("k", bf(3, 64)), kw.pop("norm", None), kw.pop("pos", i32(3)),
        kw.pop("slots", torch.arange(3, dtype=torch.int32, device=dev)), o["cache"], kw.pop("freqs", freqs), **kw)
    store()
    for bad in (dict(latent=bf(3, 256)), dict(latent=bf(2, 512)), dict(k=bf(3, 32)), dict(norm=bf(256)),
                dict(pos=i32(2)), dict(slots=i32(3).long()), dict(freqs=pkg.rotary_frequencies(32, 1e4, device=dev)),
                dict(q_rope=bf(3, 2, 32)), dict(q_rope=bf(2, 2, 64)), dict(q_out=bf(3, 2, 64)),
                dict(q_rope=bf(3, 2, 64), q_out=bf(3, 3, 64)), dict(latent=bf(3, 512).float())):
        with pytest.raises(ValueError):
            store(**bad)


def test_store_checks_slots_on_request(pkg, dev, monkeypatch):
    bf, i32, o = _operands(dev)
    freqs = pkg.rotary_frequencies(64, 1e4, device=dev)
    monkeypatch.setenv("PA_CHECK_SLOTS", "1")
    with pytest.raises(ValueError, match="slot 5"):
        pkg.latent_store(bf(3, 512), bf(3, 64), None, i32(3), torch.tensor([5, 1, 5], dtype=torch.int32, device=dev),
                         o["cache"], freqs)


def test_calls_on_two_streams(pkg, dev):
    """Decode and prefill calls of different inputs in flight on two streams give what they give alone."""
    gen = torch.Generator(device=dev).manual_seed(2)
    heads, dn, dr, r = 8, 128, 64, 512
    w = pkg.LatentWeights((torch.randn((heads * 2 * dn, r), generator=gen, device=dev) * r ** -0.5).to(torch.bfloat16),
                          num_heads=heads, nope_dim=dn, v_dim=dn)
    cache = torch.randn((200, 16, r + dr), generator=gen, device=dev).to(torch.bfloat16)
    table = torch.randperm(200, generator=gen, device=dev).to(torch.int32).view(4, 50)
    lens = torch.tensor([800, 33, 500, 1], dtype=torch.int32, device=dev)
    qd = torch.randn((4, heads, dn + dr), generator=gen, device=dev).to(torch.bfloat16)
    qp = torch.randn((700, heads, dn + dr), generator=gen, device=dev).to(torch.bfloat16)
    cu = torch.tensor([0, 300, 301, 450, 700], dtype=torch.int32, device=dev)
    kv = torch.tensor([700, 1, 150, 800], dtype=torch.int32, device=dev)
    dec = lambda: pkg.latent_decode_attention(qd[..., :dn], qd[..., dn:], cache, w, table, lens, scale=0.1)
    pre = lambda: pkg.latent_prefill_attention(qp[..., :dn], qp[..., dn:], cache, w, table, cu, kv_lens=kv,
                                               max_seqlen_q=300, total_kv_tokens=1651, scale=0.1)
    want_d, want_p = dec(), pre()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        with torch.cuda.stream(a):
            got.append(dec())
            got.append(pre())
        with torch.cuda.stream(b):
            got.append(pre())
            got.append(dec())
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want_d if i % 4 in (0, 3) else want_p)


def test_copied_weights_and_frequencies_stand_alone(pkg, dev):
    """Deep copies bring their own memory: nothing of the originals is read through them."""
    import copy

    bf, i32, o = _operands(dev)
    gen = torch.Generator(device=dev).manual_seed(5)
    o["w"].copy_(torch.randn(o["w"].shape, generator=gen, device=dev))
    o["cache"].copy_(torch.randn(o["cache"].shape, generator=gen, device=dev))
    w = pkg.LatentWeights(o["w"], num_heads=2, nope_dim=128, v_dim=128)
    lens = torch.tensor([3, 16, 9], dtype=torch.int32, device=dev)
    call = lambda w: pkg.latent_decode_attention(o["qn"], o["qr"], o["cache"], w, o["table"], lens, scale=0.1)
    x = torch.randn((3, 2, 64), generator=gen, device=dev)
    f = pkg.rotary_frequencies(64, 1e4, device=dev)
    pos = torch.tensor([7, 100, 3], dtype=torch.int32, device=dev)
    want, turned = call(w), pkg.rotary_embedding(x, pos, f)
    w2, f2 = copy.deepcopy(w), copy.deepcopy(f)
    w.w_kv.zero_()
    w.w_uk_t.zero_()
    f.inv_freq.zero_()
    assert want.any() and torch.equal(call(w2), want)
    assert torch.equal(pkg.rotary_embedding(x, pos, f2), turned)


def test_prefill_no_rows_wanted_and_a_loose_bound(pkg, dev):
    """max_seqlen_q of zero computes nothing; one far above the tokens bounds nothing."""
    bf, i32, o = _operands(dev)
    gen = torch.Generator(device=dev).manual_seed(6)
    for t in (o["qn"], o["qr"], o["cache"], o["w"]):
        t.copy_(torch.randn(t.shape, generator=gen, device=dev))
    w = pkg.LatentWeights(o["w"], num_heads=2, nope_dim=128, v_dim=128)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    call = lambda m, **kw: pkg.latent_prefill_attention(
        o["qn"], o["qr"], o["cache"], w, i32(1, 1), cu, kv_lens=torch.full((1,), 3, dtype=torch.int32, device=dev),
        max_seqlen_q=m, total_kv_tokens=3, scale=0.01, **kw)
    assert not call(0).any()
    out = torch.full((3, 2, 128), 7.0, dtype=torch.bfloat16, device=dev)
    assert (call(0, out=out) == 7).all()
    assert call(3).any() and torch.equal(call(3), call(0x7fffffff))


@pytest.mark.parametrize("slots_apart", [False, True], ids=["pages-apart", "slots-apart"])
def test_offsets_past_32_bits(pkg, dev, slots_apart):
    """Rows of a pool, of q and of a rotated tensor more than 2^32 bytes apart: what a dense copy of them gives."""
    heads, r, dr, dn = 3, 256, 32, 64
    gen = torch.Generator(device=dev).manual_seed(8)
    big = torch.empty((1 << 32) + 4096, dtype=torch.bfloat16, device=dev)
    dense = torch.randn((4, 8, r + dr), generator=gen, device=dev).to(torch.bfloat16)
    strides = (1 << 9, (1 << 29) + 2048, 1) if slots_apart else ((1 << 30) + 1024, 304, 1)
    far = big.as_strided(dense.shape, strides)
    far.copy_(dense)
    w = pkg.LatentWeights((torch.randn((heads * 2 * dn, r), generator=gen, device=dev) * r ** -0.5).to(torch.bfloat16),
                          num_heads=heads, nope_dim=dn, v_dim=dn)
    table = torch.tensor([[3, 0, 2, 1], [1, 3, 0, 2]], dtype=torch.int32, device=dev)
    lens = torch.tensor([32, 27], dtype=torch.int32, device=dev)
    q = torch.randn((57, heads, dn + dr), generator=gen, device=dev).to(torch.bfloat16)
    cu = torch.tensor([0, 30, 57], dtype=torch.int32, device=dev)

    def decode(cache):
        return pkg.latent_decode_attention(q[:2, :, :dn], q[:2, :, dn:], cache, w, table, lens, scale=0.1)

    def prefill(cache, **kw):
        return pkg.latent_prefill_attention(q[..., :dn], q[..., dn:], cache, w, table, cu, kv_lens=lens,
                                            max_seqlen_q=30, scale=0.1, **kw)

    # (a loose bound of the kv lengths makes the expanded form the dearer one)
    route = pkg._lib.load().pa_latent_prefill_route
    assert [route(2, 57, 30, total, 4, 8, heads, r, dr, dn) for total in (59, 1 << 20)] == [0, 1]
    for call in (decode, lambda c: prefill(c, total_kv_tokens=59), lambda c: prefill(c, total_kv_tokens=1 << 20)):
        want = call(dense)
        assert want.any() and torch.equal(call(far), want)
    freqs = pkg.rotary_frequencies(dr, 1e4, device=dev)
    pos = torch.arange(4, dtype=torch.int32, device=dev)
    latent, k = dense[:, 0, :r], dense[:, 0, r:]
    slots = torch.tensor([31, 1, 9, 17], dtype=torch.int32, device=dev)
    pkg.latent_store(latent, k, None, pos, slots, dense, freqs)
    pkg.latent_store(far[:, 0, :r], far[:, 0, r:], None, pos, slots, far, freqs)
    assert torch.equal(far, dense)
    x = far.transpose(0, 1) if slots_apart else far
    assert torch.equal(pkg.rotary_embedding(x, pos.repeat(2)[:x.shape[0]], freqs),
                       pkg.rotary_embedding(x.contiguous(), pos.repeat(2)[:x.shape[0]], freqs))


def test_decode_uneven_units_in_wide_tables(pkg, dev):
    """Several row tiles a sequence, lengths from nothing to long, more table than tokens: shares that end before, in
    and behind a unit's counted start."""
    import test_gpu_latent_decode as dec

    lengths = [0, 1, 2999, 33, 1500, 64, 0, 640, 100, 2000, 31, 7]
    c = dec.make(dev, lengths, 130, 256, 32, 64, 16, seed=12, width=256)
    got = dec.run(pkg, c, 130, 64, 0.1)
    w = c["w"].view(130, 2, 64, 256)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not got[b].any()
            continue
        for h in (0, 63, 64, 127, 129):
            q = c["q"][b:b + 1, h]
            o, s = ref.attend(q[:, :64], q[:, 64:], c["rows"][b], w[h, 0], w[h, 1], [n], 0.1, "absorbed")
            ref.check(got[b:b + 1, h], o, s, f"sequence {b} head {h}")
    assert torch.equal(got, dec.run(pkg, c, 130, 64, 0.1))


def test_prefill_absorbed_many_uneven_units(pkg, dev):
    """New tokens of eight row tiles a sequence behind contexts of all lengths, one of them longer than its context."""
    import test_gpu_latent_prefill as pre

    seqs = [(30, 4000), (9, 900), (1, 3000), (17, 2500), (30, 20), (25, 64), (0, 700), (12, 3500)]
    c = pre.make(dev, seqs, 16, 256, 64, 128, 32, seed=13, behind=3)
    assert pre.form(pkg, c, 16, 256, 64, 128, 32) == "absorbed"
    for by in ("cu_k", "lens"):
        pre.check(pkg, c, pre.run(pkg, c, 16, 128, 0.1, lengths=by), 16, 256, 64, 128, 32, 0.1, some_heads=[0, 15])


def test_prefill_many_tokens_without_a_sequence(pkg, dev):
    """More rows than a workgroup zeroes, before and behind the sequences, in both forms."""
    import test_gpu_latent_prefill as pre

    for heads, seqs, want in ((2, [(70, 70), (600, 600)], "expanded"), (16, [(4, 300), (3, 200)], "absorbed")):
        c = pre.make(dev, seqs, heads, 256, 32, 64, 16, seed=14, before=700, behind=1100)
        assert pre.form(pkg, c, heads, 256, 32, 64, 16) == want
        pre.check(pkg, c, pre.run(pkg, c, heads, 64, 0.1), heads, 256, 32, 64, 16, 0.1, some_heads=[0, heads - 1],
                  some_rows=20)
