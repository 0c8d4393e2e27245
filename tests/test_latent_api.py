"""The latent-attention and rotation entries without a device: the C ABI's refusals, the package's argument checks, the
frequencies, the prefill's choice of form."""
from __future__ import annotations

import math

import pytest
import torch

import latent_reference as ref
from conftest import PKG

LIB = PKG._lib.load()
FAKE = 0x10000  # 16-byte aligned, never dereferenced on the host


def _err():
    return LIB.pa_last_error().decode()


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------
def _rotary(**over):
    a = dict(dtype=0, x=FAKE, xt=64, xh=64, pos=FAKE, freq=FAKE, amp=1.0, tokens=2, heads=1, dim=64, start=0, rot=64,
             inter=0, out=2 * FAKE, ot=64, oh=64, stream=None)
    a.update(over)
    return LIB.pa_rotary_embedding(*a.values())


def test_rotary_refusals():
    assert _rotary(tokens=0) == 0
    assert _rotary(tokens=-1) == -1 and "num_tokens=-1" in _err()
    assert _rotary(heads=0) == -1
    assert _rotary(rot=63) == -1 and "even part" in _err()
    assert _rotary(rot=0) == -1
    assert _rotary(start=1) == -1
    assert _rotary(start=-2, rot=32) == -1
    assert _rotary(dim=1024, rot=514) == -2 and "514" in _err()
    assert _rotary(dtype=3) == -2
    assert _rotary(heads=1 << 20) == -2 and "2^24" in _err()
    assert _rotary(x=None) == -1 and "null" in _err()
    assert _rotary(out=FAKE, ot=128) == -1 and "in place" in _err()


def _store(**over):
    a = dict(latent=FAKE, lt=512, k=FAKE, kt=64, w=FAKE, eps=1e-6, freq=FAKE, amp=1.0, inter=1, pos=FAKE, slots=FAKE,
             tokens=2, r=512, dr=64, q=FAKE, qt=64, qh=64, heads=1, qo=FAKE, qot=64, qoh=64, cache=FAKE, pages=1, page=16,
             ps=16 * 576, ss=576, stream=None)
    a.update(over)
    return LIB.pa_latent_store(*a.values())


def test_store_refusals():
    assert _store(tokens=0) == 0
    assert _store(tokens=-1) == -1
    assert _store(pages=0) == -1
    assert _store(page=0) == -1
    for r, dr in ((384, 64), (512, 48), (1024, 64), (0, 64), (512, 0)):
        assert _store(r=r, dr=dr) == -2 and "not supported" in _err()
    assert _store(eps=float("nan")) == -1
    assert _store(eps=-1.0) == -1
    assert _store(heads=2, q=None) == -1 and "null" in _err()
    assert _store(cache=None) == -1
    assert _store(cache=FAKE + 8) == -2 and "aligned" in _err()
    assert _store(lt=513) == -2
    assert _store(qh=68) == -2


def _decode(**over):
    a = dict(qn=FAKE, qnt=2048, qnh=128, qr=FAKE, qrt=1024, qrh=64, cache=FAKE, pages=4, page=16, ps=16 * 576, ss=576,
             bt=FAKE, bts=4, pps=4, lens=FAKE, batch=2, heads=16, r=512, dr=64, dn=128, dv=128, ukt=FAKE, kv=FAKE,
             scale=0.1, out=FAKE, ot=2048, oh=128, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(over)
    return LIB.pa_latent_decode(*a.values())


def test_decode_refusals():
    assert _decode(batch=0) == 0
    assert _decode(batch=-1) == -1
    assert _decode(heads=0) == -1
    assert _decode(pages=0) == -1
    for over in (dict(r=128), dict(dr=16), dict(dn=96, dv=96), dict(dv=64), dict(heads=70000)):
        assert _decode(**over) == -2, over
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert _decode(scale=scale) == -1 and "scale" in _err()
    for name in ("qn", "qr", "cache", "lens", "ukt", "kv", "out", "bt"):
        assert _decode(**{name: None}) == -1 and "null" in _err(), name
    assert _decode(qn=FAKE + 2) == -2
    assert _decode(ss=577) == -2
    assert _decode(batch=20000) == -2 and "16384" in _err()
    assert _decode(batch=16384, pps=1 << 27) == -2 and "2^31" in _err()
    need = LIB.pa_latent_decode_workspace_size(2, 16, 512, 4, 16)
    assert need > 2 * 2 * 16 * 512 * 2
    assert _decode(wsb=need - 1) == -3 and str(need) in _err()
    assert _decode(ws=None) == -3
    assert LIB.pa_latent_decode_workspace_size(-1, 16, 512, 4, 16) == 0


def _prefill(**over):
    a = dict(qn=FAKE, qnt=2048, qnh=128, qr=FAKE, qrt=1024, qrh=64, cache=FAKE, pages=4, page=16, ps=16 * 576, ss=576,
             bt=FAKE, bts=4, pps=4, cuq=FAKE, cuk=FAKE, lens=None, batch=2, tokens=10, maxq=5, total=20, heads=16, r=512,
             dr=64, dn=128, dv=128, ukt=FAKE, kv=FAKE, scale=0.1, zero=1, out=FAKE, ot=2048, oh=128, ws=FAKE,
             wsb=1 << 40, stream=None)
    a.update(over)
    return LIB.pa_latent_prefill(*a.values())


def test_prefill_refusals():
    assert _prefill(tokens=0) == 0
    assert _prefill(batch=0, zero=0) == 0
    for name in ("batch", "tokens", "maxq", "total", "pps"):
        assert _prefill(**{name: -1}) == -1, name
    assert _prefill(heads=0) == -1
    for over in (dict(r=128), dict(dr=16), dict(dn=96, dv=96), dict(dv=64), dict(heads=70000)):
        assert _prefill(**over) == -2, over
    assert _prefill(scale=0.0) == -1
    assert _prefill(lens=FAKE) == -1 and "one of" in _err()
    assert _prefill(cuk=None) == -1
    for name in ("qn", "qr", "cache", "cuq", "ukt", "kv", "out", "bt"):
        assert _prefill(**{name: None}) == -1 and "null" in _err(), name
    assert _prefill(out=FAKE + 8) == -2
    assert _prefill(oh=132) == -2
    args = (2, 10, 5, 20, 4, 16, 16, 512, 64, 128)
    need = LIB.pa_latent_prefill_workspace_size(*args)
    assert need > 0 and _prefill(wsb=need - 1) == -3
    assert LIB.pa_latent_prefill_workspace_size(2, 10, 5, 20, 4, 16, 16, 512, 16, 128) == 0
    assert LIB.pa_latent_prefill_route(2, 10, 5, -20, 4, 16, 16, 512, 64, 128) == -1


def test_prefill_route_and_workspace():
    """Many new tokens are expanded, few behind long contexts absorbed; K and V of at most 2 GiB at a time."""
    route = lambda batch, new, kv, heads=32: LIB.pa_latent_prefill_route(  # noqa: E731
        batch, batch * new, new, batch * kv, -(-kv // 64), 64, heads, 512, 64, 128)
    expanded, absorbed = PKG._lib.PA_LATENT_EXPANDED, PKG._lib.PA_LATENT_ABSORBED
    assert route(1, 4096, 4096) == expanded
    assert route(8, 512, 8192) == expanded
    assert route(8, 8, 8192) == absorbed
    assert route(1, 1, 1 << 17) == absorbed
    assert route(1, 1, 1) == expanded                    # one row: nothing to expand
    # a batch past the absorbed kernel's is expanded whatever its shape
    assert route(20000, 1, 64) == expanded
    size = lambda t, heads: LIB.pa_latent_prefill_workspace_size(1, 4096, 4096, t, t // 64 + 1, 64, heads, 512, 64, 128)  # noqa: E731
    assert size(1 << 20, 128) < (2 << 30) + (1 << 20) * 128 + 4096
    assert size(4096, 16) >= 4096 * (16 * 512 + 128)
    assert size(1 << 24, 128) >= (1 << 24) * 512         # at least one head at a time


# ---------------------------------------------------------------------------
# frequencies
# ---------------------------------------------------------------------------
def test_frequencies():
    f = PKG.rotary_frequencies(64, 1e4, device="cpu")
    assert f.rotary_dim == 64 and f.amplitude == 1.0 and f.inv_freq.dtype == torch.float64
    want = torch.tensor([1e4 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert torch.allclose(f.inv_freq, want, rtol=1e-14, atol=0)
    lin = PKG.rotary_frequencies(64, 1e4, scaling=dict(type="linear", factor=4), device="cpu")
    assert torch.allclose(lin.inv_freq, want / 4, rtol=1e-14, atol=0)
    ntk = PKG.rotary_frequencies(64, 1e4, scaling=dict(type="ntk", factor=8), device="cpu")
    assert math.isclose(float(ntk.inv_freq[0]), 1.0) and math.isclose(float(ntk.inv_freq[31]), float(want[31]) / 8,
                                                                      rel_tol=1e-12)
    yarn = PKG.rotary_frequencies(64, 1e4, scaling=dict(type="yarn", factor=32, original_max_position=4096), device="cpu")
    assert torch.allclose(yarn.inv_freq, torch.tensor(ref.yarn_frequencies(64, 1e4, 32, 4096), dtype=torch.float64),
                          rtol=1e-13, atol=0)
    assert math.isclose(yarn.amplitude, 0.1 * math.log(32) + 1)
    assert float(yarn.inv_freq[0]) == 1.0 and math.isclose(float(yarn.inv_freq[31]), float(want[31]) / 32, rel_tol=1e-12)
    own = PKG.rotary_frequencies(64, 1e4, scaling=dict(type="yarn", factor=32, original_max_position=4096,
                                                       attention_factor=1.5, beta_fast=16, beta_slow=2), device="cpu")
    assert own.amplitude == 1.5
    assert torch.allclose(own.inv_freq, torch.tensor(ref.yarn_frequencies(64, 1e4, 32, 4096, 16, 2),
                                                     dtype=torch.float64), rtol=1e-13, atol=0)


@pytest.mark.parametrize("args,kw", [
    ((63, 1e4), {}), ((0, 1e4), {}), ((514, 1e4), {}), ((64, 0.0), {}), ((64, float("inf")), {}),
    ((64, 1e4), dict(scaling=dict(type="dynamic", factor=2))), ((64, 1e4), dict(scaling=dict(factor=2))),
    ((64, 1e4), dict(scaling=dict(type="linear", factor=0))), ((2, 1e4), dict(scaling=dict(type="ntk", factor=2))),
    ((64, 1e4), dict(scaling=dict(type="yarn", factor=2))),
    ((64, 0.5), dict(scaling=dict(type="yarn", factor=2, original_max_position=4096))),
    ((64, 1e4), dict(scaling=dict(type="yarn", factor=2, original_max_position=4096, beta_fast=0)))])
def test_frequencies_refused(args, kw):
    if kw.get("scaling", {"type": 0}).get("type", None) is None:
        # a scaling without a type scales nothing
        assert torch.equal(PKG.rotary_frequencies(*args, device="cpu", **kw).inv_freq,
                           PKG.rotary_frequencies(*args, device="cpu").inv_freq)
        return
    with pytest.raises(ValueError):
        PKG.rotary_frequencies(*args, device="cpu", **kw)


def test_frequencies_from_the_caller():
    for bad in (torch.ones(4), torch.ones((2, 2), dtype=torch.float64), torch.ones(0, dtype=torch.float64),
                torch.ones(257, dtype=torch.float64), torch.ones(8, dtype=torch.float64)[::2], [1.0]):
        with pytest.raises(ValueError):
            PKG.RotaryFrequencies(bad)
    assert PKG.RotaryFrequencies(torch.ones(3, dtype=torch.float64), 2.0).rotary_dim == 6


# ---------------------------------------------------------------------------
# there is no CPU implementation
# ---------------------------------------------------------------------------
def test_host_tensors_are_refused():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    freqs = PKG.rotary_frequencies(64, 1e4, device="cpu")
    with pytest.raises(ValueError, match="HIP device"):
        PKG.rotary_embedding(bf(2, 1, 64), i32(2), freqs)
    with pytest.raises(TypeError):
        PKG.rotary_embedding([1.0], i32(2), freqs)
    with pytest.raises(ValueError, match="HIP device"):
        PKG.latent_store(bf(2, 512), bf(2, 64), None, i32(2), i32(2), bf(1, 16, 576), freqs)
    with pytest.raises(ValueError, match="HIP device"):
        PKG.LatentWeights(bf(256, 512), num_heads=1, nope_dim=128, v_dim=128)
    with pytest.raises(TypeError, match="LatentWeights"):
        PKG.latent_decode_attention(bf(1, 1, 128), bf(1, 1, 64), bf(1, 16, 576), None, i32(1, 1), i32(1), scale=1.0)
    with pytest.raises(TypeError, match="LatentWeights"):
        PKG.latent_attention(bf(1, 16, 576), bf(1, 1, 192), bf(1, 512), bf(1, 64), None, None, freqs, None, scale=1.0)
