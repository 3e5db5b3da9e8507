"""The sliding-window operators on the GPU against their definition in 64 bits."""

import math

import pytest
import torch

from tests import window_helpers as wh

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


# ---------------------------------------------------------------------------------------------- cache

@pytest.mark.parametrize("dim", [32, 64, 128])
def test_quantised_rows_come_back_as_defined(dim):
    """Every level, border and special value of the 4-bit form; writing back what was read changes nothing."""
    from kvm_paper_b200 import window
    g = _gen(dim)
    x = torch.randn(2, 3, 200, dim, device="cuda", generator=g) * torch.exp(2 * torch.randn(2, 3, 200, 1, device="cuda", generator=g))
    x[0, 0, :40] = (torch.arange(40 * dim, device="cuda").reshape(40, dim) % 97 - 48) / 4  # levels and borders
    x[0, 1, 0] = 0.0
    x[0, 1, 1, :32] = 1e-38        # below the smallest scale
    x[0, 1, 2] = 3e38
    x[0, 1, 3, 5] = math.inf
    x[0, 1, 4, 31] = math.nan
    x[0, 1, 5, :] = -0.0
    x[0, 1, 6, :32] = 7.1e-38
    x = x.bfloat16()
    v = x.flip(2).contiguous()
    c = window.WindowCache(2, 3, dim, window=200, sinks=0, bits=4)
    c.write(x, v, 0)
    k2, v2 = c.read(200)
    for got, src in ((k2, x), (v2, v)):
        want = wh.quantised(src)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.double().nan_to_num(0), want.nan_to_num(0))
    c2 = window.WindowCache(2, 3, dim, window=200, sinks=0, bits=4)
    c2.write(k2.nan_to_num(0), v2.nan_to_num(0), 0)
    k3, v3 = c2.read(200)
    assert torch.equal(k3, k2.nan_to_num(0)) and torch.equal(v3, v2.nan_to_num(0))


@pytest.mark.parametrize("bits,dim,heads,window_,sinks", [
    (4, 128, 2, 33, 5), (4, 64, 3, 16, 0), (4, 32, 1, 100, 17), (16, 128, 1, 50, 4), (16, 64, 2, 1, 0), (16, 32, 2, 31, 16), (4, 128, 1, 1, 1)])
def test_writes_of_all_lengths_and_what_is_read(bits, dim, heads, window_, sinks):
    """Ragged writes one behind the other, shorter and longer than the ring, over its end, with sequences left out."""
    from kvm_paper_b200 import window
    g = _gen(bits + dim + window_)
    B = 4
    c = window.WindowCache(B, heads, dim, window=window_, sinks=sinks, bits=bits)
    ref = wh.Cache(B, heads, dim, window_, sinks, bits)
    have = [0] * B
    for T in (1, 3, window_ // 2 + 1, 2 * window_ + 20, 7, 16, window_ + 1):
        k, v = wh.heads_data(g, B, heads, T, dim), wh.heads_data(g, B, heads, T, dim)
        n = [T, max(T - 1, 0), (T + 1) // 2, T]
        pos = [have[0], have[1], have[2], -1]
        c.write(k, v, _ints(pos), lengths=_ints(n))
        for b in range(3):
            ref.write(b, k[b, :, :n[b]], v[b, :, :n[b]], have[b])
            have[b] += n[b]
        got = c.read(_ints(have))
        for name, y, store in (("k", got[0], 0), ("v", got[1], 1)):
            for b in range(B):
                want = ref.held(b, have[b])[store]
                assert torch.equal(y[b, :, :want.size(1)].double(), want), (name, T, b)
                assert not y[b, :, want.size(1):].any(), (name, T, b)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dim,hkv,group", [(128, 2, 1), (128, 1, 8), (128, 1, 16), (128, 2, 5), (64, 3, 2), (64, 1, 12), (32, 2, 4), (32, 1, 9)])
def test_token_attention_ragged(bits, dim, hkv, group):
    """Contexts of no, one and many tokens, windows that have wrapped or not, several chunks; both forms of the call."""
    from kvm_paper_b200 import window
    g = _gen(dim * group + hkv)
    w, s = 300, 5
    lens = [0, 1, 4, 5, 6, 16, 17, 133, 299, 305, 306, 450, 1000, 2, 607]
    B = len(lens)
    c = window.WindowCache(B, hkv, dim, window=w, sinks=s, bits=bits)
    ref = wh.Cache(B, hkv, dim, w, s, bits)
    T = max(lens)
    k, v = wh.heads_data(g, B, hkv, T, dim), wh.heads_data(g, B, hkv, T, dim)
    c.write(k, v, 0, lengths=_ints(lens))
    for b, n in enumerate(lens):
        ref.write(b, k[b, :, :n], v[b, :, :n], 0)
    q = wh.heads_data(g, B, hkv * group, 1, dim)
    got = c.attend(q, _ints(lens))
    for b, n in enumerate(lens):
        want, mag = ref.attend(b, q[b], n)
        wh.assert_near(got[b, 0], want.flatten(), mag.flatten(), bits, f"attend {n}")
    # the next token of every other sequence
    k1, v1 = wh.heads_data(g, B, hkv, 1, dim), wh.heads_data(g, B, hkv, 1, dim)
    pos = [n if i % 2 == 0 else -1 for i, n in enumerate(lens)]
    got = c.step(q, k1, v1, _ints(pos), scale=0.2)
    back = c.read(_ints([p + 1 if p >= 0 else n for p, n in zip(pos, lens)]))
    for b, p in enumerate(pos):
        if p >= 0:
            ref.write(b, k1[b], v1[b], p)
        want, mag = ref.attend(b, q[b], p + 1, 0.2)
        wh.assert_near(got[b, 0], want.flatten(), mag.flatten(), bits, f"step {p}")
        n = p + 1 if p >= 0 else lens[b]
        for y, x in zip(back, ref.held(b, n)):
            assert torch.equal(y[b, :, :x.size(1)].double(), x)
    window.check_status()


@pytest.mark.parametrize("bits,batch,hkv,group,dim,n", [
    (4, 1, 1, 4, 128, 40000), (16, 1, 2, 2, 128, 20001), (4, 3, 5, 1, 64, 9000), (16, 2, 1, 16, 64, 5000), (4, 40, 8, 2, 32, 700), (4, 200, 2, 1, 64, 130)])
def test_token_attention_long_and_many(bits, batch, hkv, group, dim, n):
    """Rows that many CTAs share, and many rows in a CTA; one length for all, given as a number."""
    from kvm_paper_b200 import window
    g = _gen(n)
    c = window.WindowCache(batch, hkv, dim, window=n, sinks=3, bits=bits)
    k, v = wh.heads_data(g, batch, hkv, n, dim), wh.heads_data(g, batch, hkv, n, dim)
    c.write(k, v, 0)
    q = wh.heads_data(g, batch, hkv * group, 1, dim)
    got = c.attend(q, n)
    hk, hv = (wh.quantised(t) if bits == 4 else t.double() for t in (k, v))
    see = torch.ones(1, n, device="cuda", dtype=torch.bool)
    for b in range(0, batch, max(batch // 7, 1)):
        want, mag = wh.attend(q[b], hk[b], hv[b], see, dim ** -0.5)
        wh.assert_near(got[b, 0], want.flatten(), mag.flatten(), bits)
    assert torch.equal(got, c.attend(q, _ints([n] * batch)))


# --------------------------------------------------------------------------------------------- prompts

@pytest.mark.parametrize("dim,hq,hkv", [(128, 2, 2), (128, 4, 2), (64, 3, 1), (64, 4, 4), (32, 8, 2), (128, 5, 1)])
@pytest.mark.parametrize("T,S,window_,sinks", [
    (1, 1, 1, 0), (1, 700, 300, 4), (17, 17, 5, 2), (128, 128, 128, 0), (129, 129, 64, 1), (255, 511, 100, 130), (300, 300, None, 0),
    (513, 700, 256, 16), (640, 640, 1, 0), (1025, 1025, 333, 3)])
def test_prompt(dim, hq, hkv, T, S, window_, sinks):
    from kvm_paper_b200 import window
    g = _gen(T + dim)
    q, k, v = wh.heads_data(g, 2, hq, T, dim), wh.heads_data(g, 2, hkv, S, dim), wh.heads_data(g, 2, hkv, S, dim)
    got = window.window_attention(q, k, v, window=window_, sinks=sinks)
    want, mag = wh.prompt(q, k, v, window_, sinks)
    wh.assert_near(got.view(2, T, hq, dim), want, mag)
    window.check_status()
