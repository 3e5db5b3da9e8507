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


@pytest.mark.parametrize("dim,hq,hkv,T,S,window_,sinks,batch", [
    (128, 2, 2, 700, 700, 200, 3, 5), (64, 4, 1, 333, 900, 256, 0, 4), (32, 2, 1, 130, 130, 40, 7, 200), (128, 4, 2, 40, 40, 40, 0, 9)])
def test_prompt_padding_is_never_looked_at(dim, hq, hkv, T, S, window_, sinks, batch):
    """Unequal lengths, none and all; what lies behind them is NaN and infinity, its output rows come back as zeros."""
    from kvm_paper_b200 import window
    g = _gen(dim + T)
    lens = [0, S, S - T, S - T + 1, S - 1] + [1 + (37 * i) % S for i in range(batch)]
    lens = lens[:batch]
    q, k, v = wh.heads_data(g, batch, hq, T, dim), wh.heads_data(g, batch, hkv, S, dim), wh.heads_data(g, batch, hkv, S, dim)
    want, mag = wh.prompt(q, k, v, window_, sinks, lengths=lens)
    for b, n in enumerate(lens):
        k[b, :, n:], v[b, :, n:] = math.nan, math.inf
        q[b, :, max(n - (S - T), 0):] = math.nan
    out = torch.full((batch, T, hq * dim), 7.0, device="cuda", dtype=torch.bfloat16)
    got = window.window_attention(q, k, v, window=window_, sinks=sinks, lengths=_ints(lens), out=out)
    assert got is out
    wh.assert_near(got.view(batch, T, hq, dim), want, mag)
    for b, n in enumerate(lens):
        assert not got[b, max(n - (S - T), 0):].any()


@pytest.mark.parametrize("dim,hq,hkv", [(128, 2, 2), (64, 2, 1), (32, 1, 1)])
def test_prompt_infinities_and_nan_stay_with_the_rows_that_see_them(dim, hq, hkv):
    from kvm_paper_b200 import window
    g = _gen(dim)
    T, w, s = 500, 130, 2
    q, k, v = wh.heads_data(g, 1, hq, T, dim), wh.heads_data(g, 1, hkv, T, dim), wh.heads_data(g, 1, hkv, T, dim)
    v[0, 0, 200, 3] = math.nan     # seen by queries 200 .. 329 in one channel
    v[0, hkv - 1, 301, 5] = math.inf
    v[0, 0, 301, 6] = -math.inf
    v[0, 0, 1, 7] = math.nan       # a sink: by all from 1 on
    k[0, 0, 420, 0] = math.nan     # whole rows from 420 on
    q[0, 0, 77, 0] = math.nan
    got = window.window_attention(q, k, v, window=w, sinks=s).view(1, T, hq, dim)
    want, mag = wh.prompt(q, k, v, w, s)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    wh.assert_near(torch.where(finite, got.double(), 0.0), torch.where(finite, want, 0.0), torch.where(finite, mag, 0.0))
    assert int(torch.isnan(got).sum()) > 130 and not torch.isnan(got[0, 330:420, 0, 3]).any()
    window.check_status()


def test_prompt_scores_far_apart():
    """Weights over the whole range of the exponential: very peaked rows, rows whose later keys raise the maximum again and
    again, equal scores, very negative ones."""
    from kvm_paper_b200 import window
    g = _gen(3)
    T, D = 600, 64
    q = wh.heads_data(g, 1, 2, T, D, scale=4.0)
    k = wh.heads_data(g, 1, 2, T, D)
    k[:, 0] *= torch.linspace(0.01, 8, T, device="cuda").view(1, T, 1).bfloat16()
    q[:, 1, 100:200] = 0
    v = wh.heads_data(g, 1, 2, T, D)
    got = window.window_attention(q, k, v, window=None).view(1, T, 2, D).double()
    want, mag = wh.prompt(q, k, v, None, 0)
    # scores up to 4 * 8 * 64^.5 * 6 / 8 < 2^8 in magnitude: 128 * 2^-24 * 2^8 = 2^-9 for a weight, twice for the quotient
    tol = (2 * wh.U_BF16 + 2.0 ** -8) * mag + wh.U_BF16 * want.abs()
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dim,group", [(128, 2), (64, 16), (32, 1)])
def test_token_special_values(bits, dim, group):
    """NaN and infinities in rows that are not seen (not yet overwritten, behind the window's end, stale rows of a cache in
    use), seen NaN, values of very unequal size, zeros."""
    from kvm_paper_b200 import window
    g = _gen(dim)
    w, s, B = 100, 3, 6
    c = window.WindowCache(B, 1, dim, window=w, sinks=s, bits=bits)
    if bits == 16:
        c.k.fill_(math.nan), c.v.fill_(math.inf)  # (memory that was never written)
    bad = torch.full((B, 1, 300, dim), math.nan, device="cuda", dtype=torch.bfloat16)
    c.write(bad, bad, 0, lengths=_ints([300, 0, 300, 0, 0, 0]))  # an earlier user of two of the places
    ref = wh.Cache(B, 1, dim, w, s, bits)
    T = 231
    k, v = wh.heads_data(g, B, 1, T, dim), wh.heads_data(g, B, 1, T, dim)
    v[:, :, ::7] *= 1e-6
    v[:, :, 5::50] *= 1e4
    k[:, :, 9::13] = 0
    v[4] = 0
    v[5, 0, 220, 1] = math.nan
    lens = [231, 40, 2, 104, 150, 231]
    c.write(k, v, 0, lengths=_ints(lens))
    for b, n in enumerate(lens):
        ref.write(b, k[b, :, :n], v[b, :, :n], 0)
    q = wh.heads_data(g, B, group, 1, dim)
    got = c.attend(q, _ints(lens)).view(B, group, dim)
    for b, n in enumerate(lens):
        want, mag = ref.attend(b, q[b], n)
        wh.assert_near(got[b], want, mag, bits, f"{b}")
    k2, v2 = c.read(_ints(lens))
    for b, n in enumerate(lens):
        for y, x in zip((k2, v2), ref.held(b, n)):
            assert torch.equal(y[b, :, :x.size(1)].double().nan_to_num(9e9), x.nan_to_num(9e9)) and not y[b, :, x.size(1):].any()


def test_token_value_scales_rise_late():
    """4 bits: each group of rows far larger than those before it, so that the reference scale rises with every one, and falls
    off again; rows 2^-20 smaller than the largest still count as far as their size matters."""
    from kvm_paper_b200 import window
    g = _gen(11)
    for dim in (128, 64):
        n = 2000
        k, v = wh.heads_data(g, 1, 1, n, dim, scale=0.3), wh.heads_data(g, 1, 1, n, dim)
        size = torch.exp2((torch.arange(n, device="cuda") // 16 * 5) % 41 - 20.0)
        v = (v.float() * size.view(1, 1, n, 1)).bfloat16()
        c = window.WindowCache(1, 1, dim, window=n, bits=4)
        c.write(k, v, 0)
        q = wh.heads_data(g, 1, 4, 1, dim)
        got = c.attend(q, n).view(4, dim)
        hk, hv = wh.quantised(k)[0], wh.quantised(v)[0]
        want, mag = wh.attend(q[0], hk, hv, torch.ones(1, n, device="cuda", dtype=torch.bool), dim ** -0.5)
        wh.assert_near(got, want[:, 0], mag[:, 0], 4)


def test_strides_and_alignment_of_inputs():
    """Views of other orders, expanded heads, odd offsets and single entries give what contiguous copies give."""
    from kvm_paper_b200 import window
    g = _gen(5)
    B, H, T, D = 2, 4, 70, 64
    big = torch.randn(B, T, 3 * H * D + 8, device="cuda", generator=g).bfloat16()
    wide = [big[..., i * H * D:(i + 1) * H * D].view(B, T, H, D).transpose(1, 2) for i in range(3)]           # columns of wider rows
    odd = [big[..., i * H * D + 1:(i + 1) * H * D + 1].unflatten(-1, (H, D)).transpose(1, 2) for i in range(3)]  # 2-byte aligned
    swapped = [torch.randn(D, T, H, B, device="cuda", generator=g).bfloat16().permute(3, 2, 1, 0) for _ in range(3)]
    one = [torch.randn(1, 1, T, D, device="cuda", generator=g).bfloat16().expand(B, H, T, D) for _ in range(3)]
    for q, k, v in (wide, odd, swapped, one):
        plain = [t.contiguous() for t in (q, k, v)]
        assert torch.equal(window.window_attention(q, k, v, window=20, sinks=2), window.window_attention(*plain, window=20, sinks=2))
        for bits in (4, 16):
            c, c2 = (window.WindowCache(B, H, D, window=50, sinks=2, bits=bits) for _ in range(2))
            c.write(k, v, 0), c2.write(*plain[1:], 0)
            a = c.step(q[:, :, :1], k[:, :, :1], v[:, :, :1], T)
            b = c2.step(plain[0][:, :, :1].contiguous(), plain[1][:, :, :1].contiguous(), plain[2][:, :, :1].contiguous(), T)
            assert torch.equal(a, b)
            assert all(torch.equal(x, y) for x, y in zip(c.read(T + 1), c2.read(T + 1)))


def test_refusals():
    from kvm_paper_b200 import window
    z = lambda *s, **kw: torch.zeros(*s, device="cuda", dtype=kw.get("dtype", torch.bfloat16))  # noqa: E731
    q, k = z(2, 4, 8, 64), z(2, 2, 8, 64)
    ok = dict(window=4, sinks=1)
    for args, kw in [((q, k, z(2, 2, 9, 64)), {}), ((q, k, z(2, 2, 8, 32)), {}), ((q, z(2, 3, 8, 64), z(2, 3, 8, 64)), {}),
                     ((q.half(), k, k), {}), ((q, k.float(), k), {}), ((z(2, 4, 9, 64), k, k), {}), ((z(2, 4, 8, 48), z(2, 2, 8, 48), z(2, 2, 8, 48)), {}),
                     ((q, k, k), dict(window=0)), ((q, k, k), dict(sinks=-1)), ((q, k, k), dict(scale=0.0)), ((q, k, k), dict(scale=math.nan)),
                     ((q, k, k), dict(lengths=3)), ((q, k, k), dict(lengths=_ints([1, 2, 3]))), ((q, k, k), dict(lengths=_ints([1, 2]).long())),
                     ((q, k, k), dict(out=z(2, 8, 255))), ((q, k, k), dict(out=z(2, 8, 256, dtype=torch.float32))), ((q, k, k), dict(out=z(2, 8, 512)[..., ::2])),
                     ((q.clone().requires_grad_(), k, k), {})]:
        with pytest.raises(ValueError):
            window.window_attention(*args, **{**ok, **kw})
    with pytest.raises(RuntimeError):
        window.window_attention(q, k.cpu(), k, **ok)
    with pytest.raises(RuntimeError):
        window.window_attention(q, k, k, **ok, lengths=torch.zeros(2, dtype=torch.int32))
    for kw in (dict(window=0), dict(window=8, sinks=-1), dict(window=8, bits=8)):
        with pytest.raises(ValueError):
            window.WindowCache(2, 2, 64, **kw)
    with pytest.raises(ValueError):
        window.WindowCache(2, 2, 80, window=8)
    c = window.WindowCache(2, 2, 64, window=8, bits=4)
    assert c.k is None and c.v is None and c.nbytes() == 4 * 18 * 64
    q1, k1 = z(2, 4, 1, 64), z(2, 2, 1, 64)
    for call in (lambda: c.attend(q, 1), lambda: c.attend(z(2, 3, 1, 64), 1), lambda: c.attend(z(2, 34, 1, 64), 1), lambda: c.attend(q1, -1),
                 lambda: c.attend(q1, _ints([1])), lambda: c.attend(q1, 1, scale=-1), lambda: c.step(q1, k1, k, 0), lambda: c.step(q1, k1, k1, -2),
                 lambda: c.write(k, k1, 0), lambda: c.write(k, k, -2), lambda: c.write(k, k, 2**31 - 5), lambda: c.write(k, k, 0, lengths=9),
                 lambda: c.write(k, k, torch.zeros(2, device="cuda", dtype=torch.int64)), lambda: c.read(-1), lambda: c.write(k[0], k[0], 0)):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():  # (parameters of a module in inference)
        window.window_attention(q.clone().requires_grad_(), k, k, **ok)
    assert window.window_attention(z(2, 4, 0, 64), k, k, **ok).shape == (2, 0, 256)
    assert window.window_attention(z(0, 4, 8, 64), z(0, 2, 8, 64), z(0, 2, 8, 64), **ok).shape == (0, 8, 256)
    c.write(z(2, 2, 0, 64), z(2, 2, 0, 64), 3)


@pytest.mark.parametrize("bits", [4, 16])
def test_prompt_then_tokens_then_the_next_prompt(bits):
    """As a serving loop uses them: a padded batch of prompts, its cache, tokens through a captured graph whose positions move on the
    device, the cache read back in front of the next chunk of one of the sequences."""
    from kvm_paper_b200 import window
    g = _gen(bits)
    B, Hq, Hkv, D, w, s, T, N = 3, 8, 2, 128, 150, 4, 400, 40
    lens = [400, 90, 213]
    q, k, v = wh.heads_data(g, B, Hq, T + N, D), wh.heads_data(g, B, Hkv, T + N, D), wh.heads_data(g, B, Hkv, T + N, D)
    scale = D ** -0.5
    n_dev = _ints(lens)
    y = window.window_attention(q[:, :, :T], k[:, :, :T], v[:, :, :T], window=w, sinks=s, lengths=n_dev)
    want, mag = wh.prompt(q[:, :, :T], k[:, :, :T], v[:, :, :T], w, s, lengths=lens)
    wh.assert_near(y.view(B, T, Hq, D), want, mag)
    c = window.WindowCache(B, Hkv, D, window=w, sinks=s, bits=bits)
    c.write(k[:, :, :T], v[:, :, :T], 0, lengths=n_dev)
    ref = wh.Cache(B, Hkv, D, w, s, bits)
    for b, n in enumerate(lens):
        ref.write(b, k[b, :, :n], v[b, :, :n], 0)
    # tokens: one graph, positions advanced inside it
    pos = _ints(lens)
    qt, kt, vt = (torch.empty(B, h, 1, D, device="cuda", dtype=torch.bfloat16) for h in (Hq, Hkv, Hkv))
    out = torch.empty(B, 1, Hq * D, device="cuda", dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step(qt, kt, vt, pos, out=out)
        pos += 1
    for i in range(N):
        qt.copy_(q[:, :, T + i:T + i + 1]), kt.copy_(k[:, :, T + i:T + i + 1]), vt.copy_(v[:, :, T + i:T + i + 1])
        graph.replay()
        for b in range(B):
            p = lens[b] + i
            ref.write(b, kt[b], vt[b], p)
            if i % 13 == 0 or i == N - 1:
                o, m = ref.attend(b, qt[b], p + 1, scale)
                wh.assert_near(out[b, 0], o.flatten(), m.flatten(), bits, f"token {i} of {b}")
    assert pos.tolist() == [n + N for n in lens]
    # the next chunk of sequence 0 behind what its cache holds
    end = lens[0] + N
    back = [t[:1, :, :min(end, s + w)] for t in c.read(pos)]
    more = [wh.heads_data(g, 1, h, 77, D) for h in (Hq, Hkv, Hkv)]
    ck, cv = (torch.cat([t, x], 2) for t, x in zip(back, more[1:]))
    y = window.window_attention(more[0], ck, cv, window=w, sinks=s).view(77, Hq, D)
    hk, hv = ([ref.k, ref.v][i][0] for i in range(2))
    full_k, full_v = torch.cat([hk, more[1][0].double()], 1), torch.cat([hv, more[2][0].double()], 1)
    o, m = wh.attend(more[0][0], full_k, full_v, wh.visible(77, end + 77, w, s, "cuda"), scale)
    wh.assert_near(y.transpose(0, 1), o, m)
    window.check_status()


def test_streams_and_graphs_do_not_share_scratch():
    """Two long attends of one cache at the same time, on two streams and in two graphs, give what they give alone."""
    from kvm_paper_b200 import window
    g = _gen(8)
    n = 60000
    c = window.WindowCache(1, 2, 64, window=n, bits=4)
    k, v = wh.heads_data(g, 1, 2, n, 64), wh.heads_data(g, 1, 2, n, 64)
    c.write(k, v, 0)
    qs = [wh.heads_data(g, 1, 8, 1, 64) for _ in range(2)]
    alone = [c.attend(q, n) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(c.attend(qs[i], n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for os, a in zip(outs, alone) for o in os)
    graphs, res = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append(c.attend(qs[i], n))
        graphs.append(gr)
    for _ in range(10):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(r, a) for r, a in zip(res, alone))


@pytest.mark.parametrize("bits,kvrows,rows", [(16, 300, 65536), (4, 1000, 65536)])
def test_offsets_beyond_32_bits(bits, kvrows, rows):
    """The last sequence of a cache of more than 4 GB per array."""
    from kvm_paper_b200 import window
    g = _gen(rows)
    c = window.WindowCache(kvrows, 1, 128, window=rows, bits=bits)
    assert c.nbytes() > (2 if bits == 16 else 1) << 32
    T = 700
    k, v = wh.heads_data(g, 1, 1, T, 128).expand(kvrows, 1, T, 128), wh.heads_data(g, 1, 1, T, 128).expand(kvrows, 1, T, 128)
    pos = torch.full((kvrows,), -1, device="cuda", dtype=torch.int32)
    pos[-1] = rows - 300                                     # over the ring's end
    c.write(k, v, pos)
    n = torch.zeros(kvrows, device="cuda", dtype=torch.int32)
    n[-1] = rows + 400
    small = window.WindowCache(1, 1, 128, window=rows, bits=bits)
    small.write(k[-1:], v[-1:], rows - 300)
    q = wh.heads_data(g, kvrows, 2, 1, 128)
    got, want = c.attend(q, n), small.attend(q[-1:].contiguous(), rows + 400)
    # (the same rows in other shares of the list: fp32 sums in another order)
    assert torch.allclose(got[-1:].float(), want.float(), rtol=2.0 ** -7, atol=1e-6)
    assert not got[:-1].any()
    step = c.step(q, k[:, :, :1], v[:, :, :1], torch.where(n > 0, n, -1))
    want = small.step(q[-1:].contiguous(), k[-1:, :, :1], v[-1:, :, :1], rows + 400)
    assert torch.allclose(step[-1:].float(), want.float(), rtol=2.0 ** -7, atol=1e-6)
    if bits == 16:
        assert torch.equal(c.k[-1], small.k[0]) and torch.equal(c.v[-1], small.v[0])


def test_many_sequences_and_repeated_calls():
    """More sequences than a launch takes, in both orders of the list, and the same bits every time."""
    from kvm_paper_b200 import window
    g = _gen(21)
    B = 1500
    lens = [(17 * i) % 90 for i in range(B)]
    for bits, dim, group in ((4, 128, 8), (16, 32, 1)):
        c = window.WindowCache(B, 1, dim, window=64, sinks=1, bits=bits)
        k, v = wh.heads_data(g, B, 1, 90, dim), wh.heads_data(g, B, 1, 90, dim)
        c.write(k, v, 0, lengths=_ints(lens))
        q = wh.heads_data(g, B, group, 1, dim)
        got = c.attend(q, _ints(lens))
        assert torch.equal(got, c.attend(q, _ints(lens)))
        ref = wh.Cache(B, 1, dim, 64, 1, bits)
        for b in list(range(0, B, 97)) + [B - 1]:
            ref.write(b, k[b, :, :lens[b]], v[b, :, :lens[b]], 0)
            want, mag = ref.attend(b, q[b], lens[b])
            wh.assert_near(got[b, 0], want.flatten(), mag.flatten(), bits, f"{b}")


def test_prompt_values_near_the_largest_number():
    """Sums of weights that are not normalised yet would pass the range of fp32; the output does not."""
    from kvm_paper_b200 import window
    g = _gen(31)
    T = 300
    q, k = wh.heads_data(g, 1, 2, T, 64), wh.heads_data(g, 1, 1, T, 64)
    v = wh.heads_data(g, 1, 1, T, 64)
    v[..., :40] = 3e38
    v[..., 40:44] *= 1e37
    got = window.window_attention(q, k, v, window=100, sinks=1).view(1, T, 2, 64)
    want, mag = wh.prompt(q, k, v, 100, 1)
    assert bool(torch.isfinite(got).all())
    wh.assert_near(got, want, mag)


def test_prompt_of_nothing_but_nan_ends_soon():
    """Every value NaN: every row is looked at again, and settled by the first key that it sees."""
    from kvm_paper_b200 import window
    g = _gen(32)
    T = 8192
    q, k = wh.heads_data(g, 1, 4, T, 128), wh.heads_data(g, 1, 2, T, 128)
    v = torch.full((1, 2, T, 128), math.nan, device="cuda", dtype=torch.bfloat16)
    window.window_attention(q, k, v, window=None)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = window.window_attention(q, k, v, window=None)
    end.record()
    torch.cuda.synchronize()
    assert bool(torch.isnan(got).all()) and start.elapsed_time(end) < 50.0


def test_lengths_and_positions_outside_their_range_touch_nothing():
    """Device numbers that no call may bring: negative lengths count as 0, positions that cannot be held leave their sequence alone."""
    from kvm_paper_b200 import window
    g = _gen(33)
    lowest, highest = -2**31, 2**31 - 1
    q, k, v = wh.heads_data(g, 4, 2, 40, 64), wh.heads_data(g, 4, 1, 300, 64), wh.heads_data(g, 4, 1, 300, 64)
    got = window.window_attention(q, k, v, window=50, lengths=_ints([lowest, -1, 300, highest]))
    want, mag = wh.prompt(q, k, v, 50, 0, lengths=[0, 0, 300, 300])
    wh.assert_near(got.view(4, 40, 2, 64), want, mag)
    for bits in (4, 16):
        c = window.WindowCache(4, 1, 64, window=32, sinks=3, bits=bits)
        c.write(k[:, :, :5], v[:, :, :5], 0)
        before = c.read(5)
        c.write(k[:, :, 5:9], v[:, :, 5:9], _ints([lowest, -1, highest, highest - 3]))
        c.write(k[:, :, 5:9], v[:, :, 5:9], 5, lengths=_ints([lowest, -1, 0, -5]))
        y = c.step(q[:, :, :1], k[:, :, 9:10], v[:, :, 9:10], _ints([lowest, -1, -2, highest]))
        assert not y.any()
        assert all(torch.equal(a, b) for a, b in zip(c.read(5), before))
        assert not any(t.any() for t in c.read(_ints([lowest, -1, 0, -7])))
        assert not c.attend(q[:, :, :1], _ints([lowest, -1, 0, -7])).any()
    window.check_status()


def test_prompts_of_more_sequences_than_are_listed():
    from kvm_paper_b200 import window
    g = _gen(34)
    B, T = 601, 150
    lens = [(61 * i) % (T + 1) for i in range(B)]
    q, k, v = wh.heads_data(g, B, 2, T, 32), wh.heads_data(g, B, 1, T, 32), wh.heads_data(g, B, 1, T, 32)
    want, mag = wh.prompt(q, k, v, 40, 2, lengths=lens)
    for b, n in enumerate(lens):
        k[b, :, n:], v[b, :, n:] = math.nan, math.inf
    got = window.window_attention(q, k, v, window=40, sinks=2, lengths=_ints(lens))
    wh.assert_near(got.view(B, T, 2, 32), want, mag)


def test_short_rows_of_a_long_cache_are_complete_for_what_follows():
    """No row is cut although the cache's length asks for the joining launch: what follows in the stream sees the output."""
    from kvm_paper_b200 import window
    g = _gen(35)
    c = window.WindowCache(1, 4, 128, window=200000, bits=4)
    k, v = wh.heads_data(g, 1, 4, 300, 128), wh.heads_data(g, 1, 4, 300, 128)
    c.write(k, v, 0)
    q = wh.heads_data(g, 1, 16, 1, 128)
    want = c.attend(q, 300).clone()
    out = torch.empty_like(want)
    for _ in range(200):
        out.fill_(math.nan)
        c.attend(q, 300, out=out)
        assert torch.equal(out.clone(), want)


@pytest.mark.parametrize("bits", [4, 16])
def test_first_calls_of_a_process_may_be_captured(bits):
    import subprocess
    import sys
    code = f"""
import torch
from kvm_paper_b200 import window
q = torch.randn(2, 4, 20, 64, device="cuda").bfloat16()
k = torch.randn(2, 2, 20, 64, device="cuda").bfloat16()
c = window.WindowCache(2, 2, 64, window=100000, sinks=4, bits={bits})
pos = torch.full((2,), 20, device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = window.window_attention(q, k, k, window=8, sinks=1)
    c.write(k, k, 0)
    z = c.step(q[:, :, :1], k[:, :, :1], k[:, :, :1], pos)
    a, b = c.read(21)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, window.window_attention(q, k, k, window=8, sinks=1))
assert torch.equal(z, c.step(q[:, :, :1], k[:, :, :1], k[:, :, :1], pos))
assert all(torch.equal(s, t) for s, t in zip((a, b), c.read(21)))
window.check_status()
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_outputs_that_cannot_be_written_are_refused():
    from kvm_paper_b200 import window
    q, k = (torch.zeros(2, h, 8, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    for out in (torch.zeros(2, 8, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True), [0], torch.zeros(2, 8, 256, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            window.window_attention(q, k, k, window=4, out=out)
    c = window.WindowCache(2, 2, 64, window=8)
    with pytest.raises(ValueError):
        c.attend(q[:, :, :1], 3, out=torch.zeros(2, 1, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True))


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("n", [40, 1500, 30000])
def test_token_values_near_the_largest_number(bits, n):
    """Sums of weights that are not normalised yet would pass the range of fp32; the output does not."""
    from kvm_paper_b200 import window
    g = _gen(41 + n)
    k, v = wh.heads_data(g, 2, 1, n, 64), wh.heads_data(g, 2, 1, n, 64)
    v[0] = 3e38
    v[0, :, :, 32:40] = -3e38
    v[1, :, :, :32] *= 5e37
    q = wh.heads_data(g, 2, 3, 1, 64)
    c = window.WindowCache(2, 1, 64, window=n, bits=bits)
    c.write(k, v, 0)
    got = c.attend(q, n).view(2, 3, 64)
    assert bool(torch.isfinite(got).all())
    hk, hv = (wh.quantised(k), wh.quantised(v)) if bits == 4 else (k.double(), v.double())
    for b in range(2):
        want, mag = wh.attend(q[b], hk[b], hv[b], torch.ones(1, n, device="cuda", dtype=torch.bool), 64 ** -0.5)
        wh.assert_near(got[b], want[:, 0], mag[:, 0], bits)
