"""The window operators at the ends of their range: numbers that are none, scores and values of any size, masks that leave a
share of the work without a score, calls that lay their tensors out in unusual ways."""

import math

import pytest
import torch

from tests import window_helpers as wh

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dim", [128, 64, 32])
@pytest.mark.parametrize("window_,sinks", [(None, 0), (300, 128)])
def test_prompt_a_key_that_is_nan_reaches_every_row_that_sees_it(dim, window_, sinks):
    """Head h has the NaN in its key h, so that every place of a tile of keys is met, in tiles that are seen whole too."""
    from kvm_paper_b200 import window
    g = _gen(dim)
    H, T = 128, 520
    q, k, v = (wh.heads_data(g, 1, H, T, dim) for _ in range(3))
    at = torch.arange(H, device="cuda")
    k[0, at, at, at % dim] = math.nan
    got = window.window_attention(q, k, v, window=window_, sinks=sinks).view(1, T, H, dim)
    want, mag = wh.prompt(q, k, v, window_, sinks)
    assert int(torch.isnan(want).sum()) > 300 * H * dim
    wh.assert_near(got, want, mag)


@pytest.mark.parametrize("bits", [16, 4])
def test_token_a_share_without_a_score_adds_nothing(bits):
    """Long rows are cut between CTAs: shares whose every score is -inf (16 bits: infinities among the keys; 4 bits: sums beyond
    fp32, of which the definition's weights are zero as well) beside shares with scores, and rows with none at all."""
    from kvm_paper_b200 import window
    g = _gen(51)
    n, dim = 40000, 64
    q = wh.heads_data(g, 1, 4, 1, dim).abs() + 0.25
    v = wh.heads_data(g, 1, 2, n, dim)
    k = wh.heads_data(g, 1, 2, n, dim)
    for head, rows in ((0, slice(0, 21000)), (1, slice(15000, n))):
        k[0, head, rows] = -3e38
        if bits == 16:
            k[0, head, rows, 7] = -math.inf
    c = window.WindowCache(1, 2, dim, window=n, bits=bits)
    c.write(k, v, 0)
    got = c.attend(q, n).view(4, dim)
    hk, hv = (wh.quantised(k), wh.quantised(v)) if bits == 4 else (k.double(), v.double())
    want, mag = wh.attend(q[0], hk[0], hv[0], torch.ones(1, n, device="cuda", dtype=torch.bool), dim ** -0.5)
    assert bool(torch.isfinite(want).all())
    wh.assert_near(got, want[:, 0], mag[:, 0], bits)
    if bits == 16:
        k[0, 0, :, 7] = -math.inf
        c.write(k, v, 0)
        got = c.attend(q, n).view(2, 2, dim)
        assert bool(torch.isnan(got[0]).all()) and torch.equal(got[1].double(), got[1].double().nan_to_num(nan=9.0))


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dim,group", [(128, 1), (64, 9), (32, 2)])
def test_token_queries_of_zeros_with_the_smallest_scales(bits, dim, group):
    """All scores 0: the mean of the values, whatever the scale, over rows that are seen in part, too."""
    from kvm_paper_b200 import window
    g = _gen(53)
    n = [1, 17, 100, 333]
    k, v = wh.heads_data(g, 4, 1, 333, dim), wh.heads_data(g, 4, 1, 333, dim)
    c = window.WindowCache(4, 1, dim, window=290, sinks=3, bits=bits)
    c.write(k, v, 0, lengths=_ints(n))
    ref = wh.Cache(4, 1, dim, 290, 3, bits)
    q = torch.zeros(4, group, 1, dim, device="cuda", dtype=torch.bfloat16)
    q[:, -1] = 1e-38
    for scale in (1e-37, 1e-20, 1e-6, 1.0):
        got = c.attend(q, _ints(n), scale=scale)
        for b in range(4):
            ref.write(b, k[b, :, :n[b]], v[b, :, :n[b]], 0)
            want, mag = ref.attend(b, q[b], n[b], scale)
            wh.assert_near(got[b, 0], want.flatten(), mag.flatten(), bits, f"scale {scale}, {n[b]} tokens")


def _one_hot(up, sign, heads, rows, dim):
    """Keys of one channel, 97 levels from 2^up on, the same again every 97 keys: scores of any size, far apart or alike."""
    k = torch.zeros(1, heads, rows, dim, device="cuda", dtype=torch.bfloat16)
    k[..., 5] = ((1 + torch.arange(rows, device="cuda") % 97 / 128) * 2.0 ** up * sign).bfloat16()
    return k


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("up", [4, 6, 8, 9, 10, 13, 14, 15, 16, 17, 18, 19, 20, 30, 50, 60])
def test_token_scores_of_any_size(bits, sign, up):
    """Scores of 2^9 to 2^121, all of them finite: the keys with the largest one share the weight."""
    from kvm_paper_b200 import window
    g = _gen(60 + up)
    for dim, group, n in ((64, 3, 500), (128, 9, 900), (32, 8, 9000)):
        k, v = _one_hot(up, sign, 1, n, dim), wh.heads_data(g, 1, 1, n, dim)
        q = torch.zeros(1, group, 1, dim, device="cuda", dtype=torch.bfloat16)
        q[..., 5] = (1.3 + torch.arange(group, device="cuda").view(1, -1, 1) / 16) * 2.0 ** up
        c = window.WindowCache(1, 1, dim, window=n, bits=bits)
        c.write(k, v, 0)
        for scale in (None, 1.0):
            got = c.attend(q, n, scale=scale).view(group, dim)
            hk, hv = (wh.quantised(k), wh.quantised(v)) if bits == 4 else (k.double(), v.double())
            want, mag = wh.attend(q[0], hk[0], hv[0], torch.ones(1, n, device="cuda", dtype=torch.bool), scale or dim ** -0.5)
            wh.assert_near(got, want[:, 0], mag[:, 0], bits)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("up", [-112, -60, 60, 112])
def test_token_queries_and_keys_of_opposite_size(bits, up):
    """Scores as in any other call, of queries near one end of the range and keys near the other."""
    from kvm_paper_b200 import window
    g = _gen(54)
    for dim, group, n in ((128, 4, 300), (64, 16, 3000), (32, 1, 70)):
        k, v, q = wh.heads_data(g, 2, 1, n, dim), wh.heads_data(g, 2, 1, n, dim), wh.heads_data(g, 2, group, 1, dim)
        k, q = (k.float() * 2.0 ** up).bfloat16(), (q.float() * 2.0 ** -up).bfloat16()
        c = window.WindowCache(2, 1, dim, window=n, bits=bits)
        c.write(k, v, 0)
        got = c.attend(q, n).view(2, group, dim)
        hk, hv = (wh.quantised(k), wh.quantised(v)) if bits == 4 else (k.double(), v.double())
        for b in range(2):
            want, mag = wh.attend(q[b], hk[b], hv[b], torch.ones(1, n, device="cuda", dtype=torch.bool), dim ** -0.5)
            wh.assert_near(got[b], want[:, 0], mag[:, 0], bits)


@pytest.mark.parametrize("bits", [4, 16])
def test_token_keys_near_the_largest_number(bits):
    """Scores of up to 2^125, all of them finite: the key with the largest one takes the whole weight."""
    from kvm_paper_b200 import window
    g = _gen(55)
    dim, n = 64, 500
    k, v = torch.zeros(1, 1, n, dim, device="cuda", dtype=torch.bfloat16), wh.heads_data(g, 1, 1, n, dim)
    best = [7, 213, 499, 64]
    for channel, i in enumerate(best):
        k[0, 0, :, 16 * channel] = (torch.arange(n, device="cuda") % 97 * 1e35).bfloat16()
        k[0, 0, i, 16 * channel] = 3.2e37  # (the largest of its row's group: held exactly or nearly)
    q = torch.zeros(1, 4, 1, dim, device="cuda", dtype=torch.bfloat16)
    for head in range(4):
        q[0, head, 0, 16 * head] = 1.0
    c = window.WindowCache(1, 1, dim, window=n, bits=bits)
    c.write(k, v, 0)
    got = c.attend(q, n).view(4, dim)
    held = c.read(n)[1][0, 0]
    assert torch.equal(got, held[best])


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("far", [-200.0, -1000.0, -math.inf])
def test_prompt_values_far_below_the_maximum_weigh_nothing(dim, far):
    """Keys whose weight is below the smallest number hold values near the largest one, in every place of a tile that is seen
    whole: 2^-200 * 2^127 and less, 2^-24 at the most for all of them."""
    from kvm_paper_b200 import window
    g = _gen(52)
    H, T = 8, 400
    q, k, v = (wh.heads_data(g, 1, H, T, dim, scale=s) for s in (1.0, 1.0, 1.0))
    q[..., 0], k[..., 0] = 1.0, 0.0
    for h in range(H):  # every eighth key: scores in units of log2
        k[0, h, h::8, 0] = far * math.log(2) * dim ** 0.5 if far > -math.inf else -math.inf
        v[0, h, h::8] = 3e38
    q, k, v = (t[:, :, 1:] if h == 0 else t for h, t in enumerate((q, k, v)))
    got = window.window_attention(q, k, v, window=None).view(1, T - 1, H, dim)
    want, mag = wh.prompt(q, k, v, None, 0)
    # (head 0's first queries may see nothing but such keys: from query 8 on every row has another one)
    want, mag, got = want[:, 8:], mag[:, 8:], got[:, 8:]
    assert float(want.abs().max()) < 10
    tol = (2 * wh.U_BF16 + 2.0 ** -8) * mag + 2.0 ** -20  # scores up to 2^10: as in the test of scores far apart
    assert bool(((got.double() - want).abs() <= tol).all())


def _timed(fn):
    fn()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out = fn()
    end.record()
    torch.cuda.synchronize()
    return out, start.elapsed_time(end)


def test_prompt_an_infinity_that_every_row_sees_costs_little():
    """An infinity in a sink: every row's values are looked through, in steps of 32 keys of about one round trip to memory
    (1000 clocks): 1024 steps of half a microsecond per row of 32768 keys, two rounds of work items."""
    from kvm_paper_b200 import window
    g = _gen(56)
    T, D = 32768, 64
    q, k, v = wh.heads_data(g, 1, 2, T, D), wh.heads_data(g, 1, 1, T, D), wh.heads_data(g, 1, 1, T, D)
    v[0, 0, 1, 9] = math.inf
    got, ms = _timed(lambda: window.window_attention(q, k, v, window=20000, sinks=4))
    assert ms < 10.0
    got = got.view(T, 2, D)
    assert bool(torch.isinf(got[1:, :, 9]).all()) and bool((got[1:, :, 9] > 0).all())
    got[1:, :, 9] = 0
    assert bool(torch.isfinite(got).all())
    v[0, 0, 1, 9] = 0
    plain = window.window_attention(q, k, v, window=20000, sinks=4).view(T, 2, D)
    plain[1:, :, 9] = 0
    assert torch.equal(got, plain)
    window.check_status()


def test_prompt_a_value_that_part_of_a_tile_does_not_see_costs_little():
    """Infinities that most of their tile's rows do not see: those rows are formed again from what they see, twice 8064 keys
    (maximum and sum, then values) of at most 2000 clocks, 18 ms; half as much again is allowed."""
    from kvm_paper_b200 import window
    g = _gen(57)
    T, D = 8192, 128
    q, k, v = wh.heads_data(g, 1, 4, T, D), wh.heads_data(g, 1, 2, T, D), wh.heads_data(g, 1, 2, T, D)
    v[0, 0, 8180, 100] = math.inf
    v[0, 1, 8150, 3] = math.nan
    got, ms = _timed(lambda: window.window_attention(q, k, v, window=None))
    assert ms < 27.0
    got = got.view(1, T, 4, D)
    assert bool(torch.isnan(got[0, 8150:, 2:, 3]).all()) and bool(torch.isinf(got[0, 8180:, :2, 100]).all())
    rows = slice(8100, T)
    want, mag = wh.prompt(q[:, :, rows], k, v, None, 0)
    got = got[:, rows]
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    wh.assert_near(torch.where(fine, got.double(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0))
    window.check_status()


@pytest.mark.parametrize("dim,hq,hkv", [(128, 3, 1), (64, 2, 2), (32, 4, 1)])
@pytest.mark.parametrize("window_,sinks", [(None, 0), (40, 70), (200, 3), (7, 0)])
def test_prompt_scattered_infinities_and_values_near_the_largest_number(dim, hq, hkv, window_, sinks):
    """Both signs in a column, in sinks, in the window and behind it; columns whose sums pass fp32's range beside them."""
    from kvm_paper_b200 import window
    g = _gen(58 + dim)
    T = 450
    q, k, v = wh.heads_data(g, 1, hq, T, dim), wh.heads_data(g, 1, hkv, T, dim), wh.heads_data(g, 1, hkv, T, dim)
    v[..., 8:12] *= 5e37
    for i, j in enumerate((0, 2, 31, 32, 69, 70, 127, 128, 200, 255, 256, 300, 301, 440, 449)):
        v[0, i % hkv, j, (5 * i) % dim] = (math.inf, -math.inf, math.nan)[i % 3]
        v[0, i % hkv, j, 20] = math.inf if i % 2 else -math.inf
    got = window.window_attention(q, k, v, window=window_, sinks=sinks).view(1, T, hq, dim)
    want, mag = wh.prompt(q, k, v, window_, sinks)
    wh.assert_near(torch.where(torch.isinf(got), 0.0, got.double()), torch.where(torch.isinf(want), 0.0, want), torch.where(torch.isinf(want), 0.0, mag))
    assert torch.equal(torch.where(torch.isinf(got), got.double(), 0.0), torch.where(torch.isinf(want), want, 0.0))
    window.check_status()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("up", [4, 6, 8, 9, 10, 13, 14, 15, 16, 17, 18, 19, 20, 30, 50, 60])
def test_prompt_scores_of_any_size(sign, up):
    from kvm_paper_b200 import window
    g = _gen(80 + up)
    for dim, hq, T, window_, sinks in ((64, 2, 500, None, 0), (128, 1, 420, 300, 128), (32, 4, 300, 100, 3)):
        k, v = _one_hot(up, sign, 1, T, dim), wh.heads_data(g, 1, 1, T, dim)
        q = torch.zeros(1, hq, T, dim, device="cuda", dtype=torch.bfloat16)
        q[..., 5] = (1 + torch.arange(T, device="cuda") % 8 / 8) * 2.0 ** up
        for scale in (None, 1.0):
            got = window.window_attention(q, k, v, window=window_, sinks=sinks, scale=scale)
            want, mag = wh.prompt(q, k, v, window_, sinks, scale)
            wh.assert_near(got.view(1, T, hq, dim), want, mag)


@pytest.mark.parametrize("bits", [4, 16])
def test_tokens_in_place_of_their_queries(bits):
    """Rows in one share and rows that are cut; the prompt call refuses it."""
    from kvm_paper_b200 import window
    g = _gen(90)
    for B, n in ((5, 40), (1, 30000)):
        c = window.WindowCache(B, 2, 64, window=n, bits=bits)
        c.write(wh.heads_data(g, B, 2, n, 64), wh.heads_data(g, B, 2, n, 64), 0)
        k1, v1 = wh.heads_data(g, B, 2, 1, 64), wh.heads_data(g, B, 2, 1, 64)
        store = torch.randn(B, 1, 8 * 64, device="cuda", generator=g).bfloat16()
        q = store.view(B, 1, 8, 64).transpose(1, 2)
        want = c.step(q.clone(), k1, v1, n)
        assert c.attend(q.clone(), n + 1).equal(want)
        assert c.step(q, k1, v1, n, out=store) is store and store.equal(want)
        with pytest.raises(ValueError, match="share memory"):
            c.attend(q[:, 0:2], 3, out=store.view(-1)[64:64 + B * 128].view(B, 1, 128))
    q, k = wh.heads_data(g, 2, 4, 50, 64), wh.heads_data(g, 2, 4, 50, 64)
    for t in (q, k):
        with pytest.raises(ValueError, match="share memory"):
            window.window_attention(q, k, k, window=9, out=t.transpose(1, 2).reshape(2, 50, 256))


@pytest.mark.parametrize("order", [(1, 0, 2), (2, 0, 1), (2, 1, 0), (1, 2, 0), (0, 2, 1)])
def test_strides_in_any_order(order):
    """Storage of batch, heads and tokens in any order (channels last), read where it lies."""
    from kvm_paper_b200 import window
    g = _gen(59)
    back = [order.index(i) for i in range(3)] + [3]
    for B, H, T, D in ((3, 4, 150, 64), (2, 2, 40, 32), (2, 3, 129, 128)):
        q, k, v = (torch.randn(*[(B, H, T)[i] for i in order], D, device="cuda", generator=g).bfloat16().permute(back) for _ in range(3))
        plain = [t.contiguous() for t in (q, k, v)]
        lens = _ints([T, T // 2, 1][:B])
        for kw in (dict(window=33, sinks=2), dict(window=None, lengths=lens)):
            assert torch.equal(window.window_attention(q, k, v, **kw), window.window_attention(*plain, **kw))
        for bits in (4, 16):
            c, c2 = (window.WindowCache(B, H, D, window=50, sinks=2, bits=bits) for _ in range(2))
            c.write(k, v, 0, lengths=lens), c2.write(*plain[1:], 0, lengths=lens)
            assert torch.equal(c.step(q[:, :, :1], k[:, :, :1], v[:, :, :1], lens), c2.step(*(t[:, :, :1].contiguous() for t in plain), lens))
            assert all(torch.equal(x, y) for x, y in zip(c.read(lens + 1), c2.read(lens + 1)))


@pytest.mark.parametrize("dim", [128, 64, 32])
def test_prompt_an_infinity_without_a_weight_is_nan(dim):
    """A key that is seen with a score of -inf has the weight 0: an infinity among its values gives 0 x inf, where another key's
    gives an infinity."""
    from kvm_paper_b200 import window
    g = _gen(91)
    T = 300
    q, k, v = (wh.heads_data(g, 1, 2, T, dim) for _ in range(3))
    q[..., 0] = 1.0
    k[0, 0, 150, 0], k[0, 1, 20:25, 0] = -math.inf, -math.inf
    v[0, 0, 150, 3], v[0, 0, 40, 7], v[0, 1, 22, 9], v[0, 1, 23, 10], v[0, 1, 25, 10] = math.inf, -math.inf, -math.inf, math.inf, math.inf
    for window_, sinks in ((None, 0), (60, 24)):
        got = window.window_attention(q, k, v, window=window_, sinks=sinks).view(1, T, 2, dim)
        want, mag = wh.prompt(q, k, v, window_, sinks)
        inf = torch.isinf(want)
        assert int(inf.sum()) > 50 and int(torch.isnan(want).sum()) > 50
        assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf])
        wh.assert_near(torch.where(inf, 0.0, got.double()), torch.where(inf, 0.0, want), torch.where(inf, 0.0, mag))


def test_prompt_of_nothing_but_infinities_costs_little():
    """Every value +inf: no key settles a column for good (a weight of 0 would make it NaN), so all of them are looked through, in
    256 steps of 32 keys that are taken in turn, some 15000 clocks: 8 ms for the four groups of columns of the longest rows;
    twice that is allowed.  (With the score of every key it was 86 ms.)"""
    from kvm_paper_b200 import window
    g = _gen(92)
    T = 8192
    q, k = wh.heads_data(g, 1, 4, T, 128), wh.heads_data(g, 1, 2, T, 128)
    v = torch.full((1, 2, T, 128), math.inf, device="cuda", dtype=torch.bfloat16)
    got, ms = _timed(lambda: window.window_attention(q, k, v, window=None))
    assert bool((got == math.inf).all()) and ms < 16.0


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 20, 2.0 ** 24, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28])
def test_token_equal_large_scores_of_values_near_the_largest_number(bits, size):
    """Keys that share the weight, however large their scores: sums that are not normalised yet stay in range."""
    from kvm_paper_b200 import window
    n, dim = 700, 64
    k, v = torch.zeros(1, 1, n, dim, device="cuda", dtype=torch.bfloat16), torch.full((1, 1, n, dim), 3e38, device="cuda", dtype=torch.bfloat16)
    v[..., 32:] = -3e38
    k[..., 5] = 6.0  # (a scale of 1 and the largest level: exact)
    q = torch.zeros(1, 3, 1, dim, device="cuda", dtype=torch.bfloat16)
    q[..., 5] = torch.tensor([size, size * 1.5, -size], device="cuda").view(1, 3, 1)
    c = window.WindowCache(1, 1, dim, window=n, bits=bits)
    c.write(k, v, 0)
    got = c.attend(q, n, scale=0.25).view(3, dim)
    held = c.read(n)[1][0, 0, :1]
    assert torch.allclose(got.double(), held.double().expand(3, dim), rtol=2 * wh.U_BF16, atol=0)
