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
