"""Shared decode attention by sets of 32 and 64 columns, which groups of that many query heads take, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from paged_util import attention_oracle, check_attention
from test_gpu_paged_shared import MANY, Shared

pytestmark = pytest.mark.gpu
F16, BF16, FP8 = M.FLOAT16, M.BFLOAT16, M.F8E4M3
FOUR = [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)]


def own_tokens(s):
    """The most that a request has for itself."""
    shared = [0] * len(s.lengths)
    for g, x in enumerate(s.shared):
        for r in range(s.starts[g], s.starts[g + 1]):
            shared[r] = x
    return max(x - y for x, y in zip(s.lengths, shared))


def run(s, most_shared=None):
    """A call with the bounds as they are; its groups have 17 columns and more on average, and 33 and more are cut into
    64s if there is no less to share than each has for itself (and heads are no wider than 128).  From 256 on it
    takes long shared tokens for another way."""
    most_shared = max(s.shared) if most_shared is None else most_shared
    each, own = len(s.lengths) * (s.hq // s.hk) // len(s.shared), own_tokens(s)
    assert each > 16 and own <= most_shared and (each < 256 or each * most_shared < 1 << 22)
    return s.run(most_shared=most_shared, most_own=own)


@pytest.mark.parametrize("dtype, cache", FOUR)
@pytest.mark.parametrize("hq, hk, dim, page, order", [(16, 1, 64, 16, "head"), (24, 2, 128, 32, "token"), (60, 1, 128, 7, "head"), (8, 1, 80, 48, "head"),
                                                      (32, 2, 48, 1, "token"), (33, 1, 112, 100, "head"), (20, 2, 16, 24, "token"), (48, 4, 96, 64, "head")])
def test_64_columns_against_f64(dtype, cache, hq, hk, dim, page, order):
    s = Shared(dtype, cache, MANY, hq, hk, dim, page, order, seed=dim + page, q_std=2.0, outside=((5, 0, 90), (33,)))
    assert len(s.lengths) * (hq // hk) // len(MANY) > 32
    s.check(*run(s))


@pytest.mark.parametrize("dtype, cache", FOUR)
@pytest.mark.parametrize("hq, hk, dim, page, order", [(10, 2, 128, 16, "head"), (5, 1, 64, 10, "token"), (24, 4, 128, 9, "head"), (5, 1, 112, 128, "head"),
                                                      (5, 1, 256, 16, "token"), (40, 1, 256, 12, "head"), (32, 2, 192, 64, "head")])
def test_32_columns_against_f64(dtype, cache, hq, hk, dim, page, order):
    s = Shared(dtype, cache, MANY, hq, hk, dim, page, order, seed=dim + page, q_std=2.0, outside=((5, 0), (33,)))
    assert len(s.lengths) * (hq // hk) // len(MANY) <= 32 or dim > 128
    s.check(*run(s))


@pytest.mark.parametrize("option", [dict(window=1), dict(window=16), dict(window=33), dict(window=130), dict(window=10 ** 9), dict(softcap=20.0), dict(slopes=True),
                                    dict(slopes=True, softcap=5.0, window=40), dict(scale=-0.3), dict(scale=0.0), dict(softcap=1e-3), dict(softcap=1e5)])
@pytest.mark.parametrize("page, dim, heads", [(16, 64, 16), (10, 128, 16), (16, 128, 5)])
def test_window_cap_and_bias(option, page, dim, heads):
    s = Shared(BF16, BF16, MANY, heads, 1, dim, page, seed=5, q_std=3.0, **dict(option))
    s.check(*run(s))


@pytest.mark.parametrize("members, group", [(3, 11), (5, 8), (9, 7), (8, 8), (5, 13), (33, 3), (2, 64), (13, 10), (63, 4), (51, 5)])
@pytest.mark.parametrize("dim, cache, page", [(64, F16, 16), (128, FP8, 10)])
def test_columns_of_every_number(members, group, dim, cache, page):
    s = Shared(F16, cache, [(300, [300 + 3 * i for i in range(members)])], group, 1, dim, page, seed=members)
    s.check(*run(s))


@pytest.mark.parametrize("dim, page, heads", [(64, 16, 16), (128, 12, 16), (128, 64, 6), (256, 16, 16)])
def test_several_parts_and_a_page_outside_the_cache(dim, page, heads):
    s = Shared(BF16, BF16, [(3000, [3001, 3100, 2990, 3000, 3600])], heads, 1, dim, page, seed=6)
    first = run(s)
    s.check(*first)
    again = run(s)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    at = 1600 // page
    s.table[0, at] = -1
    out, lse = run(s)
    for r in (0, 2, 4):
        x = s.lengths[r]
        keep = torch.arange(x)
        keep = keep[keep // page != at]
        want = attention_oracle(s.q[r: r + 1].double(), s.kv[r][0][keep], s.kv[r][1][keep], [10 ** 6], s.scale)
        check_attention(out[r: r + 1], lse[r: r + 1], want, BF16, dim)


@pytest.mark.parametrize("cache", [BF16, FP8])
@pytest.mark.parametrize("page, heads", [(16, 16), (10, 16), (16, 8), (10, 8)])
def test_not_finite_values_of_which_some_columns_see_none(cache, page, heads):
    s = Shared(BF16, cache, [(100, [101, 130, 140, 60])], heads, 1, 64, page, seed=12, window=50)
    want = s.oracle()

    def put(t, which, dim, value):
        s.cache.views[which][int(s.table[0, t // page]), t % page, 0, dim] = 127 if cache == FP8 else value

    for t, dim, what in ((70, 5, math.inf), (20, 6, math.inf), (99, 7, math.nan)):
        put(t, 1, dim, what)
    out, lse = run(s)
    got, exact = out.double().cpu(), want[0]
    assert torch.isfinite(got[:, :, 8:]).all() and torch.isfinite(lse).all()
    for dim, rows in {5: [0], 6: [3], 7: [0, 1, 2]}.items():
        for r in range(4):
            if r in rows:
                assert (torch.isnan(got[r, :, dim]) if dim == 7 or cache == FP8 else got[r, :, dim] == math.inf).all(), (dim, r)
            else:
                assert ((got[r, :, dim] - exact[r, :, dim]).abs() < 0.05).all(), (dim, r)
    put(70, 0, 3, math.nan)  # a key: the first request's row is NaN, the others' stay
    out, lse = run(s)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.isfinite(lse[1:]).all()
    assert torch.isfinite(out[1:][:, :, 8:]).all()


def test_large_scores_and_scores_that_rise_and_fall():
    s = Shared(BF16, BF16, [(300, [310, 301, 364])], 16, 1, 64, 16, seed=2, q_std=40.0)  # weights of one token alone
    s.check(*run(s))
    s = Shared(F16, F16, [(2048, [2050, 2100])], 20, 1, 64, 16, seed=3, slopes=True)
    s.slopes = torch.linspace(-3.0, 3.0, 20)
    s.check(*run(s))


@pytest.mark.parametrize("heads, most_shared", [(16, None), (100, 1 << 24)])  # 64 columns, and prefill's kernels
def test_what_cannot_be_is_never_followed(heads, most_shared):
    s = Shared(F16, F16, [(64, [64, 64, 70]), (16, [30, 31, 16])], heads, 1, 64, 16, seed=10)
    most_shared = most_shared or 70
    want = s.oracle()
    lengths = s.lengths
    s.lengths, s.shared = [10 ** 9, -4, 70, 30, 31, 16], [64, -7]
    out, lse = s.run(most_shared, 70)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    s.check(out, lse, slice(2, 3), want)
    s.lengths, s.shared = lengths, [64, 16]
    # starts that fall, or are no requests: whatever comes out, nothing else is touched
    for starts in ([6, -3, 100], [2 ** 31 - 1, -2 ** 31, 0], [0, 6, 1], [0, 6, 6]):
        s.starts = starts
        s.run(most_shared, 70)
