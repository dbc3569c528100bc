"""Attention of new tokens over a paged cache, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import TORCH, Cache, attention_oracle, check_attention, ptr, stream

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = M.FLOAT32, M.FLOAT16, M.BFLOAT16, M.F8E4M3
# (cached before, new) of each request
MIXED = [(0, 1), (0, 0), (0, 33), (7, 64), (63, 2), (0, 130), (200, 17), (64, 64), (5, 0)]


class Chunk:
    def __init__(self, dtype, cache_dtype, requests, hq, hk, dim, page, order="head", seed=0, q_std=1.0, prefix=None, gap=0, **option):
        M.init(0)
        self.dtype, self.requests, self.hq, self.hk, self.dim = dtype, requests, hq, hk, dim
        scales = dict(k_scale=0.0625, v_scale=0.5) if cache_dtype == FP8 else {}
        self.lengths = [p + f for p, f in requests]
        self.starts = [0]
        for _, f in requests:
            self.starts.append(self.starts[-1] + f)
        width = max(1, max(-(-x // page) for x in self.lengths))
        self.cache = Cache(cache_dtype, page, hk, dim, sum(-(-x // page) for x in self.lengths) + 1, order, seed, gap=gap, **scales)
        self.table = torch.full((len(requests), width + 1), -7, dtype=torch.int32)
        std = 1 / scales["k_scale"] if scales else 1.0
        self.kv = [self.cache.put(x, self.table[r], std) for r, x in enumerate(self.lengths)]
        self.q = (torch.randn(self.starts[-1], hq, dim, generator=self.cache.gen) * q_std).to(TORCH[dtype])
        self.prefix, self.option = prefix, option
        self.scale = option.pop("scale", dim ** -0.5)
        self.slopes = torch.rand(hq, generator=self.cache.gen) * 0.3 if option.pop("slopes", False) else None

    def run(self, tokens=None, most=None, longest=None, workspace=True, share=1.0, shape=None, q=None, out=None, on=None):
        n, width = len(self.requests), self.table.shape[1] - 1
        shape = shape or A.Attention(self.dtype, self.hq, self.scale, **self.option)
        tokens = self.starts[-1] if tokens is None else tokens
        most = max(f for _, f in self.requests) if most is None else most
        longest = max(self.lengths) if longest is None else longest
        d = lambda t: None if t is None else t.cuda()  # noqa: E731
        i32 = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        self.keep = q_, table, starts, lengths, prefix, slopes = (d(self.q) if q is None else q, d(self.table), i32(self.starts), i32(self.lengths),
                                                                 i32(self.prefix), d(self.slopes))
        out = torch.full((self.starts[-1], self.hq, self.dim), math.nan, dtype=TORCH[self.dtype], device="cuda") if out is None else out
        lse = torch.full((self.starts[-1], self.hq), math.nan, device="cuda")
        need = A.paged_prefill_workspace(shape, self.cache.desc, n, tokens, most, longest) if workspace else 0
        need = int(need * share)
        ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        A.paged_prefill(shape, self.cache.desc, n, tokens, most, ptr(q_), ptr(self.cache.buffers[0]), ptr(self.cache.buffers[1]), ptr(table), width,
                        ptr(starts), ptr(lengths), longest, ptr(prefix), ptr(slopes), ptr(out), ptr(lse), ptr(ws) if need else 0, need,
                        table_stride=width + 1, stream=stream() if on is None else on)
        torch.cuda.synchronize()
        return out, lse

    def oracle(self):
        rows = []
        for r, (past, fresh) in enumerate(self.requests):
            k, v = self.kv[r]
            positions = [self.lengths[r] - fresh + i for i in range(fresh)]
            prefix = min(max(self.prefix[r], 0), self.lengths[r]) if self.prefix else 0
            rows.append(attention_oracle(self.q[self.starts[r]: self.starts[r + 1]].double(), k, v, positions, self.scale,
                                         self.option.get("softcap", 0.0), self.option.get("window", 0), self.slopes, prefix))
        return [torch.cat(t) for t in zip(*rows)]

    def check(self, out, lse):
        reach = 0.0 if self.slopes is None else float(self.slopes.max()) * max(self.lengths)
        check_attention(out, lse, self.oracle(), self.dtype, self.dim, self.option.get("softcap", 0.0), reach)


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("hq, hk, dim, page, order", [(4, 1, 128, 16, "head"), (3, 3, 64, 1, "token"), (6, 2, 80, 7, "head"), (2, 1, 256, 48, "token"),
                                                      (10, 1, 96, 100, "head"), (2, 2, 16, 32, "token"), (2, 1, 192, 64, "head"), (3, 1, 112, 256, "token")])
def test_mixed_requests_against_f64(dtype, cache, hq, hk, dim, page, order):
    c = Chunk(dtype, cache, MIXED, hq, hk, dim, page, order, seed=dim + page, q_std=2.0)
    c.check(*c.run())


@pytest.mark.parametrize("dim", [8, 24, 72, 88, 136, 248])
def test_head_dims_that_end_inside_a_product(dim):
    c = Chunk(F16, F16, [(3, 40), (0, 70)], 2, 1, dim, 16, seed=dim, gap=3)
    c.check(*c.run())


PREFIX = [0, 3, 40, 1, 65, 10, 217, 500, 5]


@pytest.mark.parametrize("option", [dict(window=1), dict(window=16), dict(window=70), dict(softcap=20.0), dict(slopes=True), dict(prefix=PREFIX),
                                    dict(prefix=PREFIX, window=5), dict(prefix=PREFIX, window=66, slopes=True, softcap=8.0), dict(scale=-0.3),
                                    dict(prefix=[-3] * 9, window=2 ** 31 - 1)])
@pytest.mark.parametrize("page", [16, 10])
def test_masks_cap_and_bias(option, page):
    c = Chunk(BF16, BF16, MIXED, 4, 2, 64, page, seed=5, q_std=3.0, **dict(option))
    c.check(*c.run())


def test_a_window_far_behind_a_prefix_skips_what_lies_between():
    c = Chunk(F16, F16, [(1500, 40)], 2, 1, 64, 16, seed=8, window=30, prefix=[70])
    k, v = c.kv[0]
    for view, t in ((c.cache.views[0], torch.arange(80, 1460)), (c.cache.views[1], torch.arange(80, 1460))):
        view[c.table[0, t // 16].long().cuda(), (t % 16).cuda()] = math.nan  # nobody sees these
    c.check(*c.run())


def test_tokens_that_see_nothing_give_zeros():
    # more new tokens than the request is long: the first ones stand before its beginning
    c = Chunk(BF16, BF16, [(0, 40), (0, 5)], 4, 2, 64, 16, seed=3)
    c.lengths = [10, 0]
    c.kv = [(k[:n], v[:n]) for (k, v), n in zip(c.kv, c.lengths)]
    out, lse = c.run()
    assert (out[:30] == 0).all() and (out[40:] == 0).all() and (lse[:30] == -math.inf).all()
    c.check(out, lse)


def test_masked_places_may_hold_anything():
    # inf, -inf and NaN in keys and values of later tokens of the same tile: rows before them do not see them, rows from
    # them on do
    c = Chunk(F16, F16, [(20, 60)], 2, 1, 64, 16, seed=4)
    clean, lse_clean = c.run()
    bad = {50: math.nan, 60: math.inf, 70: -math.inf}
    for t, value in bad.items():
        c.cache.views[1][int(c.table[0, t // 16]), t % 16, 0, 7] = value
    out, lse = c.run()
    others = torch.arange(64) != 7
    assert torch.equal(lse, lse_clean) and torch.equal(out[:, :, others], clean[:, :, others])
    assert torch.equal(out[:30], clean[:30]) and torch.isnan(out[30:, :, 7]).all()
    c = Chunk(F16, F16, [(20, 60)], 2, 1, 64, 16, seed=4)
    for t, value in ((60, math.inf), (70, -math.inf)):
        c.cache.views[1][int(c.table[0, t // 16]), t % 16, 0, 7] = value
    out, _ = c.run()
    assert (out[40:50, :, 7] == math.inf).all() and torch.isnan(out[50:, :, 7]).all() and torch.equal(out[:40], clean[:40])
    c = Chunk(F16, F16, [(20, 60)], 2, 1, 64, 16, seed=4)
    c.cache.views[0][int(c.table[0, 3]), 2, 0, 9] = math.nan  # a key: token 50
    out, lse = c.run()
    assert torch.equal(out[:30], clean[:30]) and torch.equal(lse[:30], lse_clean[:30]) and torch.isnan(out[30:]).all()


def test_a_page_outside_the_cache_counts_as_masked():
    c = Chunk(BF16, BF16, [(0, 64)], 2, 1, 64, 16, seed=9)
    c.table[0, 1], c.table[0, 2] = 10 ** 6, -1
    k, v = c.kv[0]
    keep = torch.cat([torch.arange(16), torch.arange(48, 64)])
    out, lse = c.run()
    for i in (0, 15, 16, 30, 47, 48, 63):
        seen = keep[keep <= i]
        check_attention(out[i: i + 1], lse[i: i + 1], attention_oracle(c.q[i: i + 1].double(), k[seen], v[seen], [10 ** 6], c.scale), BF16, 64)


def test_rows_past_the_bounds_are_left_alone():
    c = Chunk(BF16, BF16, [(0, 40), (3, 60)], 2, 1, 64, 16, seed=11)
    out, lse = c.run(most=50)
    want = c.oracle()
    done = list(range(40)) + list(range(40, 90))
    check_attention(out[done], lse[done], [t[done] for t in want], BF16, 64)
    assert torch.isnan(out[90:]).all() and torch.isnan(lse[90:]).all()
    # starts past the rows of q and out: the second request has 25 rows, its last positions
    out, lse = c.run(tokens=65)
    assert torch.isfinite(out[:65]).all() and torch.isnan(out[65:]).all()
    check_attention(out[:40], lse[:40], [t[:40] for t in want], BF16, 64)


def test_one_new_token_is_decode():
    lengths = [1, 16, 17, 130, 600]
    c = Chunk(F16, F16, [(x - 1, 1) for x in lengths], 6, 2, 128, 16, seed=6)
    out, lse = c.run()
    c.check(out, lse)
    q, table, n = c.q.cuda(), c.table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    shape, width = A.Attention(F16, 6, c.scale), c.table.shape[1] - 1
    got, got_lse = torch.empty_like(q), torch.empty(5, 6, device="cuda")
    A.paged_decode(shape, c.cache.desc, 5, ptr(q), ptr(c.cache.buffers[0]), ptr(c.cache.buffers[1]), ptr(table), width, ptr(n), 600, 0, ptr(got),
                   ptr(got_lse), table_stride=width + 1, stream=stream())
    c.check(got, got_lse)


@pytest.mark.parametrize("hq, hk, dim", [(8, 2, 64), (3, 1, 128), (2, 1, 256)])
def test_few_rows_over_a_long_context(hq, hk, dim):
    # split over the keys, with the workspace that is asked for, with little, with none; joined in a fixed order
    c = Chunk(BF16, BF16, [(3000, 9), (0, 0), (100, 3), (0, 1)], hq, hk, dim, 16, seed=7, slopes=True)
    first = c.run()
    c.check(*first)
    c.check(*c.run(workspace=False))
    for longest in (1, 10 ** 9):
        c.check(*c.run(longest=longest))
    again = c.run()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# A large bound of the lengths: workgroups of eight waves, whole and in parts.
@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("hq, hk, dim, page, order", [(4, 1, 128, 16, "head"), (3, 1, 64, 1, "token"), (6, 2, 80, 7, "head"), (2, 1, 112, 256, "token")])
def test_a_large_bound_of_the_lengths(dtype, cache, hq, hk, dim, page, order):
    c = Chunk(dtype, cache, MIXED + [(900, 40)], hq, hk, dim, page, order, seed=dim + page, q_std=2.0)
    for workspace in (False, True):
        c.check(*c.run(longest=10 ** 9, workspace=workspace))


@pytest.mark.parametrize("option", [dict(window=1), dict(window=70), dict(slopes=True), dict(prefix=PREFIX), dict(prefix=PREFIX, window=66, slopes=True, softcap=8.0),
                                    dict(scale=-0.3)])
@pytest.mark.parametrize("page, dim", [(16, 128), (10, 64)])
def test_masks_cap_and_bias_under_a_large_bound(option, page, dim):
    c = Chunk(BF16, BF16, MIXED, 4, 2, dim, page, seed=5, q_std=3.0, **dict(option))
    for workspace in (False, True):
        c.check(*c.run(longest=10 ** 9, workspace=workspace))


@pytest.mark.parametrize("dim", [64, 128])
def test_masked_places_under_a_large_bound(dim):
    def chunk():
        return Chunk(F16, F16, [(300, 180)], 2, 1, dim, 16, seed=4)

    c = chunk()
    clean, lse_clean = c.run(longest=10 ** 9)
    c.check(clean, lse_clean)
    for t, value in ((330, math.inf), (400, math.nan), (470, -math.inf)):
        c.cache.views[1][int(c.table[0, t // 16]), t % 16, 0, 7] = value
    for workspace in (False, True):
        out, lse = c.run(longest=10 ** 9, workspace=workspace)
        others = torch.arange(dim) != 7
        check_attention(out[:, :, others], lse, [x[:, :, others] if x.ndim == 3 else x for x in c.oracle()], F16, dim)
        assert torch.isfinite(out[:30, :, 7]).all() and (out[30:100, :, 7] == math.inf).all() and torch.isnan(out[100:, :, 7]).all()
    c = chunk()
    c.cache.views[0][int(c.table[0, 25]), 2, 0, 9] = math.nan  # a key: token 402
    out, lse = c.run(longest=10 ** 9)
    assert torch.equal(out[:102], clean[:102]) and torch.equal(lse[:102], lse_clean[:102]) and torch.isnan(out[102:]).all()


def test_a_page_outside_the_cache_under_a_large_bound():
    c = Chunk(BF16, BF16, [(0, 200)], 1, 1, 64, 16, seed=9)
    c.table[0, 1], c.table[0, 10] = 10 ** 6, -1
    k, v = c.kv[0]
    keep = torch.cat([torch.arange(16), torch.arange(32, 160), torch.arange(176, 200)])
    for workspace in (False, True):
        out, lse = c.run(longest=10 ** 9, workspace=workspace)
        for i in (0, 15, 16, 31, 32, 127, 128, 159, 160, 175, 176, 199):
            seen = keep[keep <= i]
            check_attention(out[i: i + 1], lse[i: i + 1], attention_oracle(c.q[i: i + 1].double(), k[seen], v[seen], [10 ** 6], c.scale), BF16, 64)


@pytest.mark.parametrize("share", [0.03, 0.3, 0.5, 0.999])
@pytest.mark.parametrize("dim", [64, 256])
def test_less_workspace_than_is_asked_for(share, dim):
    c = Chunk(F16, F16, [(3000, 9), (700, 5)], 4, 2, dim, 16, seed=17)
    c.check(*c.run(share=share))


def test_large_scores_and_the_moving_reference():
    c = Chunk(F16, F16, [(0, 300)], 2, 1, 64, 16, seed=3, slopes=True)
    c.slopes = torch.tensor([3.0, -3.0])
    out, lse = c.run()
    check_attention(out, lse, c.oracle(), F16, 64, slope_reach=3.0 * 300)
    c = Chunk(BF16, BF16, [(0, 200)], 2, 1, 64, 16, seed=3, q_std=40.0)
    c.check(*c.run())


def test_strided_queries_and_results():
    c = Chunk(BF16, BF16, [(4, 70), (0, 3)], 4, 2, 32, 16, seed=13)
    n, row = 73, 4 * 32 + 2 * 2 * 32 + 1
    packed = torch.full((n * row + 1,), math.nan, dtype=torch.bfloat16, device="cuda")
    q = torch.as_strided(packed, (n, 4, 32), (row, 32, 1), 1)
    q.copy_(c.q)
    big = torch.full((4, n, 51), -5.0, dtype=torch.bfloat16, device="cuda")  # [head, token, dim], rows that start anywhere
    shape = A.Attention(BF16, 4, c.scale, q_strides=(row, 32), out_strides=(51, 51 * n))
    _, lse = c.run(shape=shape, q=q, out=big)
    c.check(big[:, :, :32].transpose(0, 1), lse)
    assert (big[:, :, 32:] == -5).all()


def test_pages_far_apart():
    M.init(0)
    dim, page, stride, pages = 64, 16, 1_300_000_000, 3
    k, v = (torch.empty(stride * (pages - 1) + page * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(1)
    ks, vs = (torch.randn(48, 1, dim, generator=gen).bfloat16() for _ in range(2))
    order = [2, 0, 1]
    for t, x in ((k, ks), (v, vs)):
        for j, p in enumerate(order):
            t[p * stride: p * stride + page * dim] = x[16 * j: 16 * j + 16].reshape(-1).cuda()
    q = torch.randn(48, 2, dim, generator=gen).bfloat16()
    d = [t.cuda() for t in (q, torch.tensor([order], dtype=torch.int32), torch.tensor([0, 48], dtype=torch.int32), torch.tensor([48], dtype=torch.int32))]
    out, lse = torch.empty_like(d[0]), torch.empty(48, 2, device="cuda")
    A.paged_prefill(A.Attention(BF16, 2, 0.125), A.KVCache(BF16, page, 1, dim, pages, page_stride=stride), 1, 48, 48, ptr(d[0]), ptr(k), ptr(v),
                    ptr(d[1]), 3, ptr(d[2]), ptr(d[3]), 48, 0, 0, ptr(out), ptr(lse), stream=stream())
    want = attention_oracle(q.double(), ks.double(), vs.double(), list(range(48)), 0.125)
    check_attention(out, lse, want, BF16, dim)


def test_another_stream():
    c = Chunk(BF16, BF16, MIXED, 4, 2, 64, 16, seed=14)
    c.check(*c.run(on=torch.cuda.Stream().cuda_stream))


def test_refused_arguments():
    M.init(0)
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = ptr(t)

    def call(cache=None, shape=None, **args):
        base = dict(requests=1, tokens=2, most_fresh=2, q=p, k_cache=p, v_cache=p, table=p, table_width=4, starts=p, lengths=p, longest=64, prefix=0,
                    slopes=0, out=p, lse=0)
        A.paged_prefill(A.Attention(**{"dtype": BF16, "q_heads": 4, "scale": 1.0, **(shape or {})}),
                        A.KVCache(**{"dtype": BF16, "page_size": 16, "kv_heads": 2, "head_dim": 64, "pages": 4, **(cache or {})}), **{**base, **args})

    for bad, message in ((dict(shape=dict(dtype=F32)), "f16/bf16"), (dict(shape=dict(dtype=F16)), "over a cache"), (dict(shape=dict(q_heads=3)), "evenly"),
                         (dict(shape=dict(window=-1)), "window"), (dict(cache=dict(head_dim=60)), "multiple of 8"), (dict(requests=-1), "requests"),
                         (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 30) + 1), "tokens"), (dict(most_fresh=-1), "at most"),
                         (dict(table_stride=3), "table width"), (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(starts=0), "NULL"),
                         (dict(lengths=0), "NULL"), (dict(k_cache=0), "NULL"), (dict(workspace=p + 8, workspace_bytes=64), "workspace")):
        with pytest.raises(M.MFHError, match=message):
            call(**bad)
    call(tokens=0, q=0)
    call(most_fresh=0, q=0)
    with pytest.raises(M.MFHError, match="requests"):
        A.paged_prefill_workspace(A.Attention(BF16, 4, 1.0), A.KVCache(BF16, 16, 2, 64, 4), -1, 2, 2, 5)


@pytest.mark.parametrize("cap", [60.0, 64.0, 65.0, 1e3, 1e5, 1e7, 1e30, 8e37])
@pytest.mark.parametrize("dtype, cache", [(F16, F16), (BF16, FP8)])
def test_caps_far_above_the_scores_leave_them_as_they_are(cap, dtype, cache):
    # the bounds go by the scores alone, whatever the cap; of a prompt's first token lse is the score
    c = Chunk(dtype, cache, [(0, 1), (0, 1), (0, 3), (0, 140), (60, 20)], 8, 2, 16, 16, seed=31, q_std=6.0, softcap=cap)
    for longest in (None, 10 ** 9):
        out, lse = c.run(longest=longest)
        check_attention(out, lse, c.oracle(), dtype, 16)


@pytest.mark.parametrize("cap", [65.0, 1e3])
def test_large_caps_still_cap(cap):
    c = Chunk(F16, F16, [(0, 1), (0, 140), (60, 20)], 4, 2, 16, 16, seed=32, q_std=60.0, scale=4.0, softcap=cap)
    out, lse = c.run()
    assert c.oracle()[3].max() > cap
    check_attention(out, lse, c.oracle(), F16, 16)


@pytest.mark.parametrize("below", [14.0, 16.5])
@pytest.mark.parametrize("workspace", [True, False])
def test_many_small_weights_beside_a_large_one(below, workspace):
    # one key far above a long context, whose weights are each near the smallest 16-bit number: together they are all of the result
    n = 60000
    c = Chunk(F16, F16, [(n - 2, 2)], 2, 1, 64, 16, seed=41, scale=0.125)
    c.q[:] = 0
    c.q[..., 0] = 8.0
    k, v = c.kv[0]
    k[:, 0, 0] = -below + (0.0 if below > 15 else 1.0) * torch.randn(n, generator=c.cache.gen).half().double().clamp(-4, 4)
    k[:, 0, 0] = k[:, 0, 0].half().double()
    k[5, 0, 0], v[:, 0] = 0.0, (v[:, 0].abs() + 0.5).half().double()
    v[5] = 0.0
    t = torch.arange(n)
    for view, x in zip(c.cache.views, (k, v)):
        view[c.table[0, t // 16].long().cuda(), (t % 16).cuda()] = x.half().cuda()
    out, lse = c.run(workspace=workspace)
    want = c.oracle()
    # besides every weight's relative rounding, a half step of its type: 2^-25 where the largest weight is 2^7 or more
    tail = n * 2.0 ** -32 * v.abs().max()
    u, got = 2.0 ** -11, out.double().cpu()
    assert ((got - want[0]).abs() <= u * want[0].abs() + want[2] * (u + 2.0 ** -14) + tail).all(), float(((got - want[0]) / want[0]).abs().max())
    assert (lse.double().cpu() - want[1]).abs().max() <= 2.0 ** -15


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("fresh", [3, 600])
def test_values_near_the_largest_number_stay_finite(fresh, workspace):
    # the value of a late key whose score is above all before it: weights are never above 1 there
    c = Chunk(BF16, BF16, [(700 - fresh, fresh)], 2, 1, 64, 16, seed=51, scale=0.125)
    c.q[:] = 0
    c.q[..., 0] = 8.0
    k, v = c.kv[0]
    k[:, 0, 0] = 0.0
    k[130, 0, 0], v[130] = 5.0, 2.0 ** 126
    t = torch.arange(700)
    for view, x in zip(c.cache.views, (k, v)):
        view[c.table[0, t // 16].long().cuda(), (t % 16).cuda()] = x.bfloat16().cuda()
    c.check(*c.run(workspace=workspace))
    c.check(*c.run(workspace=workspace, longest=10 ** 9))


@pytest.mark.parametrize("longest", [None, 10 ** 9])
@pytest.mark.parametrize("page", [1, 7, 16, 24, 128])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_whose_tokens_are_one_row(page, dim, longest):
    # a token stride of 0: every token of a page has the page's one key and value
    M.init(0)
    gen = torch.Generator().manual_seed(page)
    n, past = 300, 120
    pages = -(-n // page) + 1
    k, v = (torch.randn(pages, dim, generator=gen).bfloat16() for _ in range(2))
    table = torch.randperm(pages, generator=gen)[: pages - 1].to(torch.int32)
    q = torch.randn(n - past, 2, dim, generator=gen).bfloat16()
    d = [t.cuda() for t in (q, k, v, table, torch.tensor([0, n - past], dtype=torch.int32), torch.tensor([n], dtype=torch.int32))]
    out, lse = torch.full_like(d[0], math.nan), torch.empty(n - past, 2, device="cuda")
    desc, shape = A.KVCache(BF16, page, 1, dim, pages, page_stride=dim, token_stride=0, head_stride=dim), A.Attention(BF16, 2, dim ** -0.5)
    A.paged_prefill(shape, desc, 1, n - past, n - past, ptr(d[0]), ptr(d[1]), ptr(d[2]), ptr(d[3]), pages - 1, ptr(d[4]), ptr(d[5]), longest or n, 0, 0,
                    ptr(out), ptr(lse), stream=stream())
    at = table[torch.arange(n) // page].long()
    want = attention_oracle(q.double(), k[at].double()[:, None], v[at].double()[:, None], list(range(past, n)), dim ** -0.5)
    check_attention(out, lse, want, BF16, dim)


def test_more_rows_than_one_launch_dimension_joins():
    # few of very many rows are computed, over a context long enough for parts
    M.init(0)
    tokens, heads, dim, length = 2 ** 26 + 8, 4, 8, 3000
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GB of device memory")
    c = Chunk(F16, F16, [(length - 3, 3)], heads, 1, dim, 16, seed=61)
    q = torch.zeros(tokens, heads, dim, dtype=torch.float16, device="cuda")
    q[:3] = c.q.cuda()
    out = torch.full((tokens, heads, dim), -3.0, dtype=torch.float16, device="cuda")
    lse = torch.full((tokens, heads), -3.0, device="cuda")
    d = [t.cuda() for t in (c.table, torch.tensor([0, 3], dtype=torch.int32), torch.tensor([length], dtype=torch.int32))]
    shape, width = A.Attention(F16, heads, c.scale), c.table.shape[1] - 1
    room = tokens * heads * 2 * (dim + 2) * 4  # of two parts
    ws = torch.empty(room, dtype=torch.uint8, device="cuda")
    A.paged_prefill(shape, c.cache.desc, 1, tokens, 3, ptr(q), ptr(c.cache.buffers[0]), ptr(c.cache.buffers[1]), ptr(d[0]), width, ptr(d[1]), ptr(d[2]), length, 0,
                    0, ptr(out), ptr(lse), ptr(ws), room, table_stride=width + 1, stream=stream())
    c.check(out[:3], lse[:3])
    assert (out[3:] == -3).all() and (lse[3:] == -3).all()


def test_caps_too_small_for_their_reciprocal_beside_a_scale():
    # every score that is not zero ends at the cap, which is as good as zero; a zero stays one
    c = Chunk(F16, F16, [(3, 70)], 2, 1, 64, 16, seed=71, scale=100.0, softcap=2.0 ** -125)
    c.q[5] = 0
    for longest in (None, 10 ** 9):
        c.check(*c.run(longest=longest))


def test_a_captured_call():
    # lengths, starts and pages are read on the device at each replay
    c = Chunk(BF16, BF16, [(1500, 20), (0, 0), (40, 9), (0, 3)], 4, 2, 64, 16, seed=15)
    shape, width = A.Attention(BF16, 4, c.scale), c.table.shape[1] - 1
    tokens, most, longest, n = c.starts[-1], 20, 2000, 4
    q, table = c.q.cuda(), c.table.cuda()
    starts, lengths = (torch.tensor(v, dtype=torch.int32).cuda() for v in (c.starts, c.lengths))
    out, lse = torch.empty_like(q), torch.empty(tokens, 4, device="cuda")
    need = A.paged_prefill_workspace(shape, c.cache.desc, n, tokens, most, longest)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call():
        A.paged_prefill(shape, c.cache.desc, n, tokens, most, ptr(q), ptr(c.cache.buffers[0]), ptr(c.cache.buffers[1]), ptr(table), width, ptr(starts),
                        ptr(lengths), longest, 0, 0, ptr(out), ptr(lse), ptr(ws), need, table_stride=width + 1, stream=stream())

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    full, kv = list(c.lengths), c.kv
    for now, new in ((full, [20, 0, 9, 3]), ([1520, 0, 11, 0], [20, 0, 11, 0]), ([700, 0, 49, 2], [1, 0, 17, 2]), (full, [20, 0, 9, 3])):
        c.requests, c.lengths = [(x - f, f) for x, f in zip(now, new)], now
        c.kv = [(k[:x], v[:x]) for (k, v), x in zip(kv, now)]
        c.starts = [sum(new[:i]) for i in range(5)]
        starts.copy_(torch.tensor(c.starts, dtype=torch.int32))
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        rows = c.starts[-1]
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        c.check(out[:rows], lse[:rows])
        replayed = out.clone(), lse.clone()
        out.fill_(math.nan)
        call()
        torch.cuda.synchronize()
        assert torch.equal(replayed[0][:rows], out[:rows]) and torch.equal(replayed[1][:rows], lse[:rows]) and torch.isnan(replayed[0][rows:]).all()


def test_one_new_token_beside_a_request_without_one():
    # as many rows as two of three requests: not a decode step, whose rows stand one per request
    c = Chunk(BF16, BF16, [(40, 1), (25, 0), (300, 1)], 4, 2, 64, 16, seed=16)
    c.check(*c.run())


@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("prefix", [None, [40, 0]])
def test_pages_behind_a_window_may_be_gone(page, prefix):
    # a program that keeps a window returns what lies behind it and writes -1 there; long enough for parts
    def chunk():
        return Chunk(BF16, BF16, [(2500, 12), (900, 30)], 4, 2, 64, page, seed=18, window=1000, prefix=prefix)

    c = chunk()
    for workspace in (True, False):
        c.check(*c.run(workspace=workspace))
    kept = 40 // page + 1 if prefix else 0
    c.table[0, kept: (2500 - 1000) // page] = -1
    for workspace in (True, False):
        for longest in (None, 10 ** 9):
            c.check(*c.run(workspace=workspace, longest=longest))
