"""Attention of one new token per request over a paged cache, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import TORCH, Cache, attention_oracle, check_attention, ptr, stream

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = M.FLOAT32, M.FLOAT16, M.BFLOAT16, M.F8E4M3
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 200, 515]


class Step:
    """A batch of requests over one cache."""

    def __init__(self, dtype, cache_dtype, lengths, hq, hk, dim, page, order="head", seed=0, q_std=1.0, gap=0, spare=2, **option):
        M.init(0)
        self.dtype, self.lengths, self.hq, self.hk, self.dim = dtype, lengths, hq, hk, dim
        scales = dict(k_scale=0.0625, v_scale=0.5) if cache_dtype == FP8 else {}
        n = len(lengths)
        width = max(1, max(-(-x // page) for x in lengths))
        self.cache = Cache(cache_dtype, page, hk, dim, sum(-(-x // page) for x in lengths) + spare, order, seed, gap=gap, **scales)
        self.table = torch.full((n, width + 1), -7, dtype=torch.int32)
        std = 1 / scales["k_scale"] if scales else 1.0
        self.kv = [self.cache.put(x, self.table[r], std) for r, x in enumerate(lengths)]
        self.q = (torch.randn(n, hq, dim, generator=self.cache.gen) * q_std).to(TORCH[dtype])
        self.option = option
        self.scale = option.pop("scale", dim ** -0.5)
        self.slopes = torch.rand(hq, generator=self.cache.gen) * 0.3 if option.pop("slopes", False) else None
        self.want = None

    def run(self, longest=None, workspace=True, shape=None, out=None, q=None, on=None):
        n, width = len(self.lengths), self.table.shape[1] - 1
        shape = shape or A.Attention(self.dtype, self.hq, self.scale, **self.option)
        longest = max(self.lengths) if longest is None else longest
        d = lambda t: None if t is None else t.cuda()  # noqa: E731
        self.keep = q_, table, lengths, slopes = d(self.q) if q is None else q, d(self.table), d(torch.tensor(self.lengths, dtype=torch.int32)), d(self.slopes)
        out = torch.full((n, self.hq, self.dim), math.nan, dtype=TORCH[self.dtype], device="cuda") if out is None else out
        lse = torch.full((n, self.hq), math.nan, device="cuda")
        need = A.paged_decode_workspace(shape, self.cache.desc, n, longest) if workspace else 0
        ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        A.paged_decode(shape, self.cache.desc, n, ptr(q_), ptr(self.cache.buffers[0]), ptr(self.cache.buffers[1]), ptr(table), width,
                       ptr(lengths), longest, ptr(slopes), ptr(out), ptr(lse), ptr(ws) if need else 0, need, table_stride=width + 1,
                       stream=stream() if on is None else on)
        torch.cuda.synchronize()
        return out, lse

    def oracle(self, masked=()):
        rows = []
        for r, x in enumerate(self.lengths):
            k, v = self.kv[r]
            rows.append(attention_oracle(self.q[r: r + 1].double(), k, v, [x - 1], self.scale, self.option.get("softcap", 0.0),
                                         self.option.get("window", 0), self.slopes))
        return [torch.cat(t) for t in zip(*rows)]

    def check(self, out, lse):
        reach = 0.0 if self.slopes is None else float(self.slopes.max()) * max(self.lengths)
        check_attention(out, lse, self.oracle(), self.dtype, self.dim, self.option.get("softcap", 0.0), reach)


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("hq, hk, dim, page, order", [(4, 1, 128, 16, "head"), (3, 3, 64, 1, "token"), (8, 2, 80, 7, "head"),
                                                      (6, 2, 256, 48, "token"), (20, 1, 96, 100, "head"), (40, 2, 16, 32, "token"),
                                                      (2, 2, 192, 64, "head"), (5, 1, 112, 24, "token"), (4, 4, 48, 256, "head")])
def test_every_length_against_f64(dtype, cache, hq, hk, dim, page, order):
    s = Step(dtype, cache, LENGTHS, hq, hk, dim, page, order, seed=dim + page, q_std=2.0)
    s.check(*s.run())


@pytest.mark.parametrize("dim", [8, 24, 72, 88, 136, 248])
def test_head_dims_that_end_inside_a_product(dim):
    s = Step(F16, F16, [0, 5, 33, 70], 4, 2, dim, 16, seed=dim, gap=3)
    s.check(*s.run())


@pytest.mark.parametrize("option", [dict(window=1), dict(window=16), dict(window=33), dict(window=130), dict(softcap=20.0), dict(slopes=True),
                                    dict(slopes=True, softcap=5.0, window=40), dict(scale=-0.3), dict(scale=0.0), dict(softcap=1e-3)])
@pytest.mark.parametrize("page", [16, 10])
def test_window_cap_and_bias(option, page):
    s = Step(BF16, BF16, LENGTHS, 6, 2, 64, page, seed=5, q_std=3.0, **dict(option))
    s.check(*s.run())


@pytest.mark.parametrize("cache", [F16, FP8])
@pytest.mark.parametrize("lengths", [[2000] * 3, [1500, 1499, 1600, 1501], [1, 3000, 40, 600, 0, 90], [4000], [0] * 70 + [2500], [700] * 65])
def test_requests_alike_and_not(lengths, cache):
    s = Step(F16, cache, lengths, 4, 2, 64, 16, seed=len(lengths))
    s.check(*s.run())


@pytest.mark.parametrize("page", [16, 9])
def test_parts_do_not_change_what_is_computed(page):
    # one request split as far as it goes, with any hint of the lengths, with little workspace and with none
    s = Step(F16, F16, [5000, 0, 129, 3], 8, 2, 64, page, seed=1)
    for longest in (5000, 1, 700, 10 ** 9, 0):
        s.check(*s.run(longest=longest))
    s.check(*s.run(workspace=False))
    first = s.run()
    for _ in range(3):  # the parts are joined in their order
        again = s.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_large_scores_and_equal_scores():
    s = Step(BF16, BF16, [300, 64, 1], 4, 2, 64, 16, seed=2, q_std=40.0)  # weights of one token alone
    s.check(*s.run())
    s = Step(F16, F16, [300, 64, 1], 4, 2, 64, 16, seed=2, scale=0.0)
    out, _ = s.run()
    mean = s.kv[0][1].mean(0).repeat_interleave(2, 0)
    assert (out[0].double().cpu() - mean).abs().max() <= 2.0 ** -10


def test_scores_that_rise_and_fall_by_hundreds():
    # the running reference has to move up, far and often, and an early maximum has to hold
    s = Step(F16, F16, [2048], 2, 1, 64, 16, seed=3, slopes=True)
    s.slopes = torch.tensor([3.0, -3.0])
    out, lse = s.run(workspace=False)
    check_attention(out, lse, s.oracle(), F16, 64, slope_reach=3.0 * 2048)


def test_a_page_outside_the_cache_counts_as_masked():
    s = Step(BF16, BF16, [64, 48], 2, 1, 64, 16, seed=9)
    s.table[0, 1], s.table[1, 0], s.table[1, 1], s.table[1, 2] = 10 ** 6, -1, -2 ** 31, 2 ** 31 - 1
    k, v = s.kv[0]
    keep = torch.cat([torch.arange(16), torch.arange(32, 64)])
    out, lse = s.run()
    want = attention_oracle(s.q[:1].double(), k[keep], v[keep], [10 ** 6], s.scale)
    check_attention(out[:1], lse[:1], want, BF16, 64)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_lengths_that_pass_the_table_or_are_negative():
    s = Step(F16, F16, [64, 20], 2, 1, 64, 16, seed=10)
    want = s.oracle()
    s.lengths = [10 ** 9, -4]
    out, lse = s.run(longest=64)
    check_attention(out[:1], lse[:1], [t[:1] for t in want], F16, 64)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_not_finite_values_that_are_seen_come_through():
    s = Step(BF16, BF16, [40, 40, 40], 2, 1, 64, 16, seed=12)
    for r, (which, value) in enumerate(((1, math.inf), (1, math.nan), (0, math.nan))):
        t = 21
        s.cache.views[which][int(s.table[r, t // 16]), t % 16, 0, 5] = value
    out, lse = s.run()
    others = torch.arange(64) != 5
    assert (out[0, :, 5] == math.inf).all() and torch.isfinite(out[0][:, others]).all()
    assert torch.isnan(out[1, :, 5]).all() and torch.isfinite(out[1][:, others]).all()
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()


def test_strided_queries_and_results():
    s = Step(BF16, BF16, [70, 3, 129], 4, 2, 32, 16, seed=13)
    row = 4 * 32 + 2 * 2 * 32 + 1
    packed = torch.full((3 * row + 1,), math.nan, dtype=torch.bfloat16, device="cuda")
    q = torch.as_strided(packed, (3, 4, 32), (row, 32, 1), 1)
    q.copy_(s.q)
    big = torch.full((4, 3, 50), -5.0, dtype=torch.bfloat16, device="cuda")  # [head, request, dim]
    shape = A.Attention(BF16, 4, s.scale, q_strides=(row, 32), out_strides=(50, 150))
    _, lse = s.run(shape=shape, q=q, out=big)
    s.check(big[:, :, :32].transpose(0, 1), lse)
    assert (big[:, :, 32:] == -5).all()


def test_pages_far_apart():
    # page offsets past 2^32 bytes
    M.init(0)
    dim, page, stride, pages = 64, 16, 1_300_000_000, 3
    k, v = (torch.empty(stride * (pages - 1) + page * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(1)
    ks, vs = (torch.randn(48, 1, dim, generator=gen).bfloat16() for _ in range(2))
    order = [2, 0, 1]
    for t, x in ((k, ks), (v, vs)):
        for j, p in enumerate(order):
            t[p * stride: p * stride + page * dim] = x[16 * j: 16 * j + 16].reshape(-1).cuda()
    q = torch.randn(1, 2, dim, generator=gen).bfloat16()
    desc = A.KVCache(BF16, page, 1, dim, pages, page_stride=stride)
    shape = A.Attention(BF16, 2, 0.125)
    for size in (16, 12):  # pages of whole groups, and the other kind over the same memory
        if size == 12:
            desc = A.KVCache(BF16, 12, 1, dim, pages, page_stride=stride)
            at = torch.tensor([i for i in range(48) if i % 16 < 12])
        else:
            at = torch.arange(48)
        qd, table = q.cuda(), torch.tensor([order], dtype=torch.int32).cuda()
        lengths = torch.tensor([len(at)], dtype=torch.int32).cuda()
        out, lse = torch.empty_like(qd), torch.empty(1, 2, device="cuda")
        A.paged_decode(shape, desc, 1, ptr(qd), ptr(k), ptr(v), ptr(table), 3, ptr(lengths), len(at), 0, ptr(out), ptr(lse), stream=stream())
        want = attention_oracle(q.double(), ks[at].double(), vs[at].double(), [10 ** 6], 0.125)
        check_attention(out, lse, want, BF16, dim)


def test_another_stream_and_a_captured_step():
    s = Step(BF16, BF16, [300, 17, 0, 900], 4, 2, 64, 16, seed=14)
    side = torch.cuda.Stream()
    s.check(*s.run(on=side.cuda_stream))
    shape = A.Attention(BF16, 4, s.scale)
    n, width = 4, s.table.shape[1] - 1
    q, table, lengths = s.q.cuda(), s.table.cuda(), torch.tensor(s.lengths, dtype=torch.int32).cuda()
    out, lse = torch.empty_like(q), torch.empty(n, 4, device="cuda")
    need = A.paged_decode_workspace(shape, s.cache.desc, n, 900)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        A.paged_decode(shape, s.cache.desc, n, ptr(q), ptr(s.cache.buffers[0]), ptr(s.cache.buffers[1]), ptr(table), width, ptr(lengths), 900, 0,
                       ptr(out), ptr(lse), ptr(ws), need, table_stride=width + 1, stream=stream())
    full = list(s.lengths)
    for now in (full, [1, 17, 0, 33], [299, 2, 0, 512]):  # lengths are read on the device at each replay
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        s.lengths = now
        kv, s.kv = s.kv, [(k[:x], v[:x]) for (k, v), x in zip(s.kv, now)]
        s.check(out, lse)
        s.kv = kv


def test_refused_arguments():
    M.init(0)
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = ptr(t)

    def call(cache=None, shape=None, **args):
        base = dict(requests=1, q=p, k_cache=p, v_cache=p, table=p, table_width=4, lengths=p, longest=64, slopes=0, out=p, lse=0)
        A.paged_decode(A.Attention(**{"dtype": BF16, "q_heads": 4, "scale": 1.0, **(shape or {})}),
                       A.KVCache(**{"dtype": BF16, "page_size": 16, "kv_heads": 2, "head_dim": 64, "pages": 4, **(cache or {})}), **{**base, **args})

    for bad, message in ((dict(shape=dict(dtype=F32)), "f16/bf16"), (dict(shape=dict(dtype=F16)), "over a cache"),
                         (dict(cache=dict(dtype=F32)), "f16/bf16"), (dict(shape=dict(q_heads=3)), "evenly"), (dict(shape=dict(q_heads=0)), "evenly"),
                         (dict(shape=dict(scale=math.nan)), "scale"), (dict(shape=dict(softcap=-1.0)), "cap"), (dict(shape=dict(softcap=math.inf)), "cap"),
                         (dict(shape=dict(window=-1)), "window"), (dict(cache=dict(head_dim=60)), "multiple of 8"),
                         (dict(cache=dict(dtype=FP8, head_dim=72)), "multiple of 16"), (dict(cache=dict(head_dim=264)), "256"),
                         (dict(cache=dict(kv_heads=0)), "heads"), (dict(requests=-1), "requests"), (dict(table_stride=3), "table width"),
                         (dict(table_width=-1), "table width"), (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(table=0), "NULL"),
                         (dict(lengths=0), "NULL"), (dict(v_cache=0), "NULL"), (dict(workspace=0, workspace_bytes=64), "workspace"),
                         (dict(workspace=p + 8, workspace_bytes=64), "workspace")):
        with pytest.raises(M.MFHError, match=message):
            call(**bad)
    call(requests=0, q=0)
    with pytest.raises(M.MFHError, match="requests"):
        A.paged_decode_workspace(A.Attention(BF16, 4, 1.0), A.KVCache(BF16, 16, 2, 64, 4), -1, 5)


@pytest.mark.parametrize("workspace", [True, False])  # with a workspace the long request is in parts
@pytest.mark.parametrize("page", [16, 10])
def test_rows_whose_scores_are_all_nan(page, workspace):
    # NaN is not -inf: lse is NaN beside a result of NaN, also where one wave or one part has nothing else
    def step():
        return Step(BF16, BF16, [5000, 1, 33, 200, 0, 3000], 4, 2, 64, page, seed=21)

    def key(s, request, first, last):
        for t in range(first, last):
            s.cache.views[0][int(s.table[request, t // page]), t % page, 1, 3] = math.nan  # of key-value head 1: query heads 2 and 3

    s = step()
    clean, lse_clean = s.run(workspace=workspace)
    s.check(clean, lse_clean)
    s.q[0, 2, 7] = s.q[3, 1, 0] = math.nan  # a head's query in a long and in a short request
    bad = torch.zeros(6, 4, dtype=torch.bool)
    bad[0, 2] = bad[3, 1] = True
    key(s, 1, 0, 1)      # the only key
    key(s, 2, 32, 33)    # the only key of a wave
    key(s, 5, 128, 512)  # a part of the split form
    bad[1, 2:] = bad[2, 2:] = bad[5, 2:] = True
    out, lse = s.run(workspace=workspace)
    assert torch.equal(torch.isnan(lse).cpu(), bad) and torch.equal(torch.isnan(out).all(-1).cpu(), bad)
    assert torch.equal(out[~bad.cuda()], clean[~bad.cuda()]) and torch.equal(lse[~bad.cuda()], lse_clean[~bad.cuda()])


@pytest.mark.parametrize("cap", [60.0, 64.0, 65.0, 1e3, 1e5, 1e7, 1e30, 8e37])
@pytest.mark.parametrize("dtype, cache", [(F16, F16), (BF16, FP8)])
def test_caps_far_above_the_scores_leave_them_as_they_are(cap, dtype, cache):
    # the bounds go by the scores alone, whatever the cap; of a request of one token lse is the score
    s = Step(dtype, cache, [1, 1, 1, 2, 3, 70, 300], 8, 2, 16, 16, seed=31, q_std=6.0, softcap=cap)
    out, lse = s.run()
    check_attention(out, lse, s.oracle(), dtype, 16)


@pytest.mark.parametrize("cap", [65.0, 1e3])
def test_large_caps_still_cap(cap):
    s = Step(F16, F16, [1, 2, 40, 300], 4, 2, 16, 16, seed=32, q_std=60.0, scale=4.0, softcap=cap)
    out, lse = s.run()
    assert s.oracle()[3].max() > cap
    check_attention(out, lse, s.oracle(), F16, 16)


@pytest.mark.parametrize("below", [14.0, 16.5])
@pytest.mark.parametrize("workspace", [True, False])
def test_many_small_weights_beside_a_large_one(below, workspace):
    # one key far above a long context, whose weights are each near the smallest 16-bit number: together they are all of the result
    s = Step(F16, F16, [60000], 2, 1, 64, 16, seed=41, scale=0.125)
    s.q[:] = 0
    s.q[..., 0] = 8.0
    k, v = s.kv[0]
    k[:, 0, 0] = -below + (0.0 if below > 15 else 1.0) * torch.randn(60000, generator=s.cache.gen).half().double().clamp(-4, 4)
    k[:, 0, 0] = k[:, 0, 0].half().double()
    k[5, 0, 0], v[:, 0] = 0.0, (v[:, 0].abs() + 0.5).half().double()
    v[5] = 0.0
    t = torch.arange(60000)
    for view, x in zip(s.cache.views, (k, v)):
        view[s.table[0, t // 16].long().cuda(), (t % 16).cuda()] = x.half().cuda()
    out, lse = s.run(workspace=workspace)
    want = s.oracle()
    # besides every weight's relative rounding, a half step of its type: 2^-25 where the largest weight is 2^7 or more
    tail = 60000 * 2.0 ** -32 * v.abs().max()
    u, got = 2.0 ** -11, out.double().cpu()
    assert ((got - want[0]).abs() <= u * want[0].abs() + want[2] * (u + 2.0 ** -14) + tail).all(), float(((got - want[0]) / want[0]).abs().max())
    assert (lse.double().cpu() - want[1]).abs().max() <= 2.0 ** -15


@pytest.mark.parametrize("workspace", [True, False])
def test_values_near_the_largest_number_stay_finite(workspace):
    # the value of a late key whose score is above all before it: weights are never above 1 there
    s = Step(BF16, BF16, [700], 2, 1, 64, 16, seed=51, scale=0.125)
    s.q[:] = 0
    s.q[..., 0] = 8.0
    k, v = s.kv[0]
    k[:, 0, 0] = 0.0
    k[130, 0, 0], v[130] = 5.0, 2.0 ** 126
    t = torch.arange(700)
    for view, x in zip(s.cache.views, (k, v)):
        view[s.table[0, t // 16].long().cuda(), (t % 16).cuda()] = x.bfloat16().cuda()
    s.check(*s.run(workspace=workspace))
