"""Attention of one new token per request where requests have their first tokens in common, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import TORCH, Cache, attention_oracle, check_attention, ptr, stream

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = M.FLOAT32, M.FLOAT16, M.BFLOAT16, M.F8E4M3


class Shared:
    """Groups of requests over one cache: groups is a list of (shared, [lengths]); `outside` are lengths of requests
    in front of and behind all groups."""

    def __init__(self, dtype, cache_dtype, groups, hq, hk, dim, page, order="head", seed=0, q_std=1.0, gap=0, outside=((), ()), own_entries=-1,
                 **option):
        M.init(0)
        self.dtype, self.hq, self.hk, self.dim, self.page = dtype, hq, hk, dim, page
        scales = dict(k_scale=0.0625, v_scale=0.5) if cache_dtype == FP8 else {}
        std = 1 / scales["k_scale"] if scales else 1.0
        rows = [(0, x, False) for x in outside[0]]
        self.starts = [len(rows)]
        for shared, lengths in groups:
            rows += [(shared, x, True) for x in lengths]
            self.starts.append(len(rows))
        rows += [(0, x, False) for x in outside[1]]
        self.shared = [g[0] for g in groups]
        self.lengths = [x for _, x, _ in rows]
        n, width = len(rows), max(1, max([-(-max(s, x) // page) for s, x, _ in rows], default=1))
        self.cache = Cache(cache_dtype, page, hk, dim, sum(-(-max(s, x) // page) for s, x, _ in rows) + 2, order, seed, gap=gap, **scales)
        self.table = torch.full((n, width + 1), own_entries, dtype=torch.int32)
        self.kv = [None] * n
        for r, (shared, length, grouped) in enumerate(rows):
            if not grouped or r in self.starts[:-1]:  # the first of a group holds what is shared
                lead = self.cache.put(max(shared, length), self.table[r], std)
                self.kv[r] = [x[:length] for x in lead]
                continue
            # its own tokens stand in its own pages; those in front of them in the first page are NaN
            own = self.cache.put(max(length - shared // page * page, 0), self.table[r][shared // page:], std)
            if length > shared and shared % page:
                at = int(self.table[r, shared // page])
                for view in self.cache.views:
                    view[at, : shared % page] = 127 if cache_dtype == FP8 else math.nan
            self.kv[r] = [torch.cat([a[:shared], b[shared % page:]])[:length] for a, b in zip(lead, own)]
        self.q = (torch.randn(n, hq, dim, generator=self.cache.gen) * q_std).to(TORCH[dtype])
        self.option = option
        self.scale = option.pop("scale", dim ** -0.5)
        self.slopes = torch.rand(hq, generator=self.cache.gen) * 0.3 if option.pop("slopes", False) else None

    def run(self, most_shared=None, most_own=None, shape=None, out=None, q=None, on=None):
        n, width = len(self.lengths), self.table.shape[1] - 1
        shape = shape or A.Attention(self.dtype, self.hq, self.scale, **self.option)
        most_shared = max(self.shared, default=0) if most_shared is None else most_shared
        most_own = max(self.lengths) if most_own is None else most_own
        d = lambda t: None if t is None else t.cuda()  # noqa: E731
        i = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
        self.keep = [d(self.q) if q is None else q, d(self.table), i(self.lengths), d(self.slopes), i(self.starts), i(self.shared)]
        out = torch.full((n, self.hq, self.dim), math.nan, dtype=TORCH[self.dtype], device="cuda") if out is None else out
        lse = torch.full((n, self.hq), math.nan, device="cuda")
        need = A.paged_decode_shared_workspace(shape, self.cache.desc, n, len(self.shared), most_shared, most_own)
        ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        q_, table, lengths, slopes, starts, shared = self.keep
        A.paged_decode_shared(shape, self.cache.desc, n, len(self.shared), ptr(q_), ptr(self.cache.buffers[0]), ptr(self.cache.buffers[1]), ptr(table),
                              width, ptr(starts), ptr(shared), most_shared, ptr(lengths), most_own, ptr(slopes), ptr(out), ptr(lse), ptr(ws), need,
                              table_stride=width + 1, stream=stream() if on is None else on)
        torch.cuda.synchronize()
        return out, lse

    def oracle(self):
        rows = []
        for r, x in enumerate(self.lengths):
            k, v = self.kv[r]
            rows.append(attention_oracle(self.q[r: r + 1].double(), k, v, [x - 1], self.scale, self.option.get("softcap", 0.0),
                                         self.option.get("window", 0), self.slopes))
        return [torch.cat(t) for t in zip(*rows)]

    def check(self, out, lse, rows=slice(None), want=None):
        reach = 0.0 if self.slopes is None else float(self.slopes.max()) * max(self.lengths)
        want = self.oracle() if want is None else want
        check_attention(out[rows], lse[rows], [t[rows] for t in want], self.dtype, self.dim, self.option.get("softcap", 0.0), reach)


GROUPS = [(64, [65, 70, 64, 130]), (0, [3, 0]), (100, [101]), (33, [34] * 9), (1, [0, 1, 2, 40]), (515, [600, 515, 516])]


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("hq, hk, dim, page, order", [(4, 1, 128, 16, "head"), (3, 3, 64, 1, "token"), (8, 2, 80, 7, "head"), (6, 2, 256, 48, "token"),
                                                      (20, 1, 96, 100, "head"), (40, 2, 16, 32, "token"), (2, 2, 192, 64, "head"), (16, 2, 256, 10, "head"),
                                                      (5, 1, 112, 24, "token"), (4, 4, 48, 256, "head")])
def test_groups_against_f64(dtype, cache, hq, hk, dim, page, order):
    s = Shared(dtype, cache, GROUPS, hq, hk, dim, page, order, seed=dim + page, q_std=2.0, outside=((5, 0, 90), (33,)))
    s.check(*s.run())


@pytest.mark.parametrize("dim", [8, 24, 72, 88, 136, 248])
def test_head_dims_that_end_inside_a_product(dim):
    s = Shared(F16, F16, [(40, [41, 70, 50, 44, 45]), (10, [9, 11])], 8, 2, dim, 16, seed=dim, gap=3)
    s.check(*s.run())


@pytest.mark.parametrize("option", [dict(window=1), dict(window=16), dict(window=33), dict(window=130), dict(window=10 ** 9), dict(softcap=20.0), dict(slopes=True),
                                    dict(slopes=True, softcap=5.0, window=40), dict(scale=-0.3), dict(scale=0.0), dict(softcap=1e-3), dict(softcap=1e5)])
@pytest.mark.parametrize("page, heads", [(16, (6, 2)), (10, (16, 1))])
def test_window_cap_and_bias(option, page, heads):
    s = Shared(BF16, BF16, GROUPS, *heads, 64, page, seed=5, q_std=3.0, **dict(option))
    s.check(*s.run())


@pytest.mark.parametrize("members", [1, 2, 4, 5, 8, 16, 17, 63])
@pytest.mark.parametrize("dim, cache", [(64, F16), (128, FP8), (256, F16)])
def test_columns_of_every_number(members, dim, cache):
    s = Shared(F16, cache, [(300, [300 + 3 * i for i in range(members)])], 4, 1, dim, 16, seed=members)
    s.check(*s.run())


@pytest.mark.parametrize("groups", [63, 64, 65, 200])
def test_many_groups(groups):
    gen = torch.Generator().manual_seed(groups)
    sizes = torch.randint(0, 4, (groups,), generator=gen).tolist()  # empty ones too
    spec = []
    for n in sizes:
        shared = int(torch.randint(0, 90, (1,), generator=gen))
        spec.append((shared, (shared + torch.randint(-shared, 40, (n,), generator=gen)).tolist()))
    s = Shared(BF16, BF16, spec, 4, 2, 64, 16, seed=groups, outside=((20,), (7, 40)))
    s.check(*s.run())


def test_4096_groups():
    M.init(0)
    s = Shared(BF16, BF16, [(20, [21 + g % 5]) for g in range(4096)], 1, 1, 64, 16, seed=3)
    out, lse = s.run()
    for rows in (slice(0, 3), slice(2040, 2060), slice(4090, 4096)):
        want = [attention_oracle(s.q[r: r + 1].double(), *s.kv[r], [s.lengths[r] - 1], s.scale) for r in range(*rows.indices(4096))]
        check_attention(out[rows], lse[rows], [torch.cat(t) for t in zip(*want)], BF16, 64)


@pytest.mark.parametrize("page", [16, 9])
def test_parts_do_not_change_what_is_computed(page):
    s = Shared(F16, F16, [(3000, [3001, 3500, 2999, 5]), (0, [1500, 0])], 8, 2, 64, page, seed=1)
    want = s.oracle()
    for most_shared, most_own in ((3000, 1500), (1, 1), (0, 0), (-5, -5), (10 ** 9, 10 ** 9), (100, 4000)):
        s.check(*s.run(most_shared, most_own), want=want)
    first = s.run()
    for _ in range(3):  # the parts are joined in their order
        again = s.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_the_same_as_attention_of_each_alone():
    # tables that hold the shared pages in full: mfh_paged_decode gives the same to within the rounding of the results
    s = Shared(BF16, BF16, [(320, [330, 400, 351, 320])], 8, 2, 128, 16, seed=2)
    s.table[1:4, :20] = s.table[0, :20]
    out, lse = s.run()
    d = [t.cuda() for t in (s.q, s.table, torch.tensor(s.lengths, dtype=torch.int32))]
    other, other_lse = torch.empty_like(out), torch.empty_like(lse)
    A.paged_decode(A.Attention(BF16, 8, s.scale), s.cache.desc, 4, ptr(d[0]), ptr(s.cache.buffers[0]), ptr(s.cache.buffers[1]), ptr(d[1]),
                   s.table.shape[1] - 1, ptr(d[2]), 400, 0, ptr(other), ptr(other_lse), table_stride=s.table.shape[1], stream=stream())
    torch.cuda.synchronize()
    s.check(other, other_lse)
    s.check(out, lse)
    assert (lse - other_lse).abs().max() < 1e-4


def test_large_scores_and_scores_that_rise_and_fall():
    s = Shared(BF16, BF16, [(300, [310, 301, 364])], 4, 2, 64, 16, seed=2, q_std=40.0)  # weights of one token alone
    s.check(*s.run())
    s = Shared(F16, F16, [(2048, [2050, 2100])], 2, 1, 64, 16, seed=3, slopes=True)
    s.slopes = torch.tensor([3.0, -3.0])
    s.check(*s.run())


def test_a_page_outside_the_cache_counts_as_masked():
    s = Shared(BF16, BF16, [(48, [64, 50])], 2, 1, 64, 16, seed=9)
    s.table[0, 1], s.table[1, 3] = 10 ** 6, -2 ** 31
    s.table[1, 0] = 10 ** 6  # not read
    out, lse = s.run()
    keep = torch.cat([torch.arange(16), torch.arange(32, 64)])
    for r, k in ((0, keep), (1, keep[:32])):
        want = attention_oracle(s.q[r: r + 1].double(), s.kv[r][0][k], s.kv[r][1][k], [10 ** 6], s.scale)
        check_attention(out[r: r + 1], lse[r: r + 1], want, BF16, 64)


def test_what_cannot_be_is_never_followed():
    # lengths and shared tokens past the table or negative
    s = Shared(F16, F16, [(64, [64, 64]), (16, [30])], 2, 1, 64, 16, seed=10)
    want = s.oracle()
    s.lengths, s.shared = [10 ** 9, -4, 30], [64, -7]
    width = s.table.shape[1] - 1
    assert width == 4
    out, lse = s.run(64, 64)
    s.check(out, lse, slice(0, 1), want)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    s.check(out, lse, slice(2, 3), want)
    s.lengths, s.shared = [64, 64, 30], [10 ** 9, 16]
    s.check(*s.run(64, 64), want=want)
    # starts that fall, or are no requests: whatever comes out, nothing else is touched
    for starts in ([5, -3, 100], [2 ** 31 - 1, -2 ** 31, 0], [0, 3, 1]):
        s.starts = starts
        s.run(64, 64)


@pytest.mark.parametrize("cache", [BF16, FP8])
@pytest.mark.parametrize("page", [16, 10])
def test_not_finite_values_of_which_some_columns_see_none(cache, page):
    # a window ends between the requests' views of a value; the last request is shorter than the shared tokens
    s = Shared(BF16, cache, [(100, [101, 130, 140, 60]), (0, [40])], 2, 1, 64, page, seed=12, window=50)
    want = s.oracle()  # of finite values

    def put(t, which, dim, value):
        view = s.cache.views[which]
        view[int(s.table[0, t // page]), t % page, 0, dim] = 127 if cache == FP8 else value

    value = math.nan if cache == FP8 else math.inf
    put(70, 1, 5, value)    # first of the requests: 51, 80, 90; the fourth ends at 60
    put(20, 1, 6, value)    # first of the fourth: 10
    put(99, 1, 7, math.nan)  # all but the fourth
    out, lse = s.run()
    clean = [d for d in range(64) if d not in (5, 6, 7)]
    got, exact = out.double().cpu(), want[0]
    assert torch.isfinite(got[:, :, clean]).all() and torch.isfinite(lse).all()
    sees = {5: [0], 6: [3], 7: [0, 1, 2]}
    for dim, rows in sees.items():
        for r in range(5):
            if r in rows:
                assert (torch.isnan(got[r, :, dim]) if dim == 7 or cache == FP8 else got[r, :, dim] == math.inf).all(), (dim, r)
            else:
                assert ((got[r, :, dim] - exact[r, :, dim]).abs() < 0.05).all(), (dim, r)
    put(70, 0, 3, math.nan)  # a key: the first request's row is NaN, the others' stay
    out, lse = s.run()
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.isfinite(lse[1:]).all()
    assert torch.isfinite(out[1:][:, :, clean]).all()


def test_strided_queries_and_results():
    s = Shared(BF16, BF16, [(70, [70, 3, 129])], 4, 2, 32, 16, seed=13)
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
    q = torch.randn(2, 2, dim, generator=gen).bfloat16()
    shape = A.Attention(BF16, 2, 0.125)
    for size in (16, 12):  # pages of whole groups, and the other kind over the same memory
        desc = A.KVCache(BF16, size, 1, dim, pages, page_stride=stride)
        at = torch.tensor([i for i in range(48) if i % 16 < size])
        n = len(at)
        qd, table = q.cuda(), torch.tensor([order, order], dtype=torch.int32).cuda()
        i = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 2], [size + 5], [n, size + 9])]
        out, lse = torch.empty_like(qd), torch.empty(2, 2, device="cuda")
        ws = torch.empty(A.paged_decode_shared_workspace(shape, desc, 2, 1, n, n), dtype=torch.uint8, device="cuda")
        A.paged_decode_shared(shape, desc, 2, 1, ptr(qd), ptr(k), ptr(v), ptr(table), 3, ptr(i[0]), ptr(i[1]), n, ptr(i[2]), n, 0, ptr(out), ptr(lse),
                              ptr(ws), ws.numel(), stream=stream())
        for r, length in ((0, n), (1, size + 9)):
            want = attention_oracle(q[r: r + 1].double(), ks[at][:length].double(), vs[at][:length].double(), [10 ** 6], 0.125)
            check_attention(out[r: r + 1], lse[r: r + 1], want, BF16, dim)


def test_another_stream_and_a_captured_step():
    s = Shared(BF16, BF16, [(300, [301, 340, 300, 900]), (17, [18, 40])], 4, 2, 64, 16, seed=14)
    side = torch.cuda.Stream()
    s.check(*s.run(on=side.cuda_stream))
    # two graphs of one workspace, replayed in turn with the program's own work between
    q, table, lengths, _, starts, shared = s.keep
    shape = A.Attention(BF16, 4, s.scale)
    out, lse = torch.empty(6, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(6, 4, device="cuda")
    need = A.paged_decode_shared_workspace(shape, s.cache.desc, 6, 2, 300, 600)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            A.paged_decode_shared(shape, s.cache.desc, 6, 2, ptr(q), ptr(s.cache.buffers[0]), ptr(s.cache.buffers[1]), ptr(table),
                                  s.table.shape[1] - 1, ptr(starts), ptr(shared), 300, ptr(lengths), 600, 0, ptr(out), ptr(lse), ptr(ws), need,
                                  table_stride=s.table.shape[1], stream=side.cuda_stream)
    for i in range(6):
        s.q = torch.randn(6, 4, 64, generator=s.cache.gen).bfloat16()
        q.copy_(s.q)
        changed = [max(0, x - 7 * i) for x in (301, 340, 300, 900, 18, 40)]
        s.lengths = changed
        lengths.copy_(torch.tensor(changed, dtype=torch.int32))
        kept = [tuple(x[:n] for x in kv) for kv, n in zip(s.kv, changed)]
        ws.fill_(255)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        whole, s.kv = s.kv, kept
        s.check(out, lse)
        s.kv = whole


# Of 256 columns of a group on, and long shared tokens (of which only the bound is long here), prefill's kernels compute them.
MANY = [(200, [201, 330, 200, 0, 260]), (64, [65, 64, 130, 20]), (1, [2] * 6), (0, [7, 0, 1, 40]), (257, [300, 258, 259, 9])]


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("hq, hk, dim, page, order", [(64, 1, 64, 16, "head"), (130, 2, 128, 7, "token"), (64, 1, 80, 100, "head"), (64, 1, 256, 48, "token"),
                                                      (192, 2, 192, 1, "token")])
def test_many_columns_against_f64(dtype, cache, hq, hk, dim, page, order):
    s = Shared(dtype, cache, MANY, hq, hk, dim, page, order, seed=dim + page, q_std=2.0, outside=((5, 0), (33,)))
    out, lse = s.run(most_shared=1 << 24)
    s.check(out, lse)
    first = s.run(most_shared=1 << 24)
    assert torch.equal(first[0], out) and torch.equal(first[1], lse)


@pytest.mark.parametrize("option", [dict(window=1), dict(window=33), dict(window=130), dict(window=10 ** 9), dict(softcap=20.0), dict(slopes=True),
                                    dict(slopes=True, softcap=5.0, window=90), dict(scale=-0.3), dict(scale=0.0), dict(softcap=1e5)])
@pytest.mark.parametrize("page, dim", [(16, 64), (10, 128)])
def test_many_columns_with_window_cap_and_bias(option, page, dim):
    s = Shared(BF16, BF16, MANY, 64, 1, dim, page, seed=5, q_std=3.0, **dict(option))
    s.check(*s.run(most_shared=1 << 24))


def test_many_columns_over_several_parts():
    s = Shared(BF16, BF16, [(3000, [3001, 3100, 2990, 3000, 3600])], 64, 1, 64, 16, seed=6)
    s.check(*s.run(most_shared=1 << 16))
    s.table[0, 100] = -1  # a page of the shared tokens is none of the cache's
    out, lse = s.run(most_shared=1 << 16)
    keep = torch.cat([torch.arange(1600), torch.arange(1616, 3000)])
    for r in (0, 2):
        k = torch.cat([keep, torch.arange(3000, s.lengths[r])]) if s.lengths[r] > 3000 else keep[: s.lengths[r] - 16]
        want = attention_oracle(s.q[r: r + 1].double(), s.kv[r][0][k], s.kv[r][1][k], [10 ** 6], s.scale)
        check_attention(out[r: r + 1], lse[r: r + 1], want, BF16, 64)


@pytest.mark.parametrize("cache", [BF16, FP8])
def test_many_columns_and_values_that_are_not_finite(cache):
    s = Shared(BF16, cache, [(100, [101, 130, 140, 60])], 64, 1, 64, 16, seed=12, window=50)
    want = s.oracle()
    value = math.nan if cache == FP8 else math.inf
    for t, dim, what in ((70, 5, value), (20, 6, value), (99, 7, math.nan)):
        s.cache.views[1][int(s.table[0, t // 16]), t % 16, 0, dim] = 127 if cache == FP8 else what
    out, lse = s.run(most_shared=1 << 24)
    got, exact = out.double().cpu(), want[0]
    assert torch.isfinite(got[:, :, 8:]).all() and torch.isfinite(lse).all()
    for dim, rows in {5: [0], 6: [3], 7: [0, 1, 2]}.items():
        for r in range(4):
            if r in rows:
                assert (torch.isnan(got[r, :, dim]) if dim == 7 or cache == FP8 else got[r, :, dim] == math.inf).all(), (dim, r)
            else:
                assert ((got[r, :, dim] - exact[r, :, dim]).abs() < 0.05).all(), (dim, r)


def test_many_requests_with_few_tokens_of_their_own():
    # four rows a CU and more: a wave a row
    lengths = [(40, [40 + (7 * g + i) % 50 for i in range(4)]) for g in range(70)]
    s = Shared(F16, F16, lengths, 16, 8, 64, 16, seed=21, outside=((3,), ()))
    s.check(*s.run())


def test_no_requests_and_no_groups():
    s = Shared(F16, F16, [], 4, 2, 64, 16, seed=4, outside=((30, 0, 77), ()))
    s.check(*s.run())
    shape = A.Attention(F16, 4, 1.0)
    A.paged_decode_shared(shape, s.cache.desc, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def test_refused_arguments():
    M.init(0)
    t = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    p = ptr(t)

    def call(cache=None, shape=None, **args):
        base = dict(requests=2, groups=1, q=p, k_cache=p, v_cache=p, table=p, table_width=4, starts=p, shared=p, most_shared=64, lengths=p, most_own=64,
                    slopes=0, out=p, lse=0, workspace=p, workspace_bytes=1 << 20)
        A.paged_decode_shared(A.Attention(**{"dtype": BF16, "q_heads": 4, "scale": 1.0, **(shape or {})}),
                              A.KVCache(**{"dtype": BF16, "page_size": 16, "kv_heads": 2, "head_dim": 64, "pages": 4, **(cache or {})}), **{**base, **args})

    for bad, message in ((dict(shape=dict(dtype=F32)), "f16/bf16"), (dict(shape=dict(dtype=F16)), "over a cache"), (dict(cache=dict(dtype=F32)), "f16/bf16"),
                         (dict(shape=dict(q_heads=3)), "evenly"), (dict(shape=dict(scale=math.nan)), "scale"), (dict(shape=dict(softcap=-1.0)), "cap"),
                         (dict(shape=dict(window=-1)), "window"), (dict(cache=dict(head_dim=264)), "256"), (dict(requests=-1), "requests"),
                         (dict(groups=-1), "groups"), (dict(groups=4097), "groups"), (dict(requests=2 ** 31 - 1), "too many"), (dict(table_stride=3), "table width"),
                         (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(table=0), "NULL"), (dict(starts=0), "NULL"), (dict(shared=0), "NULL"),
                         (dict(lengths=0), "NULL"), (dict(v_cache=0), "NULL"), (dict(workspace=0), "workspace"), (dict(workspace=p + 8), "workspace"),
                         (dict(workspace_bytes=64), "workspace")):
        with pytest.raises(M.MFHError, match=message):
            call(**bad)
