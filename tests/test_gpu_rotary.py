"""Rotary positions and the cache's writes against f64 forms."""
import math

import numpy as np
import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import HALF_STEP, SMALLEST, TORCH, Cache, ptr, stream

gpu = pytest.mark.gpu
F32, F16, BF16, FP8 = M.FLOAT32, M.FLOAT16, M.BFLOAT16, M.F8E4M3


def turned(x, positions, freqs, rot, interleaved, inverse=False, factor=1.0):
    """x [tokens, heads, dim] f64; also the size that the error bound goes by."""
    x = x.clone()
    angle = positions.double()[:, None] * torch.as_tensor(freqs, dtype=torch.float64)
    c, s = (angle.cos() * factor)[:, None], (angle.sin() * (-factor if inverse else factor))[:, None]
    i = torch.arange(rot // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(x)
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(factor)
    return x, size


def near(got, want, size, dtype):
    # the result's rounding; products, their sum and the factor's in f32; a phase within 2^-24 of a turn
    bound = HALF_STEP[dtype] * want.abs() * 1.001 + size * (4 * 2.0 ** -24 + 2 * math.pi * 2.0 ** -24) + SMALLEST[dtype]
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim, rot", [(128, 128), (128, 64), (96, 96), (80, 40), (64, 0), (2, 2), (10, 6), (256, 256), (72, 18), (500, 500)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 37])
def test_turns_match_the_definition(dtype, dim, rot, interleaved, tokens):
    M.init(0)
    gen = torch.Generator().manual_seed(dim * 7 + rot + tokens)
    hq, hk = 5, 2
    q, k = (torch.randn(tokens, h, dim, generator=gen).to(TORCH[dtype]) for h in (hq, hk))
    positions = torch.randint(-3, 1 << 20, (tokens,), generator=gen, dtype=torch.int32)
    positions[0] = 2 ** 24 + 1
    freqs = A.rotary_frequencies(rot)
    f = torch.tensor(freqs + [0.0], dtype=torch.float64).cuda()
    qd, kd, pd = q.cuda(), k.cuda(), positions.cuda()
    for inverse in (False, True):
        shape = A.Rotary(dtype, hq, hk, dim, rot, interleaved=interleaved, inverse=inverse, factor=1.25)
        qo, ko = torch.full_like(qd, math.nan), torch.full_like(kd, math.nan)
        A.rotary(shape, tokens, ptr(qd), ptr(qo), ptr(kd), ptr(ko), ptr(pd), ptr(f), stream=stream())
        for got, x in ((qo, q), (ko, k)):
            near(got, *turned(x.double(), positions, freqs, rot, interleaved, inverse, 1.25), dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_in_place_and_strided_slices_of_a_fused_projection(dtype):
    M.init(0)
    gen = torch.Generator().manual_seed(4)
    n, hq, hk, dim, rot = 19, 6, 2, 64, 32
    row = (hq + 2 * hk) * dim + 3  # rows that start anywhere
    qkv = torch.randn(n * row + 1, generator=gen).to(TORCH[dtype]).cuda()
    before = qkv.clone()
    q = torch.as_strided(qkv, (n, hq, dim), (row, dim, 1), 1)
    k = torch.as_strided(qkv, (n, hk, dim), (row, dim, 1), 1 + hq * dim)
    want = [turned(x.double().cpu(), torch.arange(n) * 91, A.rotary_frequencies(rot), rot, False) for x in (q, k)]
    f, p = torch.tensor(A.rotary_frequencies(rot), dtype=torch.float64).cuda(), (torch.arange(n, dtype=torch.int32) * 91).cuda()
    strides = (row, dim)
    shape = A.Rotary(dtype, hq, hk, dim, rot, q_strides=strides, q_out_strides=strides, k_strides=strides, k_out_strides=strides)
    A.rotary(shape, n, ptr(q), ptr(q), ptr(k), ptr(k), ptr(p), ptr(f), stream=stream())
    near(q, *want[0], dtype)
    near(k, *want[1], dtype)
    touched = torch.zeros_like(qkv, dtype=torch.bool)
    for h, off in ((hq, 1), (hk, 1 + hq * dim)):
        torch.as_strided(touched, (n, h, dim), (row, dim, 1), off)[:] = True
    assert torch.equal(qkv[~touched], before[~touched])
    # one of the two alone
    alone = torch.empty_like(k.contiguous())
    A.rotary(A.Rotary(dtype, hq, hk, dim, rot), n, 0, 0, ptr(k.contiguous()), ptr(alone), ptr(p), ptr(f), stream=stream())
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype, hq, hk, dim, rot", [(BF16, 40, 9, 256, 192), (F32, 33, 1, 96, 96), (F16, 71, 8, 34, 10)])
def test_more_heads_than_a_workgroup_turns_at_once(dtype, hq, hk, dim, rot, interleaved):
    M.init(0)
    gen = torch.Generator().manual_seed(hq)
    q, k = (torch.randn(3, h, dim, generator=gen).to(TORCH[dtype]) for h in (hq, hk))
    positions, freqs = torch.tensor([0, 77, 40000], dtype=torch.int32), A.rotary_frequencies(rot)
    qd, kd, pd, f = q.cuda(), k.cuda(), positions.cuda(), torch.tensor(freqs, dtype=torch.float64).cuda()
    A.rotary(A.Rotary(dtype, hq, hk, dim, rot, interleaved=interleaved), 3, ptr(qd), ptr(qd), ptr(kd), ptr(kd), ptr(pd), ptr(f), stream=stream())
    for got, x in ((qd, q), (kd, k)):
        near(got, *turned(x.double(), positions, freqs, rot, interleaved), dtype)


@gpu
def test_the_inverse_is_the_gradient():
    # <g, d turn(x) / dx> by differences of the turn itself (it is linear: exact but for rounding), and turn(inverse(x)) = x
    M.init(0)
    gen = torch.Generator().manual_seed(6)
    n, h, dim = 9, 3, 24
    x, g, e = (torch.randn(n, h, dim, generator=gen) for _ in range(3))
    p, f = torch.randint(0, 5000, (n,), generator=gen, dtype=torch.int32).cuda(), torch.tensor(A.rotary_frequencies(16), dtype=torch.float64).cuda()

    def turn(t, inverse):
        d = t.float().cuda()
        out = torch.empty_like(d)
        A.rotary(A.Rotary(F32, h, 0, dim, 16, interleaved=True, inverse=inverse, factor=0.75), n, ptr(d), ptr(out), 0, 0, ptr(p), ptr(f), stream=stream())
        return out.double().cpu()

    slope = ((turn(x + e, False) - turn(x - e, False)) / 2 * g.double()).sum()
    through = (turn(g, True) * e.double()).sum()
    size = (g.abs().double() * (x.abs() + e.abs())).sum() * 2
    assert abs(float(slope - through)) <= float(size) * 16 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("dtype, cache_dtype", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("page, dim, rot, order", [(16, 128, 128, "head"), (1, 64, 32, "token"), (7, 80, 40, "head"), (100, 48, 24, "token"), (32, 256, 256, "head")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_writes_its_slots_and_nothing_else(dtype, cache_dtype, page, dim, rot, order, interleaved):
    M.init(0)
    n, hq, hk, pages = 45, 4, 3, 90 // page + 2
    ks, vs = (0.5, 0.03) if cache_dtype == FP8 else (1.0, 1.0)
    cache = Cache(cache_dtype, page, hk, dim, pages, order, k_scale=ks, v_scale=vs, gap=16)
    gen = torch.Generator().manual_seed(page + dim)
    q, k, v = (torch.randn(n, h, dim, generator=gen).to(TORCH[dtype]) for h in (hq, hk, hk))
    v[0, 0, 0], v[1, 0, 0], v[2, 0, 0] = 60000.0, -60000.0, math.nan  # past the largest code
    positions = torch.randint(0, 9999, (n,), generator=gen, dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=gen)[:n].clone()
    slots[5], slots[6], slots[7] = -1, pages * page, 2 ** 40
    freqs = A.rotary_frequencies(rot)
    d = [t.cuda() for t in (q, k, v, positions, slots, torch.tensor(freqs, dtype=torch.float64))]
    qo = torch.empty_like(d[0])
    old = [b.view(torch.uint8).clone() for b in cache.buffers]
    A.rotary_append(A.Rotary(dtype, hq, hk, dim, rot, interleaved=interleaved), cache.desc, n, ptr(d[0]), ptr(qo), ptr(d[1]), ptr(d[2]),
                    ptr(d[3]), ptr(d[4]), ptr(d[5]), ptr(cache.buffers[0]), ptr(cache.buffers[1]), stream=stream())
    near(qo, *turned(q.double(), positions, freqs, rot, interleaved), dtype)
    keep = [i for i in range(n) if 0 <= int(slots[i]) < pages * page]
    at = slots[keep]
    kw, size = turned(k.double(), positions, freqs, rot, interleaved)
    vw = v.double()
    for view, want, s, scale in ((cache.views[0], kw, size, ks), (cache.views[1], vw, torch.zeros_like(vw), vs)):
        got = view[(at // page).cuda(), (at % page).cuda()]
        got = got.view(TORCH[cache_dtype]).double().cpu() if cache_dtype == FP8 else got.double().cpu()
        w = want[keep] / scale
        if cache_dtype == FP8:
            w = w.clamp(-448, 448)
        fine = ~torch.isnan(w)
        assert torch.equal(torch.isnan(got), ~fine)
        near(got[fine], w[fine], s[keep][fine] / scale + w[fine].abs() * 2, cache_dtype)
    # everything else is as it was
    for buf, was, view in zip(cache.buffers, old, cache.views):
        mine = torch.zeros_like(was).view(torch.uint8)
        mask = torch.zeros(buf.numel(), dtype=torch.uint8, device="cuda")
        torch.as_strided(mask, view.shape, view.stride())[(at // page).cuda(), (at % page).cuda()] = 1
        size = buf.element_size()
        untouched = (mask == 0).repeat_interleave(size)
        assert torch.equal(buf.view(torch.uint8)[untouched], was[untouched])
        del mine


@gpu
def test_eight_bit_codes_are_the_nearest_ones_ties_to_even():
    # every f16 value, as the value of one element: against torch's conversion
    M.init(0)
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    n, dim = 4096, 16
    v = x.view(n, 1, dim).cuda()
    k = torch.zeros_like(v)
    cache = Cache(FP8, 64, 1, dim, 64)
    slots, positions = torch.arange(n).cuda(), torch.zeros(n, dtype=torch.int32).cuda()
    A.rotary_append(A.Rotary(F16, 0, 1, dim, 0), cache.desc, n, 0, 0, ptr(k), ptr(v), ptr(positions), ptr(slots), 0,
                    ptr(cache.buffers[0]), ptr(cache.buffers[1]), stream=stream())
    got = cache.buffers[1].view(torch.uint8).cpu().view(-1)
    f = x.float()
    want = torch.where(torch.isnan(f), f, f.clamp(-448, 448)).to(torch.float8_e4m3fn)
    nan = torch.isnan(f)
    assert torch.equal(got[~nan], want.view(torch.uint8)[~nan])
    assert ((got[nan] & 0x7F) == 0x7F).all()


def test_frequencies_follow_their_formulas():
    dim, base, factor, length = 64, 10000.0, 8.0, 4096.0
    i = np.arange(dim // 2)
    plain = base ** (-2.0 * i / dim)
    tight = dict(rtol=1e-13, atol=0)
    np.testing.assert_allclose(A.rotary_frequencies(dim, base), plain, **tight)
    np.testing.assert_allclose(A.rotary_frequencies(dim, base, A.ROTARY_LINEAR, factor), plain / factor, **tight)
    grown = np.array(A.rotary_frequencies(dim, base, A.ROTARY_BASE, factor))
    np.testing.assert_allclose(grown, (base * factor ** (dim / (dim - 2))) ** (-2.0 * i / dim), **tight)
    np.testing.assert_allclose([grown[0], grown[-1]], [1.0, plain[-1] / factor], rtol=1e-12)
    bands = np.array(A.rotary_frequencies(dim, base, A.ROTARY_BANDS, factor, length, 1.0, 4.0))
    turns = length * plain / (2 * np.pi)
    share = np.clip((turns - 1.0) / 3.0, 0, 1)
    np.testing.assert_allclose(bands, plain * share + plain / factor * (1 - share), rtol=1e-12)
    assert (share == 1).any() and (share == 0).any() and ((share > 0) & (share < 1)).any()
    assert A.rotary_frequencies(0) == [] and A.rotary_frequencies(2, scaling=A.ROTARY_BASE, factor=2.0) == [1.0]


@pytest.mark.parametrize("args, message", [
    (dict(rotary_dim=3), "even"), (dict(rotary_dim=-2), "even"), (dict(base=0.0), "base"), (dict(base=math.inf), "base"),
    (dict(scaling=9), "scaling"), (dict(scaling=A.ROTARY_LINEAR, factor=0.0), "factor"),
    (dict(scaling=A.ROTARY_BANDS, factor=2.0), "bands"),
    (dict(scaling=A.ROTARY_BANDS, factor=2.0, original_length=8.0, low=4.0, high=4.0), "bands")])
def test_refused_frequencies(args, message):
    with pytest.raises(M.MFHError, match=message):
        A.rotary_frequencies(**{"rotary_dim": 8, **args})


@gpu
def test_refused_arguments():
    M.init(0)
    t = torch.zeros(4096, dtype=torch.float64, device="cuda")
    p = ptr(t)

    def call(tokens=1, q=p, q_out=p, k=p, k_out=p, positions=p, frequencies=p, **shape):
        A.rotary(A.Rotary(**{"dtype": BF16, "q_heads": 2, "kv_heads": 1, "head_dim": 16, **shape}), tokens, q, q_out, k, k_out, positions, frequencies)

    for bad, message in ((dict(dtype=FP8), "f32/bf16/f16"), (dict(head_dim=15), "head dim"), (dict(head_dim=2048), "head dim"),
                         (dict(rotary_dim=18), "rotary dim"), (dict(rotary_dim=3), "rotary dim"), (dict(q_heads=-1), "heads"),
                         (dict(tokens=-1), "tokens"), (dict(positions=0), "NULL"), (dict(frequencies=0), "NULL"),
                         (dict(q_out=0), "without"), (dict(k=0), "without")):
        with pytest.raises(M.MFHError, match=message):
            call(**bad)
    call(tokens=0, positions=0)

    def append(shape=None, cache=None, **args):
        base = dict(tokens=1, q=p, q_out=p, k=p, v=p, positions=p, slots=p, frequencies=p, k_cache=p, v_cache=p)
        A.rotary_append(A.Rotary(**{"dtype": BF16, "q_heads": 2, "kv_heads": 1, "head_dim": 16, **(shape or {})}),
                        A.KVCache(**{"dtype": BF16, "page_size": 4, "kv_heads": 1, "head_dim": 16, "pages": 2, **(cache or {})}), **{**base, **args})

    for bad, message in ((dict(cache=dict(dtype=F32)), "f16/bf16/f8"), (dict(cache=dict(dtype=F16)), "into a cache"),
                         (dict(shape=dict(dtype=F32), cache=dict(dtype=FP8)), "into a cache"), (dict(cache=dict(kv_heads=2)), "match"),
                         (dict(cache=dict(head_dim=8)), "match"), (dict(shape=dict(inverse=True)), "inverse"),
                         (dict(cache=dict(page_size=0)), "page size"), (dict(cache=dict(pages=0)), "pages"),
                         (dict(cache=dict(k_scale=0.5)), "scale"), (dict(cache=dict(dtype=FP8, v_scale=0.0)), "scale"),
                         (dict(cache=dict(dtype=FP8, k_scale=math.nan)), "scale"), (dict(cache=dict(token_stride=-16)), "stride"),
                         (dict(cache=dict(token_stride=1 << 30)), "2 GiB"), (dict(cache=dict(page_stride=1 << 62)), "span"),
                         (dict(slots=0), "NULL"), (dict(v=0), "NULL"), (dict(k_cache=0), "NULL"), (dict(q=0), "without")):
        with pytest.raises(M.MFHError, match=message):
            append(**bad)


@gpu
def test_more_tokens_than_one_launch_dimension_holds():
    # a token a workgroup, 2^24 and more of them: against the same tokens in two calls
    M.init(0)
    n, dim, half = 2 ** 24 + 300, 258, 2 ** 23 + 7
    if torch.cuda.mem_get_info()[0] < 4 * n * dim * 2:
        pytest.skip("needs 35 GB of device memory")
    x = torch.randint(0, 1 << 14, (n, dim), dtype=torch.int16, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).view(torch.bfloat16)
    p = (torch.arange(n, device="cuda") % 100003).to(torch.int32)
    f = torch.tensor(A.rotary_frequencies(dim), dtype=torch.float64).cuda()
    shape = A.Rotary(BF16, 1, 0, dim)
    whole, parts = (torch.zeros_like(x) for _ in range(2))
    A.rotary(shape, n, ptr(x), ptr(whole), 0, 0, ptr(p), ptr(f), stream=stream())
    for first, last in ((0, half), (half, n)):
        A.rotary(shape, last - first, ptr(x[first:]), ptr(parts[first:]), 0, 0, ptr(p[first:]), ptr(f), stream=stream())
    assert torch.equal(whole.view(torch.int16), parts.view(torch.int16))
    near(whole[-50:, None], *turned(x[-50:, None].double().cpu(), p[-50:].cpu(), A.rotary_frequencies(dim), dim, False), BF16)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_keys_or_queries_alone(dtype):
    M.init(0)
    gen = torch.Generator().manual_seed(8)
    n, dim, rot = 19, 64, 32
    positions, freqs = torch.arange(n, dtype=torch.int32) * 91, A.rotary_frequencies(rot)
    p, f = positions.cuda(), torch.tensor(freqs, dtype=torch.float64).cuda()
    for hq, hk in ((6, 2), (0, 3), (5, 0)):
        for of_q in (False, True):
            x = torch.randn(n, hq if of_q else hk, dim, generator=gen).to(TORCH[dtype])
            d = x.cuda()
            alone = torch.full_like(d, math.nan)
            mine = (ptr(d), ptr(alone))
            A.rotary(A.Rotary(dtype, hq, hk, dim, rot), n, *(mine if of_q else (0, 0)), *((0, 0) if of_q else mine), ptr(p), ptr(f), stream=stream())
            near(alone, *turned(x.double(), positions, freqs, rot, False), dtype)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_turning_back_gives_what_was_turned(interleaved):
    M.init(0)
    n, h, dim, rot = 40, 3, 48, 32
    x = torch.randn(n, h, dim, generator=torch.Generator().manual_seed(9))
    d, f = x.cuda(), torch.tensor(A.rotary_frequencies(rot), dtype=torch.float64).cuda()
    there, back = torch.empty_like(d), torch.empty_like(d)
    p = (torch.arange(n, dtype=torch.int32) * 40009).cuda()
    for inverse, a, b in ((False, d, there), (True, there, back)):
        A.rotary(A.Rotary(F32, h, 0, dim, rot, interleaved=interleaved, inverse=inverse), n, ptr(a), ptr(b), 0, 0, ptr(p), ptr(f), stream=stream())
    # both turns have the same cosines and sines: c^2 + s^2 is 1 to within their errors of 2^-24 of a phase and of a value, and
    # each turn rounds two products and a sum
    size = torch.zeros_like(x)
    i = torch.arange(rot // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    size[..., first] = size[..., second] = x[..., first].abs() + x[..., second].abs()
    off = (back.cpu() - x).abs()
    assert (off <= size * 12 * 2.0 ** -24).all() and torch.equal(back.cpu()[..., rot:], x[..., rot:])
    assert not torch.equal(there.cpu()[..., :rot], x[..., :rot])
