"""The example of a served attention layer: pages, rotary positions, prefill and captured decode steps together."""
import importlib.util
import os

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from manifesto_amd.backend import Backend
from paged_util import HALF_STEP, SMALLEST, attention_oracle, check_attention, ptr

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")


def example():
    spec = importlib.util.spec_from_file_location("paged_serving", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def held(layer, request):
    """Keys and values of a request as the cache holds them, f64 on the CPU."""
    n = int(layer.lengths[request])
    t = torch.arange(n)
    pages, rows = layer.table[request].cpu()[t // layer.page_size].long(), t % layer.page_size
    assert len(set(pages.tolist())) == -(-n // layer.page_size)
    return [x.cpu()[pages, :, rows].double() * s for x, s in ((layer.keys, layer.cache.k_scale), (layer.values, layer.cache.v_scale))]


def turned(x, positions, dim):
    """[tokens, heads, dim] in f64, pairs (i, i + dim / 2)."""
    angle = positions.double()[:, None] * 10000.0 ** (-torch.arange(0, dim, 2).double() / dim)
    c, s, a, b = angle.cos()[:, None], angle.sin()[:, None], x[..., : dim // 2], x[..., dim // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("cache_dtype", [M.BFLOAT16, M.F8E4M3])
@pytest.mark.parametrize("window", [0, 20])
def test_prompts_then_captured_steps(cache_dtype, window):
    prompts, steps, dim = [1, 30, 0, 77], 5, 64
    layer = example().PagedAttention(4, 100, q_heads=4, kv_heads=2, head_dim=dim, hidden=96, cache_dtype=cache_dtype, window=window)
    gen = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(sum(prompts), 96, generator=gen, device="cuda").bfloat16()
    out, q = layer.prompts(x, prompts)

    def check(out, q, first, last, request, positions):
        keys, values = held(layer, request)
        want = attention_oracle(q[first:last].double().cpu(), keys, values, positions, dim ** -0.5, window=window)
        check_attention(out[first:last], torch.as_tensor(want[1]), want, M.BFLOAT16, dim)

    starts = layer.starts.tolist()
    for r, n in enumerate(prompts):
        check(out, q, starts[r], starts[r + 1], r, list(range(n)))
    # the cache holds the projection's keys, turned, and its values, to within the products' and the type's rounding
    qkv = (x @ layer.weight).double().cpu()
    u, tiny = HALF_STEP[cache_dtype], SMALLEST[cache_dtype] * layer.cache.k_scale
    for r, n in enumerate(prompts):
        rows = qkv[starts[r]: starts[r + 1]].reshape(n, 8, dim)
        keys, values = held(layer, r)
        want = turned(rows[:, 4:6], torch.arange(n), dim)
        size = torch.cat([torch.hypot(rows[:, 4:6, : dim // 2], rows[:, 4:6, dim // 2:])] * 2, -1)
        assert ((keys - want).abs() <= u * want.abs() * 1.001 + size * 2.0 ** -20 + tiny).all()
        assert ((values - rows[:, 6:]).abs() <= u * rows[:, 6:].abs() + tiny).all()
    # one token more per request, replayed with other work between
    token = torch.randn(4, 96, generator=gen, device="cuda").bfloat16()
    graph, out, q = layer.capture(token)
    for i in range(steps):
        token.copy_(torch.randn(4, 96, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert layer.lengths.tolist() == [n + i + 1 for n in prompts] and layer.status.tolist() == [0] * 4
        for r, n in enumerate(prompts):
            check(out, q, r, r + 1, r, [n + i])
    free = layer.free_pages()
    layer.end(3)
    assert layer.free_pages() == free + -(-(77 + steps) // 16) and layer.lengths.tolist() == [6, 35, 5, 0]
    graph.replay()  # the ended request begins anew, with a page that is free
    torch.cuda.synchronize()
    for r, n in enumerate([7, 36, 6, 1]):
        check(out, q, r, r + 1, r, [n - 1])


def test_prompts_that_find_no_pages_are_refused():
    layer = example().PagedAttention(2, 64, q_heads=2, kv_heads=1, head_dim=64, hidden=32, pages=3)
    with pytest.raises(RuntimeError, match=r"requests \[1\]"):
        layer.prompts(torch.zeros(50, 32, dtype=torch.bfloat16, device="cuda"), [30, 20])
    assert layer.lengths.tolist() == [30, 0]


def test_a_step_over_resident_tensors():
    # caches, queries and results that are the backend's own tensors
    b, p = Backend(0), lambda t: t.dispatch_pointer()  # noqa: E731
    gen = torch.Generator().manual_seed(5)
    n, hq, hk, dim, page, pages = 21, 4, 2, 64, 16, 4

    def up(t, dtype):
        return b.upload(list(t.shape), dtype, t.contiguous().view(torch.uint8).numpy().tobytes())

    x = torch.randn(n, hq + 2 * hk, dim, generator=gen).bfloat16()
    q, k, v = x[:, :hq].contiguous(), x[:, hq: hq + hk].contiguous(), x[:, hq + hk:].contiguous()
    slots = torch.cat([torch.arange(16) + 32, torch.arange(5)])  # pages 2 and 0
    dq, dk, dv = (up(t, M.BFLOAT16) for t in (q, k, v))
    turned_q, out = (up(torch.zeros(n, hq, dim, dtype=torch.bfloat16), M.BFLOAT16) for _ in range(2))
    keys, values = (up(torch.zeros(pages, hk, page, dim, dtype=torch.bfloat16), M.BFLOAT16) for _ in range(2))
    d = [t.cuda() for t in (torch.arange(n, dtype=torch.int32), slots, torch.tensor(A.rotary_frequencies(dim), dtype=torch.float64),
                            torch.tensor([[2, 0]], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32))]
    cache, shape = A.KVCache(M.BFLOAT16, page, hk, dim, pages), A.Attention(M.BFLOAT16, hq, dim ** -0.5)
    for t in (dq, dk, dv, turned_q, out, keys, values):
        t.sync()
    torch.cuda.synchronize()
    A.rotary_append(A.Rotary(M.BFLOAT16, hq, hk, dim), cache, n, p(dq), p(turned_q), p(dk), p(dv), ptr(d[0]), ptr(d[1]), ptr(d[2]), p(keys), p(values))
    A.paged_prefill(shape, cache, 1, n, n, p(turned_q), p(keys), p(values), ptr(d[3]), 2, ptr(d[4]), ptr(d[5]), n, 0, 0, p(out), 0)
    torch.cuda.synchronize()

    def down(t, *shape):
        return torch.frombuffer(bytearray(bytes(b.download(t)[1])), dtype=torch.bfloat16).view(*shape)

    at = torch.tensor([2, 0])[torch.arange(n) // page]
    ks, vs = (down(t, pages, hk, page, dim)[at, :, torch.arange(n) % page] for t in (keys, values))
    assert torch.equal(vs, v)
    want = turned(k.double(), torch.arange(n), dim)
    assert ((ks.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all()
    rows = attention_oracle(down(turned_q, n, hq, dim).double(), ks.double(), vs.double(), list(range(n)), dim ** -0.5)
    check_attention(down(out, n, hq, dim), rows[1], rows, M.BFLOAT16, dim)
    last, one = up(torch.zeros(1, hq, dim, dtype=torch.bfloat16), M.BFLOAT16), turned_q.slice((n - 1) * hq * dim, hq * dim)
    last.sync()
    A.paged_decode(shape, cache, 1, p(one), p(keys), p(values), ptr(d[3]), 2, ptr(d[5]), n, 0, p(last), 0)
    torch.cuda.synchronize()
    check_attention(down(last, 1, hq, dim), rows[1][-1:], [t[-1:] for t in rows], M.BFLOAT16, dim)
