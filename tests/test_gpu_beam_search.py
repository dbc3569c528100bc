"""The example of a beam search: forks, copies, shared attention, selection and captured steps together."""
import importlib.util
import os

import pytest
import torch

import manifesto_amd as M
from paged_util import HALF_STEP, SMALLEST, attention_oracle, check_attention

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "beam_search.py")


def example():
    spec = importlib.util.spec_from_file_location("beam_search", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def held(search, row, length):
    """Keys and values of a row as the cache holds them, f64 on the CPU."""
    t = torch.arange(length)
    pages, rows = search.table[row].cpu()[t // search.page_size].long(), t % search.page_size
    return [x.cpu()[pages, :, rows].double() * s for x, s in ((search.keys, search.cache.k_scale), (search.values, search.cache.v_scale))]


def check_cache(search):
    """Every beam's keys and values are those of its history's tokens, whoever computed and copied them."""
    dim, heads = search.head_dim, search.kv_heads
    u, tiny = HALF_STEP[search.cache.dtype], SMALLEST[search.cache.dtype] * search.cache.k_scale
    lengths, known = search.lengths.tolist(), search.known.tolist()
    for row, length in enumerate(lengths):
        if length == 0:
            continue
        assert length == known[row // search.beams] - 1  # the last token is not computed yet
        text = search.history[row, :length].long()
        qkv = (search.embedding[text] @ search.weight).double().cpu().reshape(length, -1, dim)[:, -2 * heads:]
        k, v = qkv[:, :heads], qkv[:, heads:]
        angle = torch.arange(length).double()[:, None] * 10000.0 ** (-torch.arange(0, dim, 2).double() / dim)
        c, s, a, b = angle.cos()[:, None], angle.sin()[:, None], k[..., : dim // 2], k[..., dim // 2:]
        want = torch.cat([a * c - b * s, b * c + a * s], -1)
        size = torch.cat([torch.hypot(a, b)] * 2, -1)
        keys, values = held(search, row, length)
        # the projection's library product may sum in another order for another number of rows: half a step of bf16 twice
        assert ((keys - want).abs() <= u * want.abs() * 1.001 + size * (2.0 ** -7 + 2.0 ** -20) + tiny).all(), row
        assert ((values - v).abs() <= u * v.abs() + v.abs() * 2.0 ** -7 + 2.0 ** -8 * 2.0 ** -7 + tiny).all(), row


def check_pages(search):
    page, pages = search.page_size, search.ring.numel()
    holders = torch.zeros(pages, dtype=torch.int64)
    table = search.table.cpu()
    for row, length in enumerate(search.lengths.tolist()):
        holders[table[row, : -(-length // page)].long()] += 1
    for row, length in enumerate(search.lengths.tolist()):
        assert length % page == 0 or holders[int(table[row, length // page])] == 1  # it grows
    head, tail = search.ring_state.tolist()
    free = search.ring.cpu()[torch.arange(head, tail) % pages].long()
    assert torch.equal((holders - 1).clamp_min(0), search.shares.cpu().long())
    assert sorted(torch.cat([free, holders.nonzero().flatten()]).tolist()) == list(range(pages))


@pytest.mark.parametrize("cache_dtype", [M.BFLOAT16, M.F8E4M3])
@pytest.mark.parametrize("beams, prompts, end", [(3, [5, 40, 16], -1), (8, [100, 33], 7), (1, [20], -1)])
def test_a_search(cache_dtype, beams, prompts, end):
    dim, vocab = 64, 500
    search = example().BeamSearch(len(prompts), beams, 130, vocab=vocab, end_token=end, q_heads=4, kv_heads=2, head_dim=dim, hidden=96,
                                  cache_dtype=cache_dtype)
    gen = torch.Generator().manual_seed(beams)
    search.begin([torch.randint(8, vocab, (n,), generator=gen).tolist() for n in prompts])
    torch.cuda.synchronize()
    assert search.status.tolist() == [0] * search.requests and search.lengths.tolist() == [n for n in prompts for _ in range(beams)]
    check_cache(search)
    check_pages(search)
    graph, out, q = search.capture_search()
    for step in range(20):
        before = search.history.cpu(), search.scores.cpu(), search.known.tolist(), search.ended.cpu()
        graph.replay()
        torch.cuda.synchronize()
        assert search.status.tolist() == [0] * search.requests
        parents, tokens = search.parents.cpu().long(), search.tokens.cpu()
        for row in range(search.requests):
            g = row // beams
            assert int(parents[row]) // beams == g
            n = before[2][g]
            assert torch.equal(search.history[row, :n].cpu(), before[0][parents[row], :n]) and int(search.history[row, n]) == int(tokens[row])
            assert float(search.scores[row]) <= float(before[1][parents[row]]) and (row % beams == 0 or search.scores[row] <= search.scores[row - 1])
            if end >= 0 and before[3][parents[row]]:
                assert int(tokens[row]) == end and float(search.scores[row]) == float(before[1][parents[row]])
        if step in (0, 7, 19):
            check_cache(search)
            check_pages(search)
    # the last step's attention, of the beams as they were before its selection: those whose parents are themselves
    stay = [r for r in range(search.requests) if int(search.parents[r]) == r]
    for row in stay:
        length = int(search.lengths[row])
        keys, values = held(search, row, length)
        want = attention_oracle(q[row: row + 1].double().cpu(), keys, values, [length - 1], dim ** -0.5)
        check_attention(out[row: row + 1], torch.as_tensor(want[1]), want, M.BFLOAT16, dim)
    search.fork(torch.full((search.requests,), -1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert search.free_pages() == search.ring.numel() and int(search.shares.abs().sum()) == 0
