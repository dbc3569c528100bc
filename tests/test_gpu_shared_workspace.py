"""One workspace for calls of every size: what is enough for a call is enough for all smaller ones."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import ptr, stream
from test_gpu_paged_shared import Shared

pytestmark = pytest.mark.gpu
F16, BF16 = M.FLOAT16, M.BFLOAT16


def need(requests, groups, shared, own, q_heads=16, kv_heads=4, dim=128):
    M.init(0)
    return A.paged_decode_shared_workspace(A.Attention(BF16, q_heads, 1.0), A.KVCache(BF16, 16, kv_heads, dim, 100), requests, groups, shared, own)


@pytest.mark.parametrize("prompts, beams, shared, longest", [(8, 4, 18436, 18500), (4, 4, 64000, 64016), (2, 32, 30000, 30064), (4, 16, 30000, 30064)])
def test_fewer_own_tokens_need_no_more(prompts, beams, shared, longest):
    # with few own tokens the shared ones have the whole card, in twice as many parts
    assert need(prompts * beams, prompts, longest, longest) >= need(prompts * beams, prompts, shared, longest - shared)


def test_fewer_requests_need_no_more():
    sizes = [need(n, 1, 30000, 30, 32, 8) for n in range(1, 300)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("q_heads, kv_heads, dim", [(16, 4, 128), (32, 8, 128), (8, 8, 64), (16, 2, 256), (64, 1, 96), (71, 1, 64), (130, 2, 80)])
def test_smaller_sizes_need_no_more(q_heads, kv_heads, dim):
    gen = torch.Generator().manual_seed(q_heads)

    def up_to(most):
        return min(most, int(math.exp(float(torch.rand((), generator=gen)) * math.log(most + 1))))

    for _ in range(3000):
        large = up_to(2000), up_to(100), up_to(200_000), up_to(20_000)
        small = tuple(up_to(x) for x in large)
        assert need(*small, q_heads, kv_heads, dim) <= need(*large, q_heads, kv_heads, dim), (small, large)
        assert need(large[0], 0, *large[2:], q_heads, kv_heads, dim) <= need(*large, q_heads, kv_heads, dim)


@pytest.mark.parametrize("hq, hk, dim, groups", [(8, 2, 64, [(3000, [3001, 3040, 2999]), (700, [720, 700])]), (4, 4, 256, [(2000, [2001])]),
                                                 (64, 1, 128, [(3000, [3001, 3040, 3003, 3000])]), (32, 2, 64, [])])
def test_calls_of_several_sizes_in_one_workspace(hq, hk, dim, groups):
    # nothing is written behind what the call asks for
    s = Shared(F16, F16, groups, hq, hk, dim, 16, seed=7, outside=((1500, 3), (0,)))
    want = s.oracle()
    n, k, shape = len(s.lengths), len(s.shared), A.Attention(F16, hq, s.scale)
    s.run()
    q, table, lengths, _, starts, shared = s.keep
    room = A.paged_decode_shared_workspace(shape, s.cache.desc, 2 * n, k + 1, 5000, 5000)
    for most_shared, most_own in ((5000, 5000), (3000, 1500), (3000, 40), (1 << 20, 40), (100, 5000), (1, 1)):
        asked = A.paged_decode_shared_workspace(shape, s.cache.desc, n, k, most_shared, most_own)
        assert asked <= room or most_shared > 5000
        ws = torch.full((asked + 4096,), 255, dtype=torch.uint8, device="cuda")
        out, lse = torch.full_like(q, math.nan), torch.full((n, hq), math.nan, device="cuda")
        A.paged_decode_shared(shape, s.cache.desc, n, k, ptr(q), ptr(s.cache.buffers[0]), ptr(s.cache.buffers[1]), ptr(table), s.table.shape[1] - 1,
                              ptr(starts), ptr(shared), most_shared, ptr(lengths), most_own, 0, ptr(out), ptr(lse), ptr(ws), asked,
                              table_stride=s.table.shape[1], stream=stream())
        torch.cuda.synchronize()
        s.check(out, lse, want=want)
        assert (ws[asked:] == 255).all()
