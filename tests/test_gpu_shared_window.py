"""A window over shared tokens: those in front of every request's are not read, whether or not some requests have ended."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import attention_oracle, check_attention, ptr, stream

pytestmark = pytest.mark.gpu
BF16 = M.BFLOAT16


@pytest.mark.parametrize("heads, groups", [(64, 16), (8, 16)])  # prefill's kernels, and 32 columns
def test_ended_requests_do_not_widen_the_window(heads, groups):
    M.init(0)
    gen = torch.Generator().manual_seed(heads)
    tokens, members, window, page, dim = 1 << 17, 4, 64, 16, 64
    n, pages = groups * members, tokens // page + 1
    desc, shape = A.KVCache(BF16, page, 1, dim, pages), A.Attention(BF16, heads, dim ** -0.5, window=window)
    k, v = (torch.randn(pages, page, dim, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(n, heads, dim, generator=gen).bfloat16()
    on_card = [x.cuda() for x in (q, k, v, torch.arange(pages, dtype=torch.int32).repeat(n, 1))]
    starts, shared = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (list(range(0, n + 1, members)), [tokens] * groups))
    out, lse = torch.empty_like(on_card[0]), torch.empty(n, heads, device="cuda")
    ws = torch.empty(A.paged_decode_shared_workspace(shape, desc, n, groups, tokens, page), dtype=torch.uint8, device="cuda")
    going = (tokens + torch.arange(n) % 9).to(torch.int32)
    some = going.clone()
    some[members - 1:: members] = 0
    micros = []
    for lengths in (going, some):
        its = lengths.cuda()

        def call():
            A.paged_decode_shared(shape, desc, n, groups, *(ptr(x) for x in on_card), pages, ptr(starts), ptr(shared), tokens, ptr(its), page, 0,
                                  ptr(out), ptr(lse), ptr(ws), ws.numel(), stream=stream())

        times = []
        for _ in range(8):
            ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            call()
            ends[0].record()
            for _ in range(10):
                call()
            ends[1].record()
            torch.cuda.synchronize()
            times.append(ends[0].elapsed_time(ends[1]) * 100)
        micros.append(min(times))
        for r in range(0, n, 7):
            x = int(lengths[r])
            first = max(0, x - window - 5)
            keys, values = (t.reshape(-1, 1, dim)[first:x].double() for t in (k, v))
            want = attention_oracle(q[r: r + 1].double(), keys, values, [x - 1 - first], dim ** -0.5, window=window)
            check_attention(out[r: r + 1], lse[r: r + 1], want, BF16, dim)
    print(micros)
    # of 131072 tokens 64 are seen: with all of them read a call takes many times as long
    assert micros[1] < 2.5 * micros[0], micros
