"""Shared decode attention where nothing is shared: the result of attention of each request alone."""
import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import HALF_STEP, ptr, stream
from test_gpu_paged_shared import Shared

pytestmark = pytest.mark.gpu
F16, BF16, FP8 = M.FLOAT16, M.BFLOAT16, M.F8E4M3
LENGTHS = [1, 700, 0, 33, 64, 250]


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (F16, F16), (BF16, FP8)])
@pytest.mark.parametrize("hq, hk, dim, page", [(8, 2, 128, 16), (20, 1, 64, 10), (4, 4, 256, 32)])
@pytest.mark.parametrize("groups, outside", [([], LENGTHS), ([(0, [x]) for x in LENGTHS], []), ([(0, LENGTHS)], []), ([(0, [])] * 3, LENGTHS)])
def test_the_same_as_attention_of_each_alone(dtype, cache, hq, hk, dim, page, groups, outside):
    s = Shared(dtype, cache, groups, hq, hk, dim, page, seed=dim, outside=((), outside))
    assert s.lengths == LENGTHS
    out, lse = s.run()
    want = s.oracle()
    s.check(out, lse, want=want)
    q, table, lengths = s.keep[:3]
    other, other_lse = torch.empty_like(out), torch.empty_like(lse)
    shape = A.Attention(dtype, hq, s.scale)
    need = A.paged_decode_workspace(shape, s.cache.desc, 6, 700)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    A.paged_decode(shape, s.cache.desc, 6, ptr(q), ptr(s.cache.buffers[0]), ptr(s.cache.buffers[1]), ptr(table), table.shape[1] - 1, ptr(lengths), 700,
                   0, ptr(other), ptr(other_lse), ptr(ws), need, table_stride=table.shape[1], stream=stream())
    torch.cuda.synchronize()
    s.check(other, other_lse, want=want)
    assert (out[2] == 0).all() and (other[2] == 0).all()
    # results rounded once each, of weights rounded once each
    apart = (out.double() - other.double()).abs().cpu()
    scores = (want[3] * (dim + 8) * 2.0 ** -23 + 16 * 2.0 ** -21)[..., None]  # as a relative error of every weight
    u = HALF_STEP[dtype]
    assert (apart <= 2 * (u * want[0].abs() * 1.02 + want[2] * (1.02 * u + 4 * scores)) + 2.0 ** -24).all()
    there = torch.arange(6) != 2
    assert ((lse - other_lse).abs().double().cpu()[there] <= (4 * scores[..., 0] + want[1].abs() * 2.0 ** -21)[there]).all()
