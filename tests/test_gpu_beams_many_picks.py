"""Selection of groups with many candidates a pick: what decides is found in the lists of the best heads, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import beams as B
from paged_util import ptr, stream
from test_gpu_beams import rows_of, same, select, select_oracle

pytestmark = pytest.mark.gpu
F32, F16, BF16 = M.FLOAT32, M.FLOAT16, M.BFLOAT16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("groups, beams, picks, vocab", [(3, 31, 62, 68), (1, 17, 64, 1000), (2, 40, 63, 5000), (1, 256, 64, 300), (5, 20, 64, 70), (1, 8, 16, 84690),
                                                         (1, 31, 62, 50000), (2, 63, 17, 3000), (1, 100, 11, 9000), (1, 3, 64, 30000), (1, 256, 5, 20000)])
def test_many_candidates(dtype, groups, beams, picks, vocab):
    gen = torch.Generator().manual_seed(beams + picks)
    x = rows_of(gen, groups * beams, vocab, dtype)
    for spread in (0.0, 1.0, 30.0):  # beams of one score; some far behind the others
        scores = -torch.rand(groups * beams, generator=gen) * spread
        same(select(x, scores, beams, picks, dtype=dtype), select_oracle(x.cpu(), scores, beams, picks))


@pytest.mark.parametrize("beams, picks, vocab", [(32, 64, 40000), (40, 33, 500)])
def test_ended_masked_and_spoilt_beams(beams, picks, vocab):
    gen = torch.Generator().manual_seed(beams)
    x = rows_of(gen, 2 * beams, vocab, BF16)
    x[::5, vocab // 2:] = -math.inf
    x[1::7] = -math.inf
    x[3::7, 7] = math.nan
    scores = -torch.rand(2 * beams, generator=gen) * 6
    ended = (torch.rand(2 * beams, generator=gen) < 0.5).to(torch.uint8)
    want_x = x.cpu()
    want_x[3::7] = -math.inf  # a beam with NaN has no continuation
    for end_token in (0, vocab - 1):
        args = dict(ended=ended, end_token=end_token)
        same(select(x, scores, beams, picks, dtype=BF16, **args), select_oracle(want_x, scores, beams, picks, **args))


@pytest.mark.parametrize("step", [0.0, 0.125, 4.0])
def test_candidates_of_every_rank_and_equal_ones(step):
    # entry i of beam b is worth -(i + b step): many equal scores, and every pick a rank of its own
    beams, vocab = 64, 1500
    t = torch.randperm(vocab, generator=torch.Generator().manual_seed(1)).float()
    x = (-t * 0.25).repeat(beams, 1).cuda()
    scores = -torch.arange(beams).float() * step
    same(select(x, scores, beams, 64), select_oracle(x.cpu(), scores, beams, 64))


@pytest.mark.parametrize("dtype, groups, beams, picks, vocab", [(F16, 3, 31, 62, 68), (F32, 1, 17, 64, 4000), (BF16, 1, 60, 64, 2000), (F16, 1, 31, 62, 100000)])
def test_the_time_of_many_picks(dtype, groups, beams, picks, vocab):
    # beside a call with as many rows and few picks
    gen = torch.Generator().manual_seed(3)
    M.init(0)
    x = rows_of(gen, groups * beams, vocab, dtype)
    scores = (-torch.rand(groups * beams, generator=gen) * 9).cuda()
    micros = []
    for n in (8, picks):
        shape = B.Beams(dtype, beams, n, vocab)
        ws = torch.empty(B.beam_select_workspace(shape, groups), dtype=torch.uint8, device="cuda")
        out = [torch.empty(groups * n, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]

        def call():
            B.beam_select(shape, groups, ptr(x), ptr(scores), 0, *(ptr(t) for t in out), 0, 0, 0, 0, ptr(ws), ws.numel(), stream=stream())

        times = []
        for _ in range(6):
            ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            call()
            ends[0].record()
            for _ in range(10):
                call()
            ends[1].record()
            torch.cuda.synchronize()
            times.append(ends[0].elapsed_time(ends[1]) * 100)
        micros.append(min(times))
    print(micros)
    assert micros[1] < 5 * micros[0], micros
