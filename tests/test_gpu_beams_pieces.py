"""Beam search's selection by pieces of 1, 2, 4 and 8 packets a thread, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from test_gpu_beams import rows_of, same, select, select_oracle
from paged_util import TORCH

pytestmark = pytest.mark.gpu
F32, F16, BF16 = M.FLOAT32, M.FLOAT16, M.BFLOAT16
THREADS, CUS = 512, 256


def rows_for(packets, dtype, vocab):
    """The fewest rows (in beams of four) that are cut into pieces of that many packets a thread: a piece is as large as
    leaves every CU two."""
    def pieces(n):
        return -(-vocab // (THREADS * n * (4 if dtype == F32 else 8)))

    if packets == 1:
        return 4
    rows = -(-2 * CUS // pieces(packets)) + 3 & ~3
    assert packets == 8 or rows * pieces(2 * packets) < 2 * CUS
    return rows


def vocab_for(dtype):
    """A piece of 8 packets holds the row, two of 4 do, three of 2, six of 1; the last one ends inside a packet."""
    return 9999 if dtype == F32 else 19999


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packets", [1, 2, 4, 8])
@pytest.mark.parametrize("picks", [1, 7, 64])
def test_pieces(dtype, packets, picks):
    vocab = vocab_for(dtype)
    rows = rows_for(packets, dtype, vocab)
    gen = torch.Generator().manual_seed(packets + picks)
    x = rows_of(gen, rows, vocab, dtype, stride=vocab + packets)
    scores = -torch.rand(rows, generator=gen) * 5
    same(select(x, scores, 4, picks, dtype=dtype), select_oracle(x.cpu(), scores, 4, picks))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packets", [2, 4])
def test_pieces_of_masked_equal_and_ended_rows(dtype, packets):
    vocab = vocab_for(dtype)
    rows = rows_for(packets, dtype, vocab)
    gen = torch.Generator().manual_seed(packets)
    x = rows_of(gen, rows, vocab, dtype)
    x[::4, vocab // 3:] = -math.inf  # pieces without a candidate
    x[1::8] = 0.5  # rows of one value
    x[2::12] = -math.inf
    x[2::12, vocab - 1] = 0.25  # one token, the last
    scores = -torch.rand(rows, generator=gen) * 4
    ended = (torch.rand(rows, generator=gen) < 0.25).to(torch.uint8)
    args = dict(ended=ended, end_token=5)
    same(select(x, scores, 4, 9, dtype=dtype, **args), select_oracle(x.cpu(), scores, 4, 9, **args))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packets", [2, 4])
def test_pieces_with_large_logits_in_few_columns_of_threads(dtype, packets):
    # more than the list holds
    per, vocab = 4 if dtype == F32 else 8, vocab_for(dtype)
    rows = rows_for(packets, dtype, vocab)
    gen = torch.Generator().manual_seed(packets)
    token = torch.arange(vocab)
    x = torch.where(token // per % 64 < 40, torch.rand(rows, vocab, generator=gen) * 8 + 4, torch.randn(rows, vocab, generator=gen) * 0.1)
    x, scores = x.to(TORCH[dtype]).cuda(), -torch.rand(rows, generator=gen)
    for picks in (3, 64):
        same(select(x, scores, 4, picks, dtype=dtype), select_oracle(x.cpu(), scores, 4, picks))


@pytest.mark.parametrize("packets", [1, 2, 4])
def test_results_that_are_missing_are_not_marked_as_ended(packets):
    vocab = vocab_for(BF16)
    rows = rows_for(packets, BF16, vocab)
    gen = torch.Generator().manual_seed(packets)
    x = torch.full((rows, vocab), -math.inf, dtype=torch.bfloat16, device="cuda")
    x[::4, 3] = 1.0  # one candidate in a group; those of the others are not numbers, and one has none
    x[1::4], x[2::4, 7] = math.nan, math.inf
    scores = -torch.rand(rows, generator=gen)
    ended = torch.zeros(rows, dtype=torch.uint8)
    ended[3::8] = 1
    scores[3::16] = -math.inf
    out = select(x, scores, 4, 6, dtype=BF16, ended=ended, end_token=0)
    got = {k: v.cpu().view(-1, 6) for k, v in out.items() if v is not None}
    for g in range(rows // 4):
        end = 4 * g + 3 if bool(ended[4 * g + 3]) and float(scores[4 * g + 3]) > -math.inf else -1
        want = sorted([(float(scores[4 * g]), 4 * g, 3, 0)] + ([(float(scores[end]), end, 0, 1)] if end >= 0 else []), reverse=True)
        want += [(-math.inf, -1, -1, 0)] * (6 - len(want))
        for i, (score, parent, token, marked) in enumerate(want):
            assert got["parents"][g, i] == parent and got["tokens"][g, i] == token and got["ended"][g, i] == marked, (g, i)
            assert float(got["scores"][g, i]) == pytest.approx(score, rel=2.0 ** -23)


def test_a_score_past_the_range_of_f32():
    # it is a continuation like any other, and -inf once rounded
    x = torch.full((2, 3000), -3e38, device="cuda")
    x[:, 11] = 2.0
    out = select(x, torch.tensor([-1.0, -1e38]), 2, 4)
    assert out["tokens"].tolist() == [11, 11, 0, 1] and out["parents"].tolist() == [0, 1, 0, 0]
    assert out["scores"].tolist()[:2] == torch.tensor([-1.0, -1e38]).tolist()
    out = select(x[:1], torch.tensor([-1e38]), 1, 3)
    assert out["tokens"].tolist() == [11, 0, 1] and out["parents"].tolist() == [0, 0, 0]
    assert out["scores"].tolist()[1:] == [-math.inf] * 2
