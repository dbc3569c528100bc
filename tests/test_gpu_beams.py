"""Beam search's selection over beams and vocabulary, against f64."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import beams as B
from paged_util import TORCH, ptr, stream

pytestmark = pytest.mark.gpu
F32, F16, BF16 = M.FLOAT32, M.FLOAT16, M.BFLOAT16
OUT = ("scores", "tokens", "parents", "ended", "history")


def select_oracle(x, scores, beams, picks, ended=None, end_token=-1, history=None, known=None, history_out=None):
    """x [rows, vocab] on the CPU.  Candidates in the order of score (f64), beam, logit and token."""
    rows, vocab = x.shape
    x, groups = x.double(), rows // beams
    z = torch.logsumexp(x, -1)
    out = {"scores": torch.full((groups * picks,), -math.inf, dtype=torch.float64), "tokens": torch.full((groups * picks,), -1),
           "parents": torch.full((groups * picks,), -1), "ended": torch.zeros(groups * picks, dtype=torch.uint8),
           "history": None if history is None else history_out.clone()}
    for g in range(groups):
        found = []
        for row in range(g * beams, (g + 1) * beams):
            s = float(scores[row].double())
            if ended is not None and ended[row]:
                found.append((s, -row, 0.0, -end_token))
                continue
            best = torch.sort(x[row], descending=True, stable=True).indices[:picks]
            found += [(s + (float(x[row, t]) - float(z[row])), -row, float(x[row, t]), -int(t)) for t in best]
        found = sorted((f for f in found if -math.inf < f[0] < math.inf), reverse=True)[:picks]
        for i, (s, row, _, token) in enumerate(found):
            at = g * picks + i
            out["scores"][at], out["tokens"][at], out["parents"][at] = s, -token, -row
            out["ended"][at] = int((ended is not None and bool(ended[-row])) or -token == end_token)
            if history is not None:
                n, width = min(max(int(known[g]), 0), history.shape[1]), history.shape[1]
                out["history"][at, :n] = history[-row, :n]
                if n < width:
                    out["history"][at, n] = -token
    return out


def select(x, scores, beams, picks, vocab=None, dtype=F32, ended=None, end_token=-1, history=None, known=None, history_out=None, on=None):
    """x may be strided: its rows are taken as they stand."""
    M.init(0)
    d = lambda t: None if t is None else t.cuda()  # noqa: E731
    rows, vocab = x.shape
    groups, n = rows // beams, rows // beams * picks
    shape = B.Beams(dtype, beams, picks, vocab, end_token=end_token, logits_stride=x.stride(0) if rows > 1 else 0,
                    history_stride=0 if history is None else history.shape[1])
    need = B.beam_select_workspace(shape, groups)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
    out = {"scores": torch.full((n,), 7.0, device="cuda"), "tokens": torch.full((n,), -9, dtype=torch.int32, device="cuda"),
           "parents": torch.full((n,), -9, dtype=torch.int32, device="cuda"), "ended": torch.full((n,), 9, dtype=torch.uint8, device="cuda"),
           "history": d(history_out)}
    keep = [d(t) for t in (scores, ended, history, known)]
    torch.cuda.synchronize()
    B.beam_select(shape, groups, ptr(x), ptr(keep[0]), ptr(keep[1]), ptr(out["scores"]), ptr(out["tokens"]), ptr(out["parents"]), ptr(out["ended"]),
                  ptr(keep[2]), ptr(keep[3]), ptr(out["history"]), ptr(ws), need, stream=stream() if on is None else on)
    torch.cuda.synchronize()
    return out


def same(got, want):
    for k in ("tokens", "parents", "ended", "history"):
        if want[k] is not None:
            assert torch.equal(got[k].cpu().long(), want[k].long()), k
    got, want = got["scores"].double().cpu(), want["scores"]
    none = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & (got < 0), none)
    # the result's rounding, and that of the exponentials' arguments, 2^-24 of up to 30 log2(e) each, in their sum
    assert ((got - want)[~none].abs() <= want[~none].abs() * 2.0 ** -24 + 30 * 2.0 ** -24).all()


def rows_of(gen, rows, vocab, dtype, std=2.5, stride=None):
    x = torch.empty(rows, stride or vocab, dtype=TORCH[dtype], device="cuda")[:, :vocab]
    x.copy_(torch.randn(rows, vocab, generator=gen) * std)
    return x


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 511, 4095, 4096, 4097, 32003, 70001])
@pytest.mark.parametrize("groups, beams, picks", [(1, 1, 1), (1, 4, 4), (3, 5, 10), (2, 3, 64)])
def test_selection(dtype, vocab, groups, beams, picks):
    gen = torch.Generator().manual_seed(vocab + picks)
    x = rows_of(gen, groups * beams, vocab, dtype)
    scores = -torch.rand(groups * beams, generator=gen) * 5
    same(select(x, scores, beams, picks, dtype=dtype), select_oracle(x.cpu(), scores, beams, picks))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups, beams, vocab", [(60, 9, 20000), (40, 16, 3000), (300, 4, 100), (1, 256, 5000), (17, 31, 40000)])
def test_many_rows(dtype, groups, beams, vocab):
    # pieces of every size: as many as there are rows to fill the card
    gen = torch.Generator().manual_seed(groups)
    x = rows_of(gen, groups * beams, vocab, dtype)
    scores = -torch.rand(groups * beams, generator=gen) * 5
    same(select(x, scores, beams, 7, dtype=dtype), select_oracle(x.cpu(), scores, beams, 7))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("stride", [1003, 1004, 1008, 1100])
def test_rows_at_any_stride(dtype, stride):
    gen = torch.Generator().manual_seed(stride)
    x = rows_of(gen, 6, 1001, dtype, stride=stride)
    scores = -torch.rand(6, generator=gen)
    same(select(x, scores, 3, 6, dtype=dtype), select_oracle(x.cpu(), scores, 3, 6))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lowest", [-math.inf, None])
@pytest.mark.parametrize("allowed", [0, 1, 3, 40])
def test_masked_rows(dtype, lowest, allowed):
    # -inf is no candidate; the type's lowest value is one, the lowest tokens first
    gen = torch.Generator().manual_seed(allowed)
    low = float(torch.finfo(TORCH[dtype]).min) if lowest is None else lowest
    x = torch.full((4, 50001), low, dtype=TORCH[dtype], device="cuda")
    for row in range(4):
        at = torch.randperm(50001, generator=gen)[:allowed]
        x[row, at.cuda()] = (torch.randn(allowed, generator=gen) * 3).to(x.dtype).cuda()
    scores = torch.tensor([-1.0, -2.0, -0.5, -3.0])
    want = select_oracle(x.cpu(), scores, 2, 10)
    assert bool((want["tokens"] < 0).any()) == (lowest is not None and 2 * allowed < 10)
    got = select(x, scores, 2, 10, dtype=dtype)
    if lowest is None and allowed < 10:  # scores of 3e38 and more: as they are rounded
        assert torch.equal(got["tokens"].cpu().long(), want["tokens"]) and torch.equal(got["parents"].cpu().long(), want["parents"])
        assert ((got["scores"].cpu().double() - want["scores"]).abs() <= want["scores"].abs() * 2.0 ** -23).all()
    else:
        same(got, want)


def test_equal_logits_and_equal_beams():
    x = torch.zeros(6, 9000, device="cuda")
    x[1, 100:8000:7] = 1.0
    x[2] = x[1]
    scores = torch.tensor([0.0, -0.5, -0.5, 0.0, 0.0, 0.0])
    got = select(x, scores, 3, 12)
    same(got, select_oracle(x.cpu(), scores, 3, 12))
    assert got["tokens"][12:].tolist() == list(range(12)) and got["parents"][12:].tolist() == [3] * 12
    minus = torch.where(torch.arange(5000) % 2 == 0, -0.0, 0.0).repeat(2, 1).cuda()  # one value
    assert select(minus, torch.zeros(2), 2, 5)["tokens"].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("packets", [1, 8])
def test_large_logits_in_few_columns_of_threads(dtype, packets):
    # more than the list holds: all of the largest lie with threads of the same column
    per = 4 if dtype == F32 else 8
    rows = 4 if packets == 1 else 600
    vocab = 512 * per * packets
    gen = torch.Generator().manual_seed(packets)
    base = torch.randn(rows, vocab, generator=gen) * 0.1
    token = torch.arange(vocab)
    inside = (token // per % 64) < 40
    order = torch.rand(rows, vocab, generator=gen) * 8 + 4
    x = torch.where(inside, order, base).to(TORCH[dtype]).cuda()
    scores = -torch.rand(rows, generator=gen)
    for picks in (3, 41, 64):
        same(select(x, scores, 2, picks, dtype=dtype), select_oracle(x.cpu(), scores, 2, picks))


def test_values_that_are_not_finite():
    gen = torch.Generator().manual_seed(6)
    x = rows_of(gen, 12, 5000, F32)
    x[1, 17], x[2, 4999], x[3, 0] = math.nan, math.inf, -math.inf
    x[6:9] = math.nan
    scores = torch.tensor([-1.0] * 12)
    scores[4], scores[5], scores[9], scores[10] = -math.inf, math.nan, math.inf, -1e30
    got = select(x, scores, 3, 6)
    ok = [0, 3, 10, 11]
    for g in range(4):
        parents = got["parents"][6 * g: 6 * g + 6].tolist()
        mine = [r for r in ok if r // 3 == g]
        assert set(parents) <= set(mine) | {-1} and (parents == [-1] * 6) == (not mine)
        for name, value in (("tokens", -1), ("scores", -math.inf), ("ended", 0)):
            part = got[name][6 * g: 6 * g + 6].tolist()
            assert all((p < 0) == (t == value) for p, t in zip(parents, part) if name != "ended")
    clean = select_oracle(x[:1].cpu(), scores[:1], 1, 6)
    assert torch.equal(got["tokens"][:6].cpu().long(), clean["tokens"])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("groups, beams, picks, width", [(1, 4, 4, 30), (5, 3, 6, 300), (2, 8, 16, 9000), (40, 2, 2, 1)])
def test_ended_beams_and_histories(dtype, groups, beams, picks, width):
    gen = torch.Generator().manual_seed(width)
    rows, vocab = groups * beams, 1234
    x = rows_of(gen, rows, vocab, dtype)
    x[:, 5] += 6  # the end is likely
    scores = -torch.rand(rows, generator=gen) * 4
    ended = (torch.rand(rows, generator=gen) < 0.4).to(torch.uint8) * 3
    ended[0] = 1
    x[0] = math.nan  # which does not matter
    history = torch.randint(0, vocab, (rows, width), generator=gen, dtype=torch.int32)
    known = torch.randint(-1, width + 3, (groups,), generator=gen, dtype=torch.int32)
    fill = torch.full((groups * picks, width), -3, dtype=torch.int32)
    args = dict(ended=ended, end_token=5, history=history, known=known, history_out=fill)
    want = select_oracle(x.cpu(), scores, beams, picks, **args)
    assert int(want["ended"].sum()) > 0
    same(select(x, scores, beams, picks, dtype=dtype, **args), want)
    same(select(x[1:3].contiguous(), scores[1:3], 2, 3, dtype=dtype, end_token=5),  # marks without beams that had ended before
         select_oracle(x[1:3].cpu(), scores[1:3], 2, 3, end_token=5))


def test_all_beams_have_ended():
    x = torch.zeros(3, 100, device="cuda")
    got = select(x, torch.tensor([-2.0, -1.0, -2.0]), 3, 5, ended=torch.ones(3, dtype=torch.uint8), end_token=0)
    assert got["parents"].tolist() == [1, 0, 2, -1, -1] and got["tokens"].tolist() == [0, 0, 0, -1, -1]
    assert got["scores"].tolist()[:3] == [-1.0, -2.0, -2.0] and got["ended"].tolist() == [1, 1, 1, 0, 0]


@pytest.mark.parametrize("at", [-1.0, -1000.0])
def test_beams_that_are_close_are_compared_before_rounding(at):
    # beams alike but for one unlikely token, which moves their sums by 1e-5 each; f32 has steps of 6e-5 at 1000
    gen = torch.Generator().manual_seed(11)
    x = rows_of(gen, 8, 3001, F32, std=1.0)
    x[:] = x[0].clone()
    order = torch.tensor([3, 0, 6, 1, 7, 2, 5, 4])
    x[:, 77] = torch.log(0.05 * (order + 1.0)).cuda()  # of a sum of about 5000
    scores = torch.full((8,), at)
    want = select_oracle(x.cpu(), scores, 8, 64)
    assert (want["scores"][:7] - want["scores"][1:8] < 2e-5).all() and want["parents"][:8].tolist() == torch.argsort(order).tolist()
    same(select(x, scores, 8, 64), want)


def test_a_large_vocabulary_and_rows_past_2_to_the_31():
    M.init(0)
    vocab = 1 << 24
    x = torch.full((140, vocab), -20.0, dtype=torch.bfloat16, device="cuda")  # 2.3e9 logits
    gen = torch.Generator().manual_seed(2)
    top = torch.randint(0, vocab, (140, 6), generator=gen)
    top[139, 0] = vocab - 1
    x.scatter_(1, top.cuda(), (torch.arange(6).float()[None, :] + 2).expand(140, 6).bfloat16().cuda())
    scores = -torch.rand(140, generator=gen)
    got = select(x, scores, 2, 4, dtype=BF16)
    for g in (0, 30, 69):
        rows = slice(2 * g, 2 * g + 2)
        want = select_oracle(x[rows].cpu(), scores[rows], 2, 4)
        same({"scores": got["scores"][4 * g: 4 * g + 4], "tokens": got["tokens"][4 * g: 4 * g + 4], "parents": got["parents"][4 * g: 4 * g + 4] - 2 * g,
              "ended": got["ended"][4 * g: 4 * g + 4]}, want)


def test_another_stream_and_a_captured_selection():
    gen = torch.Generator().manual_seed(3)
    x = rows_of(gen, 8, 10007, BF16)
    scores = (-torch.rand(8, generator=gen)).cuda()
    side = torch.cuda.Stream()
    want = select_oracle(x.cpu(), scores.cpu(), 4, 4)
    same(select(x, scores, 4, 4, dtype=BF16, on=side.cuda_stream), want)
    shape = B.Beams(BF16, 4, 4, 10007)
    ws = torch.empty(B.beam_select_workspace(shape, 2), dtype=torch.uint8, device="cuda")
    out = {"scores": torch.zeros(8, device="cuda"), "tokens": torch.zeros(8, dtype=torch.int32, device="cuda"),
           "parents": torch.zeros(8, dtype=torch.int32, device="cuda"), "ended": torch.zeros(8, dtype=torch.uint8, device="cuda")}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        B.beam_select(shape, 2, ptr(x), ptr(scores), 0, ptr(out["scores"]), ptr(out["tokens"]), ptr(out["parents"]), ptr(out["ended"]), 0, 0, 0,
                      ptr(ws), ws.numel(), stream=side.cuda_stream)
    for _ in range(4):
        x.copy_(torch.randn(8, 10007, generator=gen))
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        same(out, select_oracle(x.cpu(), scores.cpu(), 4, 4))


def test_refused_arguments():
    M.init(0)
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = ptr(t)

    def call(shape=None, **args):
        base = dict(groups=1, logits=p, scores=p, ended=0, scores_out=p + 1024, tokens=p, parents=p, ended_out=0, history=0, known=0, history_out=0,
                    workspace=p, workspace_bytes=1 << 16)
        B.beam_select(B.Beams(**{"dtype": F32, "beams": 2, "picks": 2, "vocab": 10, **(shape or {})}), **{**base, **args})

    for bad, message in ((dict(shape=dict(dtype=M.F8E4M3)), "f32/f16/bf16"), (dict(shape=dict(beams=0)), "beams"), (dict(shape=dict(beams=257)), "beams"),
                         (dict(shape=dict(picks=0)), "picks"), (dict(shape=dict(picks=65)), "picks"), (dict(shape=dict(vocab=0)), "tokens"),
                         (dict(shape=dict(vocab=(1 << 24) + 1)), "tokens"), (dict(shape=dict(end_token=10)), "end token"),
                         (dict(shape=dict(end_token=-2)), "end token"), (dict(shape=dict(logits_stride=9)), "overlap"),
                         (dict(shape=dict(history_stride=-1)), "history"), (dict(groups=-1), "groups"), (dict(groups=2 ** 31 - 1), "too many"),
                         (dict(logits=0), "NULL"), (dict(scores=0), "NULL"), (dict(parents=0), "NULL"), (dict(history=p), "NULL"),
                         (dict(shape=dict(history_stride=4), history=p, known=p, history_out=p + 16), "history_out"),
                         (dict(scores_out=p + 4), "scores_out"), (dict(shape=dict(end_token=1), ended=p, ended_out=p + 1), "ended_out"), (dict(ended=p), "end token"), (dict(workspace=0), "workspace"),
                         (dict(workspace=p + 8), "workspace"), (dict(workspace_bytes=40), "workspace")):
        with pytest.raises(M.MFHError, match=message):
            call(**bad)
    call(groups=0, logits=0)
