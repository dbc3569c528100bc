"""Selection's workspace: what is enough for a call is enough for all smaller ones."""
import math

import pytest
import torch

import manifesto_amd as M
from manifesto_amd import beams as B
from paged_util import ptr, stream
from test_gpu_beams import rows_of, same, select_oracle

pytestmark = pytest.mark.gpu
F32, F16, BF16 = M.FLOAT32, M.FLOAT16, M.BFLOAT16


def need(dtype, groups, beams, picks, vocab):
    M.init(0)
    return B.beam_select_workspace(B.Beams(dtype, beams, picks, vocab), groups)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [100, 32003, 131072])
def test_fewer_groups_need_no_more(dtype, vocab):
    sizes = [need(dtype, n, 4, 8, vocab) for n in range(1, 400)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_smaller_sizes_need_no_more(dtype):
    gen = torch.Generator().manual_seed(1)

    def up_to(most):
        return max(1, min(most, int(math.exp(float(torch.rand((), generator=gen)) * math.log(most + 1)))))

    for _ in range(5000):
        large = up_to(1000), up_to(256), up_to(64), up_to(1 << 20)
        small = tuple(up_to(x) for x in large)
        assert need(dtype, *small) <= need(dtype, *large), (small, large)


@pytest.mark.parametrize("dtype, vocab", [(F32, 20000), (BF16, 40000)])
def test_one_workspace_for_fewer_and_fewer_groups(dtype, vocab):
    # pieces of 8, 4, 2 and 1 packets; nothing is written behind what the largest call asks for
    gen = torch.Generator().manual_seed(2)
    x = rows_of(gen, 520, vocab, dtype)
    scores = -torch.rand(520, generator=gen) * 5
    room = need(dtype, 260, 2, 6, vocab)
    ws = torch.full((room + 4096,), 255, dtype=torch.uint8, device="cuda")
    shape, on_card = B.Beams(dtype, 2, 6, vocab), scores.cuda()
    for groups in (260, 128, 65, 33, 1):
        out = {"scores": torch.zeros(6 * groups, device="cuda"), "ended": torch.zeros(6 * groups, dtype=torch.uint8, device="cuda"),
               **{k: torch.zeros(6 * groups, dtype=torch.int32, device="cuda") for k in ("tokens", "parents")}}
        B.beam_select(shape, groups, ptr(x), ptr(on_card), 0, ptr(out["scores"]), ptr(out["tokens"]), ptr(out["parents"]), ptr(out["ended"]), 0, 0, 0,
                      ptr(ws), room, stream=stream())
        torch.cuda.synchronize()
        want = select_oracle(x[: 2 * groups].cpu(), scores[: 2 * groups], 2, 6)
        same(out, {**want, "history": None})
        assert (ws[room:] == 255).all()
