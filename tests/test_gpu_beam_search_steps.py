"""The example of a beam search, step by step: captured steps against steps by themselves, every row's attention, and every
selection against the logits that it was made from."""
import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import attention_oracle, check_attention
from test_gpu_beam_search import example, held
from test_gpu_beams import same, select_oracle

pytestmark = pytest.mark.gpu
STATE = ("tokens", "parents", "scores", "ended", "history", "known", "lengths", "table", "shares", "ring", "ring_state", "status", "copy_from",
         "copy_to", "copy_tokens")


def begun(beams, prompts, longest=130, **layer):
    search = example().BeamSearch(len(prompts), beams, longest, vocab=500, q_heads=4, kv_heads=2, head_dim=64, hidden=96, **layer)
    gen = torch.Generator().manual_seed(beams)
    search.begin([torch.randint(8, 500, (n,), generator=gen).tolist() for n in prompts])
    return search


@pytest.mark.parametrize("beams, prompts, end", [(3, [5, 40, 16], -1), (8, [100, 33], 7)])
def test_captured_steps_and_steps_by_themselves(beams, prompts, end):
    one, other = begun(beams, prompts, end_token=end), begun(beams, prompts, end_token=end)
    graph, _, _ = one.capture_search()
    for step in range(24):
        graph.replay()
        out, _ = other.advance()
        other.select(out.flatten(1) @ other.to_vocab)
        torch.cuda.synchronize()
        for name in STATE:
            assert torch.equal(getattr(one, name), getattr(other, name)), (step, name)
        for row in range(0, one.requests, 3):
            n = int(one.lengths[row])
            assert all(torch.equal(a, b) for a, b in zip(held(one, row, n), held(other, row, n)))


@pytest.mark.parametrize("cache_dtype", [M.BFLOAT16, M.F8E4M3])
@pytest.mark.parametrize("beams, prompts, end", [(3, [5, 40, 16], -1), (8, [100, 33], 7), (16, [64, 20], -1)])
def test_every_row_of_every_step(cache_dtype, beams, prompts, end, monkeypatch):
    search = begun(beams, prompts, end_token=end, cache_dtype=cache_dtype)
    decode, lse = A.paged_decode_shared, torch.empty(search.requests, 4, device="cuda")
    monkeypatch.setattr(A, "paged_decode_shared", lambda *a, **k: decode(*a[:16], lse.data_ptr(), *a[17:], **k))
    for step in range(12):
        out, q = search.advance()
        torch.cuda.synchronize()
        for row in range(search.requests):
            length = int(search.lengths[row])
            keys, values = held(search, row, length)
            want = attention_oracle(q[row: row + 1].double().cpu(), keys, values, [length - 1], search.head_dim ** -0.5)
            check_attention(out[row: row + 1], lse[row: row + 1], want, M.BFLOAT16, search.head_dim)
        logits = out.flatten(1) @ search.to_vocab
        before = {k: getattr(search, k).cpu() for k in ("scores", "ended", "history", "known", "next_history")}
        search.select(logits)
        torch.cuda.synchronize()
        want = select_oracle(logits.cpu(), before["scores"], beams, beams, before["ended"] if end >= 0 else None, end, before["history"],
                             before["known"], before["next_history"])
        same({"scores": search.next_scores, "tokens": search.tokens, "parents": search.parents, "ended": search.next_ended,
              "history": search.next_history}, want)
