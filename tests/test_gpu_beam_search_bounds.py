"""The example of a beam search: the bounds that it names hold, behind prompts of any length."""
import pytest
import torch

from manifesto_amd import attention as A
from test_gpu_beam_search import check_cache, check_pages, example

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams, prompts, longest", [(3, [16, 31], 40), (2, [5, 33, 64, 1], 70), (2, [1, 3], 224), (4, [18436] + [3] * 7, 18440)])
def test_no_request_has_more_than_the_bounds(beams, prompts, longest, monkeypatch):
    module = example()
    search = module.BeamSearch(len(prompts), beams, longest, vocab=200, q_heads=16, kv_heads=4, head_dim=64, hidden=64)
    gen = torch.Generator().manual_seed(beams)
    search.begin([torch.randint(0, 200, (n,), generator=gen).tolist() for n in prompts])
    calls = []

    def watched(*args, **kwargs):
        calls.append((args[11], args[13]))
        return decode(*args, **kwargs)

    decode = A.paged_decode_shared
    monkeypatch.setattr(A, "paged_decode_shared", watched)
    for _ in range(longest - max(prompts)):
        out, _ = search.advance()
        own = search.lengths.cpu() - search.shared.cpu().repeat_interleave(beams)
        assert int(search.shared.max()) <= calls[-1][0] and int(own.max()) <= calls[-1][1]
        assert search.status.tolist() == [0] * search.requests
        search.select(out.flatten(1) @ search.to_vocab)
    assert int(search.lengths.max()) == longest and len(calls) == longest - max(prompts)
    if longest < 1000:
        check_cache(search)
    check_pages(search)
