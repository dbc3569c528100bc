"""Forks: results over what is still read are refused."""
import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import ptr, stream

pytestmark = pytest.mark.gpu
ONCE_A_REQUEST = ("lengths", "status", "copy_from", "copy_to", "copy_tokens")


def arguments(n=4, page=16, width=2, pages=8):
    M.init(0)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    t = {"parents": i(0, 0, 2, -1), "before": i(20, 0, 16, 3), "table": i(0, 1, -1, -1, 2, -1, 3, -1), "ring": i(4, 5, 6, 7, -1, -1, -1, -1),
         "ring_state": torch.tensor([0, 4, -1, -1], device="cuda"), "shares": i(*[0] * 8), "table_out": i(*[-5] * 8), "shares_out": i(*[-5] * 8),
         "ring_state_out": torch.tensor([-5, -5], device="cuda"), **{k: i(*[-5] * n) for k in ONCE_A_REQUEST},
         "workspace": torch.empty(A.page_fork_workspace(n, pages), dtype=torch.uint8, device="cuda")}
    args = {k: ptr(x) for k, x in t.items()}
    return t, dict(args, keep=0, requests=n, page_size=page, table_width=width, pages=pages, ring_size=pages, workspace_bytes=t["workspace"].numel(),
                   stream=stream())


@pytest.mark.parametrize("entries", [-1, 0, 1])
def test_ring_states(entries):
    t, args = arguments()
    with pytest.raises(M.MFHError, match="ring_state_out"):
        A.page_fork(**{**args, "ring_state": args["ring_state"] + 8, "ring_state_out": args["ring_state"] + 8 + 8 * entries})


@pytest.mark.parametrize("name", ONCE_A_REQUEST)
@pytest.mark.parametrize("other", ["before", "table"])
def test_results_of_requests(name, other):
    # the tables are written by a launch of their own where there are many requests
    t, args = arguments()
    size = t[other].numel()
    for entry in (0, 3 - size, size - 1, 1 - 4):
        if -3 <= entry < size:
            with pytest.raises(M.MFHError, match=f"{name} overlaps {other}"):
                A.page_fork(**{**args, name: args[other] + 4 * entry})


def test_what_may_be_one_buffer():
    # parents and keep are read before anything is written
    t, args = arguments()
    A.page_fork(**{**args, "lengths": args["parents"], "shares_out": args["shares"], "ring_state_out": args["ring_state"] + 16})
    torch.cuda.synchronize()
    assert t["parents"].tolist() == [20, 20, 16, 0] and t["status"].tolist() == [0] * 4
    assert t["table_out"].tolist() == [0, 1, 0, 4, 2, -5, -5, -5] and t["shares"].tolist() == [1] + [0] * 7
    assert t["copy_from"].tolist() == [-1, 1, -1, -1] and t["copy_to"].tolist() == [-1, 4, -1, -1] and t["copy_tokens"].tolist() == [0, 4, 0, 0]
    assert t["ring_state"].tolist() == [0, 4, 1, 5] and t["ring"].tolist() == [4, 5, 6, 7, 3, -1, -1, -1]
