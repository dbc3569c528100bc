"""Block tables and slot maps from request lengths, against a loop over the requests."""
import ctypes

import numpy as np
import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import plan_oracle, ptr, stream

pytestmark = pytest.mark.gpu
OUT = ("table", "ring", "ring_state", "slots", "positions", "starts", "lengths", "status")


def plan(before, after, page, table, width, ring, head, tail, tokens):
    M.init(0)
    dev = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in (
        ("before", before), ("after", after), ("table", table), ("ring", ring), ("state", np.array([head, tail], np.int64)))}
    n = len(before)
    out = {"ring_state": torch.full((2,), -9, dtype=torch.int64, device="cuda"),
           "slots": torch.full((tokens,), -9, dtype=torch.int64, device="cuda"),
           "positions": torch.full((tokens,), -9, dtype=torch.int32, device="cuda"),
           "starts": torch.full((n + 1,), -9, dtype=torch.int32, device="cuda"),
           "lengths": torch.full((n,), -9, dtype=torch.int32, device="cuda"),
           "status": torch.full((n,), -9, dtype=torch.int32, device="cuda")}
    A.page_plan(ptr(dev["before"]), ptr(dev["after"]), n, page, ptr(dev["table"]), width, ptr(dev["ring"]), len(ring),
                ptr(dev["state"]), ptr(out["ring_state"]), ptr(out["slots"]), ptr(out["positions"]), tokens, ptr(out["starts"]),
                ptr(out["lengths"]), ptr(out["status"]), table_stride=table.shape[1], stream=stream())
    out.update(table=dev["table"], ring=dev["ring"])
    torch.cuda.synchronize()
    return {k: out[k].cpu().numpy() for k in OUT}


def state(rng, n, page, width, longest, spare, stride=None, turn=0):
    """Requests that hold pages, the free ones in a ring that starts anywhere."""
    before = rng.integers(0, longest + 1, n).astype(np.int32)
    have = -(-before // page)
    pages = int(have.sum()) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((n, stride or max(width, 1)), -1, np.int32)
    at = 0
    for r in range(n):
        table[r, : have[r]] = order[at: at + have[r]]
        at += have[r]
    head = turn * pages + int(rng.integers(0, pages + 1))
    ring = np.full(max(pages, 1), -1, np.int32)
    ring[(head + np.arange(spare)) % len(ring)] = order[at:]
    return before, table, ring, head, head + spare


def same(got, want):
    for k in OUT:
        assert np.array_equal(got[k], want[k]), k


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("page", [1, 16, 100])
def test_mixed_steps_match_the_loop(n, page):
    rng = np.random.default_rng(n * 1000 + page)
    longest = 70 if n > 100 else 700
    width = -(-2 * longest // page) + 1
    before, table, ring, head, tail = state(rng, n, page, width, longest, spare=int(1.2 * n * longest / page) + n, stride=width + 3, turn=5)
    after = np.where(rng.random(n) < 0.5, before + rng.integers(0, longest, n), rng.integers(0, longest, n)).astype(np.int32)
    after[rng.random(n) < 0.1] = 0
    tokens = int(np.maximum(after - before, 0).sum()) + 5
    args = (before, after, page, table, width, ring, head, tail, tokens)
    want = plan_oracle(*args)
    assert (want["status"] == 0).all()
    same(plan(*args), want)


@pytest.mark.parametrize("seed", range(8))
def test_refusals_leave_a_request_as_it_was(seed):
    # too few pages, rows that are too narrow, tokens past the end, negative lengths
    rng = np.random.default_rng(seed)
    n, page, width = 300, 8, 12
    before, table, ring, head, tail = state(rng, n, page, width, 90, spare=int(rng.integers(0, 900)))
    after = rng.integers(0, 100, n).astype(np.int32)
    after[rng.random(n) < 0.03] = 2_000_000_000
    after[rng.random(n) < 0.03] = -5
    before[rng.random(n) < 0.02] = -1
    tokens = int(rng.integers(0, 2 * np.maximum(np.minimum(after, 100) - before, 0).sum()))
    args = (before, after, page, table, width, ring, head, tail, tokens)
    want = plan_oracle(*args)
    assert len(set(want["status"].tolist())) >= 2
    same(plan(*args), want)


def test_no_requests_no_tokens_no_table():
    none = np.zeros(0, np.int32)
    got = plan(none, none, 16, np.zeros((0, 1), np.int32), 0, np.zeros(1, np.int32), 3, 3, 4)
    assert got["starts"].tolist() == [0] and got["slots"].tolist() == [-1] * 4 and got["ring_state"].tolist() == [3, 3]
    got = plan(np.zeros(2, np.int32), np.array([0, 1], np.int32), 16, np.zeros((2, 1), np.int32), 0, np.zeros(1, np.int32), 0, 1, 1)
    assert got["status"].tolist() == [0, 2] and got["lengths"].tolist() == [0, 0] and got["slots"].tolist() == [-1]


def test_a_page_whose_number_is_negative_gives_no_slot():
    got = plan(np.array([3], np.int32), np.array([5], np.int32), 4, np.array([[-1, -1]], np.int32), 2, np.array([6, 7], np.int32), 0, 2, 2)
    assert got["slots"].tolist() == [-1, 24] and got["positions"].tolist() == [3, 4]


def test_pages_are_never_lost_or_held_twice_over_many_steps():
    rng = np.random.default_rng(3)
    n, page, width, pages = 40, 4, 30, 500
    table = np.full((n, width), -1, np.int32)
    ring, head, tail = rng.permutation(pages).astype(np.int32), 0, pages
    length = np.zeros(n, np.int32)
    for _ in range(60):
        after = np.where(rng.random(n) < 0.15, 0, length + rng.integers(0, 12, n)).astype(np.int32)
        tokens = int(np.maximum(after - length, 0).sum())
        got = plan(length, after, page, table, width, ring, head, tail, tokens)
        same(got, plan_oracle(length, after, page, table, width, ring, head, tail, tokens))
        table, ring, length = got["table"], got["ring"], got["lengths"]
        head, tail = got["ring_state"].tolist()
        held = np.concatenate([table[r, : -(-length[r] // page)] for r in range(n)])
        free = ring[(head + np.arange(tail - head)) % pages]
        assert sorted(np.concatenate([held, free]).tolist()) == list(range(pages))


def test_refused_arguments():
    M.init(0)
    t = torch.zeros(64, dtype=torch.int64, device="cuda")
    p = ptr(t)
    good = dict(before=p, after=p, requests=1, page_size=16, table=p, table_width=4, ring=p, ring_size=4, ring_state=p,
                ring_state_out=p + 64, slots=p, positions=p, tokens=4, starts=p, lengths=p, status=p)
    for bad, message in (({"requests": -1}, "negative number of requests"), ({"page_size": 0}, "page size"),
                         ({"tokens": -1}, "tokens"), ({"tokens": (1 << 30) + 1}, "tokens"), ({"ring_size": 0}, "ring"),
                         ({"table_width": -1}, "table width"), ({"table_stride": 3}, "table width"),
                         ({"before": 0}, "NULL"), ({"table": 0}, "NULL"), ({"slots": 0}, "NULL"), ({"ring": 0}, "NULL"),
                         ({"starts": 0}, "NULL"), ({"ring_state_out": p}, "ring_state_out")):
        with pytest.raises(M.MFHError, match=message):
            A.page_plan(**{**good, **bad})


def test_lengths_in_place():
    # where one workgroup does it all; with more of them the others still read what it writes
    M.init(0)
    page, width = 16, 40
    for n, each, fits in ((3, 170, True), (600, 0, True), (3, 171, False), (600, 1, False)):
        before = np.arange(n, dtype=np.int32) % 30
        after = before + each
        pages = int((-(-after // page)).sum()) + 1
        table = np.full((n, width), -1, np.int32)
        held = 0
        for r in range(n):
            have = -(-int(before[r]) // page)
            table[r, :have] = np.arange(held, held + have)
            held += have
        ring = np.concatenate([np.arange(held, pages), np.full(held, -1)]).astype(np.int32)
        tokens = n * each
        want = plan_oracle(before, after, page, table, width, ring, 0, pages - held, tokens)
        for target in ("before", "after"):
            d = {k: torch.from_numpy(v.copy()).cuda() for k, v in (("before", before), ("after", after), ("table", table), ("ring", ring))}
            state, state_out = torch.tensor([0, pages - held]).cuda(), torch.zeros(2, dtype=torch.int64, device="cuda")
            slots, positions = torch.zeros(tokens, dtype=torch.int64, device="cuda"), torch.zeros(tokens, dtype=torch.int32, device="cuda")
            starts, status = torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")

            def call(lengths):
                A.page_plan(ptr(d["before"]), ptr(d["after"]), n, page, ptr(d["table"]), width, ptr(d["ring"]), pages, ptr(state), ptr(state_out),
                            ptr(slots), ptr(positions), tokens, ptr(starts), lengths, ptr(status), stream=stream())

            if not fits:
                for lengths in (ptr(d[target]), ptr(d[target]) + 4 * (n - 1)):
                    with pytest.raises(M.MFHError, match="lengths is before or after"):
                        call(lengths)
                continue
            call(ptr(d[target]))
            torch.cuda.synchronize()
            got = {"lengths": d[target], "slots": slots, "positions": positions, "status": status, "table": d["table"], "starts": starts}
            for k, v in got.items():
                assert np.array_equal(v.cpu().numpy(), want[k]), k
