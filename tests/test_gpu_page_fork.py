"""Requests that share pages: forks against a loop over the requests, copies of pages against indexing."""
import numpy as np
import pytest
import torch

import manifesto_amd as M
from manifesto_amd import attention as A
from paged_util import ptr, stream

pytestmark = pytest.mark.gpu
F16, BF16, FP8 = M.FLOAT16, M.BFLOAT16, M.F8E4M3
OUT = ("table_out", "shares_out", "ring", "ring_state", "lengths", "status", "copy_from", "copy_to", "copy_tokens")


def fork_oracle(parents, before, keep, page, table, table_out, width, shares, ring, head, tail):
    """mfh_page_fork, request by request, with the holders of every page counted anew."""
    n, size, pages = len(parents), len(ring), len(shares)
    table_out, ring, shares = table_out.copy(), ring.copy(), np.maximum(shares, 0)
    held = lambda tokens: -(-tokens // page)  # noqa: E731
    odd = [b < 0 or held(b) > width for b in before.tolist()]
    lengths, status = np.zeros(n, np.int32), np.zeros(n, np.int32)
    copies = np.stack([np.full(n, -1), np.full(n, -1), np.zeros(n)]).astype(np.int32)
    kept, asked, taken = set(), 0, 0
    change = np.zeros(pages, np.int64)
    for r in range(n):
        if not odd[r]:
            for j in range(held(int(before[r]))):
                if 0 <= table[r, j] < pages:
                    change[table[r, j]] -= 1
    for r in range(n):
        p = int(parents[r])
        if p < 0:
            continue
        if p >= n or odd[p]:
            status[r] = 2
            continue
        take = min(int(before[p]), max(int(keep[r]), 0)) if keep is not None else int(before[p])
        last = take // page
        own = -1
        if take % page:
            if last == int(before[p]) // page and p not in kept:
                kept.add(p)
            else:
                asked += 1
                if asked > tail - head:
                    status[r] = 1
                    continue
                own = ring[(head + taken) % size]
                taken += 1
                copies[:, r] = table[p, last], own, take % page
        lengths[r] = take
        for j in range(held(take)):
            copied = j == last and copies[2, r] > 0
            table_out[r, j] = own if copied else table[p, j]
            if not copied and 0 <= table[p, j] < pages:
                change[table[p, j]] += 1
    shares = shares + change
    freed = np.flatnonzero(shares < 0)
    ring_out = ring.copy()
    for i, g in enumerate(freed):
        ring_out[(tail + i) % size] = g
    return {"table_out": table_out, "shares_out": np.maximum(shares, 0).astype(np.int32), "ring": ring_out,
            "ring_state": np.array([head + taken, tail + len(freed)]), "lengths": lengths, "status": status,
            "copy_from": copies[0], "copy_to": copies[1], "copy_tokens": copies[2]}


def fork(parents, before, keep, page, table, table_out, width, shares, ring, head, tail, in_place=False, on=None):
    M.init(0)
    n, pages = len(parents), len(shares)
    d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    dev = {k: d(v) for k, v in (("parents", parents), ("before", before), ("table", table), ("table_out", table_out), ("shares", shares),
                                ("ring", ring), ("state", np.array([head, tail], np.int64)))}
    keep = None if keep is None else d(keep)
    out = {k: torch.full((n,), -9, dtype=torch.int32, device="cuda") for k in OUT[4:]}
    out["ring_state"] = torch.full((2,), -9, dtype=torch.int64, device="cuda")
    out["shares_out"] = dev["shares"] if in_place else torch.full((pages,), -9, dtype=torch.int32, device="cuda")
    need = A.page_fork_workspace(n, pages)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    A.page_fork(ptr(dev["parents"]), ptr(dev["before"]), ptr(keep), n, page, ptr(dev["table"]), ptr(dev["table_out"]), width,
                ptr(dev["shares"]), ptr(out["shares_out"]), pages, ptr(dev["ring"]), len(ring), ptr(dev["state"]), ptr(out["ring_state"]),
                ptr(out["lengths"]), ptr(out["status"]), ptr(out["copy_from"]), ptr(out["copy_to"]), ptr(out["copy_tokens"]), ptr(ws), need,
                table_stride=table.shape[1], stream=stream() if on is None else on)
    torch.cuda.synchronize()
    out.update(table_out=dev["table_out"], ring=dev["ring"])
    return {k: out[k].cpu().numpy() for k in OUT}


def state(rng, n, page, width, longest, spare, beams=4, stride=None, more_pages=0):
    """Requests in groups that share some leading whole pages; the free pages in a ring that has turned."""
    before = rng.integers(0, longest + 1, n).astype(np.int32)
    table = np.full((n, stride or max(width, 1)), -1, np.int32)
    holders, at = [], 0
    for r in range(n):
        have, first = -(-int(before[r]) // page), r // beams * beams
        common = int(min(before[r], before[first]) // page * rng.random() * 1.2) if r != first else 0
        common = min(common, int(min(before[r], before[first])) // page)
        table[r, :common] = table[first, :common]
        table[r, common:have] = np.arange(at, at + have - common)
        at += have - common
    pages = at + spare + more_pages
    order = rng.permutation(pages).astype(np.int32)
    table = np.where(table >= 0, order[np.maximum(table, 0)], -1).astype(np.int32)
    shares = np.maximum(np.bincount(table[table >= 0], minlength=pages) - 1, 0).astype(np.int32)
    head = int(rng.integers(0, 5 * pages + 1))
    ring = np.full(pages + int(rng.integers(0, 3)), -1, np.int32)
    ring[(head + np.arange(spare)) % len(ring)] = order[at: at + spare]
    return before, table, shares, ring, head, head + spare


def same(got, want):
    for k in OUT:
        assert np.array_equal(got[k], want[k]), k


def check_counts(got, page, pages, head_tail):
    """No page is lost, held twice without a count, or free and held."""
    head, tail = head_tail
    holders = np.zeros(pages, int)
    for r, length in enumerate(got["lengths"].tolist()):
        row = got["table_out"][r, : -(-length // page)]
        np.add.at(holders, row, 1)
    for r, length in enumerate(got["lengths"].tolist()):
        assert length % page == 0 or holders[got["table_out"][r, length // page]] == 1
    assert np.array_equal(np.maximum(holders - 1, 0), got["shares_out"])
    free = got["ring"][np.arange(head, tail) % len(got["ring"])]
    assert sorted(np.concatenate([free, np.flatnonzero(holders)]).tolist()) == list(range(pages))


@pytest.mark.parametrize("n", [1, 2, 5, 64, 65, 1000, 1024, 1025, 3001])
@pytest.mark.parametrize("page, keep", [(1, True), (16, False), (16, True), (100, True)])
def test_forks_match_the_loop(n, page, keep):
    rng = np.random.default_rng(n * 1000 + page + keep)
    longest = 70 if n > 100 else 700
    width = -(-longest // page) + 1
    before, table, shares, ring, head, tail = state(rng, n, page, width, longest, spare=n, stride=width + 3)
    parents = np.where(rng.random(n) < 0.5, np.arange(n), rng.integers(-n // 4 - 1, n, n)).astype(np.int32)
    cut = rng.integers(-3, 2 * longest, n).astype(np.int32) if keep else None
    out = np.full_like(table, -5)
    args = (parents, before, cut, page, table, out, width, shares, ring, head, tail)
    want = fork_oracle(*args)
    assert (want["status"] == 0).all()
    check_counts(want, page, len(shares), want["ring_state"].tolist())
    same(fork(*args), want)
    same(fork(*args, in_place=True), want)


@pytest.mark.parametrize("n, pages", [(100, 16384), (102, 16384), (103, 16384), (100, 16385), (300, 32769), (300, 100_001)])
def test_many_pages(n, pages):
    # the count in LDS ends at 16384 pages and 12288 entries; pages that go back stand in many chunks
    rng = np.random.default_rng(pages)
    page, width = 4, 120
    before, table, shares, ring, head, tail = state(rng, n, page, width, 400, spare=400)
    more = pages - len(shares)
    assert more > 0
    names = rng.permutation(pages).astype(np.int32)  # the same pages under numbers from all over
    table, ring = np.where(table >= 0, names[np.maximum(table, 0)], -1).astype(np.int32), np.where(ring >= 0, names[np.maximum(ring, 0)], -1).astype(np.int32)
    wide = np.zeros(pages, np.int32)
    wide[names[: len(shares)]] = shares
    turned = np.full(pages, -1, np.int32)
    turned[(head + np.arange(tail - head)) % pages] = ring[(head + np.arange(tail - head)) % len(ring)]
    parents = rng.integers(-40, n, n).astype(np.int32)
    args = (parents, before, None, page, table, np.full_like(table, -5), width, wide, turned, head, tail)
    same(fork(*args), fork_oracle(*args))


@pytest.mark.parametrize("n", [40, 1500])
def test_a_long_table(n):
    # rows of several workgroups, and of few requests
    rng = np.random.default_rng(n)
    page, width, longest = 2, 2500 if n == 40 else 300, 4900 if n == 40 else 590
    before, table, shares, ring, head, tail = state(rng, n, page, width, longest, spare=n)
    parents = rng.integers(-3, n, n).astype(np.int32)
    args = (parents, before, rng.integers(0, 2 * longest, n).astype(np.int32), page, table, np.full_like(table, -5), width, shares, ring, head, tail)
    same(fork(*args), fork_oracle(*args))


@pytest.mark.parametrize("n, seed", [(50, 0), (50, 1), (1200, 2), (8192, 3)])
def test_refusals_leave_a_request_empty(n, seed):
    # too few pages, parents that are none, lengths that cannot be
    rng = np.random.default_rng(seed)
    page, width = 8, 12
    before, table, shares, ring, head, tail = state(rng, n, page, width, 90, spare=n // 5)
    parents = rng.integers(0, n, n).astype(np.int32)
    parents[rng.random(n) < 0.03] = n
    parents[rng.random(n) < 0.03] = 2 ** 31 - 1
    parents[rng.random(n) < 0.03] = -2 ** 31
    before[rng.random(n) < 0.03] = -1
    before[rng.random(n) < 0.03] = width * page + 1
    before[rng.random(n) < 0.03] = 2 ** 31 - 1
    args = (parents, before, None, page, table, np.full_like(table, -5), width, shares, ring, head, tail)
    want = fork_oracle(*args)
    assert set(want["status"].tolist()) == {0, 1, 2}
    same(fork(*args), want)


@pytest.mark.parametrize("many", [False, True])
def test_all_end_and_all_become_one(many):
    rng = np.random.default_rng(8)
    n, page, width = (1100 if many else 30), 16, 9
    before, table, shares, ring, head, tail = state(rng, n, page, width, 140, spare=n)
    for parents in (np.full(n, -1, np.int32), np.full(n, n // 2, np.int32)):
        before[n // 2] = 99  # three pages and three tokens of a fourth... of the others all but one copy
        have = -(-99 // page)
        table[n // 2, :have] = np.maximum(table[n // 2, :have], 0)
        args = (parents, before, None, page, table, np.full_like(table, -5), width, shares, ring, head, tail)
        got = fork(*args)
        same(got, fork_oracle(*args))
        assert got["lengths"].tolist() == [0 if parents[0] < 0 else 99] * n


def test_page_numbers_outside_the_cache_are_handed_on_and_not_counted():
    for n in (3, 1100):
        before = np.full(n, 20, np.int32)
        table = np.tile(np.array([[-7, 10 ** 6, -1]], np.int32), (n, 1))
        parents = np.arange(n, dtype=np.int32)
        parents[1], parents[2] = 0, -1
        args = (parents, before, None, 16, table, np.full_like(table, -5), 3, np.zeros(4, np.int32), np.array([2, 3, -1, -1], np.int32), 0, 2)
        got = fork(*args)
        same(got, fork_oracle(*args))
        assert got["copy_from"][1] == 10 ** 6 and got["copy_to"][1] == 2 and got["shares_out"].tolist() == [0] * 4


def test_no_requests():
    none = np.zeros(0, np.int32)
    for pages in (3, 40000):
        got = fork(none, none, None, 16, np.zeros((0, 1), np.int32), np.zeros((0, 1), np.int32), 0, np.arange(pages, dtype=np.int32) - 1,
                   np.zeros(pages, np.int32), 7, 9)
        assert got["shares_out"][:3].tolist() == [0, 0, 1] and got["ring_state"].tolist() == [7, 9]


@pytest.mark.parametrize("n, pages", [(24, 700), (24, 40000)])
def test_many_steps_of_a_beam_search(n, pages):
    # fork, then one token more each: page_plan takes the pages
    rng = np.random.default_rng(n)
    page, width, beams = 4, 40, 6
    table, other = np.full((n, width), -1, np.int32), np.full((n, width), -1, np.int32)
    ring, head, tail = rng.permutation(pages).astype(np.int32), 0, pages
    shares, length = np.zeros(pages, np.int32), np.zeros(n, np.int32)
    for step in range(30):
        group = np.arange(n) // beams * beams
        parents = (group + rng.integers(0, beams, n)).astype(np.int32)
        if step % 7 == 6:
            parents[group == group[rng.integers(0, n)]] = -1  # a search has ended
        args = (parents, length, None, page, table, other, width, shares, ring, head, tail)
        got = fork(*args)
        same(got, fork_oracle(*args))
        assert (got["status"] == 0).all()
        other, table, shares, ring, length = table, got["table_out"], got["shares_out"], got["ring"], got["lengths"]
        head, tail = got["ring_state"].tolist()
        check_counts(got, page, pages, (head, tail))
        d = {k: torch.from_numpy(v.copy()).cuda() for k, v in (("before", length), ("after", length + 1), ("table", table), ("ring", ring))}
        state_in, state_out = torch.tensor([head, tail]).cuda(), torch.zeros(2, dtype=torch.int64, device="cuda")
        slots, rest = torch.zeros(n, dtype=torch.int64, device="cuda"), [torch.zeros(n + 1, dtype=torch.int32, device="cuda") for _ in range(4)]
        A.page_plan(ptr(d["before"]), ptr(d["after"]), n, page, ptr(d["table"]), width, ptr(d["ring"]), pages, ptr(state_in), ptr(state_out),
                    ptr(slots), ptr(rest[0]), n, ptr(rest[1]), ptr(rest[2]), ptr(rest[3]), stream=stream())
        torch.cuda.synchronize()
        assert len(set(slots.tolist())) == n and min(slots.tolist()) >= 0  # nobody writes where another one does
        table, ring, length = d["table"].cpu().numpy(), d["ring"].cpu().numpy(), rest[2][:n].cpu().numpy()
        head, tail = state_out.tolist()


def test_refused_arguments():
    M.init(0)
    t, big = torch.zeros(4096, dtype=torch.int64, device="cuda"), torch.zeros(4096, dtype=torch.int64, device="cuda")
    p, o = ptr(t), ptr(big)
    good = dict(parents=p, before=p, keep=0, requests=2, page_size=16, table=p, table_out=o, table_width=4, shares=p, shares_out=o, pages=4,
                ring=p, ring_size=4, ring_state=p, ring_state_out=p + 64, lengths=o, status=o, copy_from=o, copy_to=o, copy_tokens=o,
                workspace=o, workspace_bytes=4096)
    for bad, message in (({"requests": -1}, "requests"), ({"requests": 8193}, "8192"), ({"page_size": 0}, "page size"), ({"pages": 0}, "pages"),
                         ({"pages": (1 << 30) + 1}, "pages"), ({"ring_size": 3}, "ring"), ({"ring_size": (1 << 30) + 1}, "ring"),
                         ({"table_width": -1}, "table width"), ({"table_stride": 3}, "table width"), ({"parents": 0}, "NULL"), ({"before": 0}, "NULL"),
                         ({"table": 0}, "NULL"), ({"shares": 0}, "NULL"), ({"ring": 0}, "NULL"), ({"lengths": 0}, "NULL"), ({"copy_to": 0}, "NULL"),
                         ({"ring_state_out": p}, "ring_state_out"), ({"table_out": p + 16}, "table_out overlaps"), ({"lengths": p + 4}, "lengths overlaps"),
                         ({"shares_out": p + 8}, "shares_out overlaps"), ({"workspace": 0}, "workspace"), ({"workspace": o + 8}, "workspace"),
                         ({"workspace_bytes": 16}, "workspace")):
        with pytest.raises(M.MFHError, match=message):
            A.page_fork(**{**good, **bad})
    cache = dict(dtype=BF16, page_size=16, kv_heads=2, head_dim=64, pages=4)
    copy = dict(pairs=1, page_from=p, page_to=p, tokens=p, k_cache=p, v_cache=p)
    for shape, bad, message in ((dict(dtype=M.FLOAT32), {}, "f16/bf16"), (dict(head_dim=60), {}, "multiple of 8"), ({}, dict(pairs=-1), "pairs"),
                                ({}, dict(page_from=0), "NULL"), ({}, dict(page_to=0), "NULL"), ({}, dict(k_cache=0, v_cache=0), "NULL"),
                                (dict(page_size=100_000), dict(pairs=2 ** 31 - 1), "too many")):
        with pytest.raises(M.MFHError, match=message):
            A.page_copy(A.KVCache(**{**cache, **shape}), **{**copy, **bad})
    A.page_copy(A.KVCache(**cache), **{**copy, "pairs": 0, "page_from": 0})


@pytest.mark.parametrize("many", [False, True])
def test_captured_forks(many):
    # replayed with the program's own work between: each result is the eager one
    rng = np.random.default_rng(4)
    n, page, width = (1300 if many else 60), 8, 20
    before, table, shares, ring, head, tail = state(rng, n, page, width, 150, spare=n)
    d = {k: torch.from_numpy(v.copy()).cuda() for k, v in (("before", before), ("table", table), ("shares", shares), ("ring", ring),
                                                          ("state", np.array([head, tail], np.int64)))}
    parents = torch.zeros(n, dtype=torch.int32, device="cuda")
    out = {k: torch.zeros(n, dtype=torch.int32, device="cuda") for k in OUT[4:]}
    out["table_out"], out["shares_out"], out["ring_state"] = torch.full_like(d["table"], -5), torch.zeros_like(d["shares"]), torch.zeros_like(d["state"])
    need = A.page_fork_workspace(n, len(shares))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        A.page_fork(ptr(parents), ptr(d["before"]), 0, n, page, ptr(d["table"]), ptr(out["table_out"]), width, ptr(d["shares"]), ptr(out["shares_out"]),
                    len(shares), ptr(d["ring"]), len(ring), ptr(d["state"]), ptr(out["ring_state"]), ptr(out["lengths"]), ptr(out["status"]),
                    ptr(out["copy_from"]), ptr(out["copy_to"]), ptr(out["copy_tokens"]), ptr(ws), need, stream=side.cuda_stream)
    for _ in range(4):
        its = rng.integers(-5, n, n).astype(np.int32)
        parents.copy_(torch.from_numpy(its))
        d["ring"].copy_(torch.from_numpy(ring))
        out["table_out"].fill_(-5)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        out["ring"] = d["ring"]
        same({k: out[k].cpu().numpy() for k in OUT},
             fork_oracle(its, before, None, page, table, np.full_like(table, -5), width, shares, ring, head, tail))


# ---- copies -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, FP8])
@pytest.mark.parametrize("hk, dim, page, order, gap", [(8, 128, 16, "head", 0), (3, 80, 7, "token", 0), (1, 16, 1, "head", 0), (2, 256, 100, "token", 3),
                                                       (5, 48, 33, "head", 1), (1, 64, 300, "token", 0)])
def test_copies_of_pages(dtype, hk, dim, page, order, gap):
    M.init(0)
    gen = torch.Generator().manual_seed(dim + page)
    pairs, pages, row = 9, 24, dim + gap
    strides = (hk * page * row, row, page * row) if order == "head" else (hk * page * row, hk * row, row)  # page, token, head
    k, v = (torch.randint(0, 256, (pages * hk * page * row * (1 if dtype == FP8 else 2),), generator=gen, dtype=torch.uint8) for _ in range(2))
    at = torch.randperm(pages, generator=gen)
    source, target = at[9:18].clone(), at[:9].clone()
    source[3] = source[0]  # read twice
    target[4], source[5], target[6], source[6] = -1, pages, 2 ** 31 - 1, -2 ** 31  # not pages
    source[7] = target[7]
    tokens = torch.randint(0, page + 1, (pairs,), generator=gen)
    tokens[0], tokens[1], tokens[2] = -4, 10 ** 9, 0
    desc = A.KVCache(dtype, page, hk, dim, pages, page_stride=strides[0], token_stride=strides[1], head_stride=strides[2])
    kind = torch.uint8 if dtype == FP8 else torch.int16
    ints = lambda t: t.to(torch.int32).cuda()  # noqa: E731
    for whole in (False, True):
        for sides in ("kv", "k", "v"):
            want = [k.clone().view(kind), v.clone().view(kind)]
            for side, buffer in zip("kv", want):
                view = torch.as_strided(buffer, (pages, page, hk, dim), (strides[0], strides[1], strides[2], 1))
                for i in range(pairs):
                    if side in sides and 0 <= source[i] < pages and 0 <= target[i] < pages:
                        n = page if whole else min(max(int(tokens[i]), 0), page)
                        view[target[i], :n] = view[source[i], :n].clone()
            dk, dv = k.cuda(), v.cuda()
            t = [ints(source), ints(target), ints(tokens)]
            A.page_copy(desc, pairs, ptr(t[0]), ptr(t[1]), 0 if whole else ptr(t[2]), ptr(dk) if "k" in sides else 0, ptr(dv) if "v" in sides else 0,
                        stream=stream())
            torch.cuda.synchronize()
            assert torch.equal(dk.cpu().view(kind), want[0]) and torch.equal(dv.cpu().view(kind), want[1])


def test_copies_of_pages_far_apart():
    # offsets past 2^32 bytes
    M.init(0)
    stride, page, dim = 1_300_000_000, 16, 64
    k = torch.zeros(2 * stride + page * dim, dtype=torch.int16, device="cuda")
    k[2 * stride:] = torch.arange(page * dim, device="cuda", dtype=torch.int16)
    t = [torch.tensor([x], dtype=torch.int32, device="cuda") for x in (2, 1)]
    A.page_copy(A.KVCache(BF16, page, 1, dim, 3, page_stride=stride), 1, ptr(t[0]), ptr(t[1]), 0, ptr(k), 0, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(k[stride: stride + page * dim], k[2 * stride:]) and int(k[stride + page * dim:][:1000].abs().sum()) == 0
