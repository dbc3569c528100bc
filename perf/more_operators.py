"""Operators for several sequences that grow out of one, as measurable cases.

Beams, parallel answers and requests behind one long prompt, over the paged
key-value cache.  Four operators, in the order in which a beam search's step
runs them:

  shared  attention of one new token per request, where the requests of a group
          have their first tokens in common, whose keys are read once for all
  select  the best continuations of a group's beams over the vocabulary, with
          the beams' histories put in their new order
  fork    block tables in the beams' new order: whole pages are shared and
          counted, partly filled ones are listed for copying, pages that nobody
          holds any more go back
  copy    the pages that a fork listed

`run` computes each in elementary torch operations (`own` false) or by the
library's calls (`own` true).  Heads and widths are those of the 4096-wide
layers of this repository's benchmark (32 query heads of 128, 8 key-value
heads) and generic ones around them.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0
# What an FP8 cache is stored with: values are codes times these.
K_SCALE, V_SCALE = 0.0625, 0.03125


def listed():
    return [
        # one request's step of a beam search of four
        {"name": "select_step_f32", "op": "select", "groups": 1, "beams": 4, "picks": 4, "vocab": 32003, "dtype": "f32",
         "allowed": 0, "ended": False, "history": 200, "stride": 256},
        # a batch of beam searches, some beams of which have ended
        {"name": "select_batch_bf16", "op": "select", "groups": 32, "beams": 8, "picks": 8, "vocab": 131072, "dtype": "bf16",
         "allowed": 0, "ended": True, "history": 1500, "stride": 2048},
        # a grammar allows few tokens; twice as many picks as beams, from which the caller takes those that have not ended
        {"name": "select_masked_f16", "op": "select", "groups": 7, "beams": 5, "picks": 10, "vocab": 50001, "dtype": "f16",
         "allowed": 37, "ended": False, "history": 0, "stride": 0},
        # the tables of 16 searches of four beams
        {"name": "fork_beams", "op": "fork", "requests": 64, "beams": 4, "page": 16, "longest": 2000, "kind": "beams"},
        # a server's batch: requests go on, end, or begin with part of another one's prompt
        {"name": "fork_serving", "op": "fork", "requests": 1021, "beams": 8, "page": 16, "longest": 8192, "kind": "serving"},
        # the partly filled last pages of a step's beams, one layer
        {"name": "copy_beams_bf16", "op": "copy", "pairs": 64, "page": 16, "kv_heads": 8, "dim": 128, "cache": "bf16", "kind": "last"},
        # whole pages of an 8-bit cache
        {"name": "copy_pages_e4m3", "op": "copy", "pairs": 1000, "page": 64, "kv_heads": 8, "dim": 128, "cache": "e4m3", "kind": "whole"},
        # four beams over a prompt of a thousand tokens
        {"name": "shared_beams_bf16", "op": "shared", "groups": 1, "members": 4, "shared": 1008, "own": 17, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "ragged": False, "softcap": 0.0, "window": 0,
         "slopes": False},
        # groups of different sizes over prompts of different lengths in FP8, capped scores
        {"name": "shared_ragged_e4m3", "op": "shared", "groups": 24, "members": 8, "shared": 6000, "own": 300, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 32, "ragged": True, "softcap": 30.0, "window": 0,
         "slopes": False},
        # eight beams each over two very long prompts, wide heads, positions by a bias
        {"name": "shared_long_f16", "op": "shared", "groups": 2, "members": 8, "shared": 131072, "own": 200, "q_heads": 16,
         "kv_heads": 2, "dim": 256, "dtype": "f16", "cache": "f16", "page": 64, "ragged": False, "softcap": 0.0, "window": 0,
         "slopes": True},
        # a batch behind one prompt
        {"name": "shared_batch_bf16", "op": "shared", "groups": 1, "members": 64, "shared": 8192, "own": 512, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "ragged": False, "softcap": 0.0, "window": 0,
         "slopes": False},
        # a full server behind one long prompt: the matrix cores
        {"name": "shared_server_bf16", "op": "shared", "groups": 1, "members": 256, "shared": 16384, "own": 300, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "ragged": False, "softcap": 0.0, "window": 0,
         "slopes": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["select", "fork", "copy", "shared", "shared"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 31])
        groups = _log(rng, 1, 256 // beams)
        vocab = _log(rng, 17, min(262144, (1 << 25) // (groups * beams)))
        history = rng.choice([0, _log(rng, 1, 2000)])
        return {"op": op, "groups": groups, "beams": beams, "picks": beams * rng.choice([1, 1, 2]), "vocab": vocab,
                "dtype": rng.choice(["f32", "f16", "bf16"]) if groups * beams * vocab <= 1 << 24 else rng.choice(["f16", "bf16"]),
                "allowed": rng.choice([0, 0, _log(rng, 1, vocab)]), "ended": rng.random() < 0.4, "history": history,
                "stride": history + rng.randint(1, 50) if history else 0}
    if op == "fork":
        requests = _log(rng, 1, 1021)
        return {"op": op, "requests": requests, "beams": rng.choice([1, 2, 3, 4, 5, 8, 16]), "page": page,
                "longest": _log(rng, 1, 8192 * 1021 // requests * page // 16 if requests > 500 else 8192),
                "kind": rng.choice(["beams", "serving"])}
    cache = rng.choice(["f16", "bf16", "e4m3"])
    dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if op == "copy":
        most = 1000 * 65536 // (page * kv_heads * dim * BYTES[cache])
        return {"op": op, "pairs": _log(rng, 1, min(1000, most)), "page": page, "kv_heads": kv_heads, "dim": dim, "cache": cache,
                "kind": rng.choice(["last", "whole"])}
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8, 16])
    groups = _log(rng, 1, 48)
    members = _log(rng, 1, 256 // groups)
    n = groups * members
    shared = _log(rng, 1, min(131072, (1 << 27) // (groups * kv_heads * dim), (1 << 36) // (4 * n * q_heads * dim)))
    dtype = rng.choice(["bf16", "f16"])
    return {"op": op, "groups": groups, "members": members, "shared": shared, "own": _log(rng, 1, min(1000, (1 << 26) // (n * kv_heads * dim))),
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache if cache == "e4m3" else dtype, "page": page,
            "ragged": rng.random() < 0.6, "softcap": rng.choice([0.0, 0.0, 30.0]), "window": rng.choice([0, 0, 0, _log(rng, 1, shared)]),
            "slopes": rng.random() < 0.3}


# ---- sizes: from the case alone, so that `work` knows them --------------------------------

def _uniform(case, n, salt=0):
    gen = torch.Generator().manual_seed(salt + sum(v * (i + 3) for i, v in enumerate(v for v in case.values() if isinstance(v, int))))
    return torch.rand(n, generator=gen, dtype=torch.float64)


def _pages_of(lengths, page):
    return (lengths + page - 1) // page


def _fork_rows(case):
    """Per row: the tokens it has, how many leading whole pages it shares with its group's first row, and that row."""
    n, beams, page = case["requests"], case["beams"], case["page"]
    r = torch.arange(n)
    first = r // beams * beams
    before = (_uniform(case, n)[first] * case["longest"]).long() + 1
    if case["kind"] == "serving":
        before[r % 16 == 15] = 0  # rows that wait for a request
    common = torch.minimum((_uniform(case, n, 1) * 1.3).clamp_max(1.0) * (before // page), before[first] // page).long()
    return before, common, first


def _copy_tokens(case):
    if case["kind"] == "whole":
        return torch.full((case["pairs"],), case["page"])
    return (_uniform(case, case["pairs"]) * case["page"]).long()  # none, too


def _shared_rows(case):
    """Per group: members and shared tokens; per request: its group and length."""
    groups, members, shared, most = case["groups"], case["members"], case["shared"], case["own"]
    count, common = torch.full((groups,), members), torch.full((groups,), shared)
    if case["ragged"]:
        count = (_uniform(case, groups, 1) * members).long() + 1
        common = torch.exp(_uniform(case, groups, 2) * math.log(shared)).round().long()
        common[-1] = shared
    group = torch.repeat_interleave(torch.arange(groups), count)
    length = common[group] + (_uniform(case, len(group), 3) * most).long() + 1
    if case["ragged"] and len(group) > 2:
        length[1] = 0  # a beam that has ended
    return count, common, group, length


# ---- inputs -----------------------------------------------------------------------------

def _normal(gen, shape, dtype, std=1.0):
    if dtype == torch.float8_e4m3fn:
        return _normal(gen, shape, torch.bfloat16, std).clamp_(-E4M3_MAX, E4M3_MAX).to(dtype)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _int(values):
    return values.to(torch.int32).cuda()


def _scales(case):
    return (K_SCALE, V_SCALE) if case["cache"] == "e4m3" else (1.0, 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    {"select": _prepare_select, "fork": _prepare_fork, "copy": _prepare_copy, "shared": _prepare_shared}[case["op"]](case, gen, s)
    if own:
        _handles(case, s)
    return s


def _prepare_select(case, gen, s):
    groups, beams, vocab, picks = case["groups"], case["beams"], case["vocab"], case["picks"]
    rows = groups * beams
    s["logits"] = _normal(gen, (rows, vocab), TORCH[case["dtype"]], 2.5)
    if case["allowed"]:
        keep = torch.randint(0, vocab, (groups, case["allowed"]), generator=gen, device="cuda")
        mask = torch.ones(groups, vocab, dtype=torch.bool, device="cuda").scatter_(1, keep, False)
        s["logits"].view(groups, beams, vocab).masked_fill_(mask[:, None], -math.inf)
    s["scores"] = -_normal(gen, (rows,), torch.float32, 3.0).abs()
    s["ended"], s["end_token"] = None, -1
    if case["ended"]:
        s["ended"] = (torch.rand(rows, generator=gen, device="cuda") < 0.25).to(torch.uint8)
        s["end_token"] = 2
    n = groups * picks
    s["scores_out"] = torch.empty(n, device="cuda")
    s["tokens"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["parents"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["ended_out"] = torch.empty(n, dtype=torch.uint8, device="cuda") if case["ended"] else None
    s["history"] = s["history_out"] = s["known"] = None
    if case["history"]:
        s["history"] = torch.randint(0, vocab, (rows, case["stride"]), generator=gen, device="cuda", dtype=torch.int32)
        s["history_out"] = torch.zeros(n, case["stride"], dtype=torch.int32, device="cuda")
        s["known"] = torch.randint(0, case["history"] + 1, (groups,), generator=gen, device="cuda", dtype=torch.int32)


def _prepare_fork(case, gen, s):
    n, beams, page = case["requests"], case["beams"], case["page"]
    before, common, first = _fork_rows(case)
    have = _pages_of(before, page)
    width = int(have.max()) + 1
    col = torch.arange(width)[None, :]
    rows = torch.arange(n)
    alone = (col < have[:, None]) & ((col >= common[:, None]) | (rows == first)[:, None])
    held = int(alone.sum())
    pages = held + n + held // 8 + 7
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    number = torch.where(alone, alone.flatten().cumsum(0).view(n, width) - 1, 0).cuda()
    table = torch.where(alone.cuda(), order[number], -1)
    like_first = ((col < have[:, None]) & ~alone).cuda()
    s["table"] = torch.where(like_first, table[first.cuda()], table).contiguous()
    s["shares"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
    s["shares"].scatter_add_(0, s["table"][s["table"] >= 0].long(), torch.ones((), dtype=torch.int32, device="cuda").expand(int(have.sum())))
    s["shares"] = (s["shares"] - 1).clamp_min(0)
    s["before"] = _int(before)
    u = torch.rand(n, generator=gen, device="cuda")
    r, sibling = rows.cuda(), first.cuda() + torch.randint(0, beams, (n,), generator=gen, device="cuda")
    sibling = sibling.clamp_max(n - 1)
    if case["kind"] == "beams":
        s["parents"], s["keep"] = sibling.to(torch.int32), None
    else:
        # most go on, some are forked, some begin with part of another request's tokens, some end
        other = torch.randint(0, n, (n,), generator=gen, device="cuda")
        s["parents"] = torch.where(u < 0.6, r, torch.where(u < 0.75, sibling, torch.where(u < 0.85, other, -1))).to(torch.int32)
        cut = (torch.rand(n, generator=gen, device="cuda") * (case["longest"] + 1)).to(torch.int32)
        s["keep"] = torch.where((u >= 0.75) & (u < 0.85), cut, 1 << 30).to(torch.int32)
    free = pages - held
    head = int(torch.randint(0, 4 * pages, (1,), generator=gen, device="cuda"))
    s["ring"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    s["ring"][(head + torch.arange(free, device="cuda")) % pages] = order[held:]
    s["ring_state"] = torch.tensor([head, head + free], dtype=torch.int64, device="cuda")
    s["table_out"] = torch.full_like(s["table"], -1)
    s["shares_out"], s["ring_state_out"] = torch.empty_like(s["shares"]), torch.empty_like(s["ring_state"])
    for name in ("lengths", "status", "copy_from", "copy_to", "copy_tokens"):
        s[name] = torch.empty(n, dtype=torch.int32, device="cuda")


def _prepare_copy(case, gen, s):
    n = case["pairs"]
    tokens = _copy_tokens(case)
    pages = 2 * n + 3
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    s["pages"] = pages
    s["k_cache"], s["v_cache"] = (_normal(gen, shape, TORCH[case["cache"]], 100.0 if case["cache"] == "e4m3" else 1.0) for _ in range(2))
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    # several children of one beam: a page is copied more than once
    source = order[n: n + (n + 1) // 2][torch.randint(0, (n + 1) // 2, (n,), generator=gen, device="cuda")] if case["kind"] == "last" else order[n: 2 * n]
    some = torch.tensor([True] * n if case["kind"] == "whole" else [i % 4 != 3 for i in range(n)], device="cuda")
    s["from"] = torch.where(some, source, -1).to(torch.int32)
    s["to"] = torch.where(some, order[:n], -1).to(torch.int32)
    s["tokens"] = _int(tokens)
    s["spare"] = order[2 * n].long()


def _prepare_shared(case, gen, s):
    count, common, group, length = _shared_rows(case)
    page, n = case["page"], len(group)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)])
    have = _pages_of(length, page)
    width = int(have.max())
    # what the first of a group holds in front, the others have in their tables too
    ahead = _pages_of(common, page)[group].clamp_max(width)
    leader = starts[group]
    have[leader] = torch.maximum(have[leader], ahead[leader])
    col = torch.arange(width)[None, :]
    alike = (col < (common // page)[group][:, None]) & (torch.arange(n) != leader)[:, None]
    alone = (col < have[:, None]) & ~alike
    pages = int(alone.sum()) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    number = torch.where(alone, alone.flatten().cumsum(0).view(n, width) - 1, 0).cuda()
    table = torch.where(alone.cuda(), order[number], -1)
    s["table"] = torch.where((alike & (col < have[:, None])).cuda(), table[leader.cuda()], table).to(torch.int32).contiguous()
    s["pages"], s["requests"], s["members"] = pages, n, int(count.max())
    s["most_shared"], s["most_own"] = int(common.max()), int((length - common[group]).max())
    fp8 = case["cache"] == "e4m3"
    shape = (pages, case["kv_heads"], page, case["dim"])
    s["k_cache"] = _normal(gen, shape, TORCH[case["cache"]], 1 / K_SCALE if fp8 else 1.0)
    s["v_cache"] = _normal(gen, shape, TORCH[case["cache"]], 1 / V_SCALE if fp8 else 1.0)
    s["starts"], s["shared"], s["lengths"] = _int(starts), _int(common), _int(length)
    s["q"] = _normal(gen, (n, case["q_heads"], case["dim"]), TORCH[case["dtype"]], 1.5)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((n, case["q_heads"]), dtype=torch.float32, device="cuda")
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    h = torch.arange(1, case["q_heads"] + 1, dtype=torch.float32, device="cuda")
    s["slopes"] = torch.exp2(-8.0 * h / case["q_heads"]) if case["slopes"] else None


# ---- the library's calls ------------------------------------------------------------------

def _handles(case, s):
    """What a program keeps between the library's calls: descriptors and a workspace."""
    import manifesto_amd as M
    from manifesto_amd import attention as A, beams as B
    M.init(torch.cuda.current_device())
    code = {"f32": M.FLOAT32, "f16": M.FLOAT16, "bf16": M.BFLOAT16, "e4m3": M.F8E4M3}
    s["A"], s["B"] = A, B
    need = 0
    if case["op"] == "select":
        s["shape"] = B.Beams(code[case["dtype"]], case["beams"], case["picks"], case["vocab"], end_token=s["end_token"],
                             history_stride=case["stride"])
        need = B.beam_select_workspace(s["shape"], case["groups"])
    elif case["op"] == "fork":
        need = A.page_fork_workspace(case["requests"], s["shares"].numel())
    else:
        k_scale, v_scale = _scales(case)
        s["cache"] = A.KVCache(code[case["cache"]], case["page"], case["kv_heads"], case["dim"], s["pages"],
                               k_scale=k_scale, v_scale=v_scale)
    if case["op"] == "shared":
        s["attention"] = A.Attention(code[case["dtype"]], case["q_heads"], s["scale"], softcap=case["softcap"],
                                     window=case["window"])
        need = A.paged_decode_shared_workspace(s["attention"], s["cache"], s["requests"], case["groups"], s["most_shared"],
                                               s["most_own"])
    s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def _ptr(t):
    return t.data_ptr() if t is not None else 0


def _run_own(s):
    A, B, case = s["A"], s["B"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    op = case["op"]
    if op == "select":
        B.beam_select(s["shape"], case["groups"], _ptr(s["logits"]), _ptr(s["scores"]), _ptr(s["ended"]), _ptr(s["scores_out"]),
                      _ptr(s["tokens"]), _ptr(s["parents"]), _ptr(s["ended_out"]), _ptr(s["history"]), _ptr(s["known"]),
                      _ptr(s["history_out"]), _ptr(s["workspace"]), s["workspace"].numel(), stream=stream)
        return {k: s[k] for k in ("scores_out", "tokens", "parents", "ended_out", "history_out") if s[k] is not None}
    if op == "fork":
        A.page_fork(_ptr(s["parents"]), _ptr(s["before"]), _ptr(s["keep"]), case["requests"], case["page"], _ptr(s["table"]),
                    _ptr(s["table_out"]), s["table"].shape[1], _ptr(s["shares"]), _ptr(s["shares_out"]), s["shares"].numel(),
                    _ptr(s["ring"]), s["ring"].numel(), _ptr(s["ring_state"]), _ptr(s["ring_state_out"]), _ptr(s["lengths"]),
                    _ptr(s["status"]), _ptr(s["copy_from"]), _ptr(s["copy_to"]), _ptr(s["copy_tokens"]), _ptr(s["workspace"]),
                    s["workspace"].numel(), stream=stream)
        return {k: s[k] for k in ("table_out", "shares_out", "ring", "ring_state_out", "lengths", "status", "copy_from", "copy_to", "copy_tokens")}
    if op == "copy":
        A.page_copy(s["cache"], case["pairs"], _ptr(s["from"]), _ptr(s["to"]), _ptr(s["tokens"]), _ptr(s["k_cache"]),
                    _ptr(s["v_cache"]), stream=stream)
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    A.paged_decode_shared(s["attention"], s["cache"], s["requests"], case["groups"], _ptr(s["q"]), _ptr(s["k_cache"]), _ptr(s["v_cache"]),
                          _ptr(s["table"]), s["table"].shape[1], _ptr(s["starts"]), _ptr(s["shared"]), s["most_shared"],
                          _ptr(s["lengths"]), s["most_own"], _ptr(s["slopes"]), _ptr(s["out"]), _ptr(s["lse"]),
                          _ptr(s["workspace"]), s["workspace"].numel(), stream=stream)
    return {"out": s["out"], "lse": s["lse"]}


# ---- the plain forms ------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"select": _plain_select, "fork": _plain_fork, "copy": _plain_copy, "shared": _plain_shared}[s["case"]["op"]](s)


def _plain_select(s):
    """Candidates are ordered by score; those of equal score by beam, and those of one beam by logit and token.  In 64
    bits, for two beams' candidates may lie next to each other."""
    case = s["case"]
    groups, beams, vocab, picks = case["groups"], case["beams"], case["vocab"], case["picks"]
    x = s["logits"].float() + 0.0
    top = x.amax(-1, keepdim=True)
    z = top.double() + torch.exp(x.double() - torch.where(top == -math.inf, 0.0, top).double()).sum(-1, keepdim=True).log()
    # a row's largest, equal ones in their order: logits as whole numbers in front of the tokens counted down
    bits = x.view(torch.int32)
    key = (torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32) + (vocab - 1 - torch.arange(vocab, device="cuda"))
    most = min(picks, vocab)
    token = vocab - 1 - (torch.topk(key, most, dim=-1).values & 0xffffffff)
    before = s["scores"].double()[:, None]
    score = before + (x.gather(-1, token).double() - z)
    score = torch.where(torch.isnan(score), -math.inf, score)
    if case["ended"]:
        only = torch.cat([before, torch.full_like(score[:, 1:], -math.inf)], -1)
        score = torch.where(s["ended"][:, None] != 0, only, score)
        token = torch.where(s["ended"][:, None] != 0, s["end_token"], token)
    score, token = score.view(groups, -1), token.view(groups, -1)
    if score.shape[1] < picks:
        extra = picks - score.shape[1]
        score, token = torch.nn.functional.pad(score, (0, extra), value=-math.inf), torch.nn.functional.pad(token, (0, extra))
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    best, at = best[:, :picks], at[:, :picks]
    there = best > -math.inf
    token = torch.where(there, token.gather(1, at), -1)
    parent = torch.where(there, torch.arange(groups, device="cuda")[:, None] * beams + at // most, -1)
    out = {"scores_out": best.reshape(-1).float(), "tokens": token.reshape(-1).to(torch.int32), "parents": parent.reshape(-1).to(torch.int32)}
    if case["ended"]:
        done = (s["ended"][parent.clamp_min(0)] != 0) | (token == s["end_token"])
        out["ended_out"] = (done & there).reshape(-1).to(torch.uint8)
    if case["history"]:
        known = s["known"].long().repeat_interleave(picks)[:, None]
        col = torch.arange(case["stride"], device="cuda")
        rows = torch.where(col < known, s["history"][parent.reshape(-1).clamp_min(0)],
                           torch.where(col == known, out["tokens"][:, None], 0))
        out["history_out"] = torch.where(out["parents"][:, None] >= 0, rows, 0).to(torch.int32)
    return out


def _plain_fork(s):
    """Row r becomes the first `keep` tokens of its parent.  Of the rows that reach into their parent's partly filled last
    page the first keeps it; every other partly filled page is a copy, in a page from the ring's head.  A row for whose copy
    no page is left becomes empty.  Pages that no row holds any more go to the ring's tail in the order of their numbers."""
    case, page, n = s["case"], s["case"]["page"], s["case"]["requests"]
    width, pages, size = s["table"].shape[1], s["shares"].numel(), s["ring"].numel()
    r = torch.arange(n, device="cuda")
    b, p = s["before"].long(), s["parents"].long()
    odd = (b < 0) | (b > width * page)
    bad = (p >= n) | ((p >= 0) & odd[p.clamp(0, n - 1)])
    none = bad | (p < 0)
    p = torch.where(none, 0, p)
    take = torch.where(none, 0, b[p] if s["keep"] is None else torch.minimum(s["keep"].long(), b[p]).clamp_min(0))
    part, row = take % page, take // page
    reaches = (part > 0) & (row == b[p] // page)
    first = torch.full((n,), n, device="cuda").scatter_reduce_(0, p, torch.where(reaches, r, n), "amin")
    need = (part > 0) & (first[p] != r)
    head, tail = s["ring_state"][0], s["ring_state"][1]
    refused = need & (need.cumsum(0) > tail - head)
    granted = need & ~refused
    take = torch.where(refused, 0, take)
    fresh = s["ring"][(head + granted.cumsum(0) - 1).clamp_min(0) % size]
    col = torch.arange(width, device="cuda")[None, :]
    holds = col < _pages_of(take, page)[:, None]
    copied = holds & granted[:, None] & (col == row[:, None])
    table = torch.where(holds, torch.where(copied, fresh[:, None], s["table"][p]), -1)
    # holders: those of the old rows less, those of the new rows more
    held = col < torch.where(odd, 0, _pages_of(b, page))[:, None]
    change = torch.zeros(pages, dtype=torch.int32, device="cuda")
    for mask, numbers, by in ((held, s["table"], -1), (holds & ~copied, table, 1)):
        inside = mask & (numbers >= 0) & (numbers < pages)
        change.scatter_add_(0, torch.where(inside, numbers, 0).long().flatten(), torch.where(inside, by, 0).to(torch.int32).flatten())
    shares = s["shares"].clamp_min(0) + change
    free = shares < 0
    at = torch.where(free, (tail + free.cumsum(0) - 1) % size, size)  # past the end: nowhere
    ring = torch.cat([s["ring"], s["ring"][:1]])
    ring[at] = torch.arange(pages, device="cuda", dtype=torch.int32)
    narrow = lambda t: t.to(torch.int32)  # noqa: E731
    return {"table_out": narrow(table), "shares_out": shares.clamp_min(0), "ring": ring[:size],
            "ring_state_out": torch.stack([head + granted.sum(), tail + free.sum()]), "lengths": narrow(take),
            "status": narrow(torch.where(bad, 2, torch.where(refused, 1, 0))),
            "copy_from": narrow(torch.where(granted, s["table"][p, row.clamp_max(width - 1)], -1)),
            "copy_to": narrow(torch.where(granted, fresh, -1)), "copy_tokens": narrow(torch.where(granted, part, 0))}


def _plain_copy(s):
    case, n = s["case"], s["case"]["pairs"]
    row = torch.arange(case["page"], device="cuda")[None, :].expand(n, -1)
    inside = (row < s["tokens"][:, None]) & (s["from"] >= 0)[:, None]
    # what is not copied: a spare page's rows onto themselves
    source, target = (torch.where(inside, s[name].long()[:, None], s["spare"]) for name in ("from", "to"))
    out = {}
    for name in ("k_cache", "v_cache"):
        cache = s[name].view(torch.uint8) if case["cache"] == "e4m3" else s[name]
        cache[target, :, row] = cache[source, :, row]
        out[name] = s[name]
    return out


def _plain_shared(s):
    """Scores over the shared tokens for all members of a group at once, over their own request by request, one softmax."""
    case = s["case"]
    hk, hq, dim, page, n = case["kv_heads"], case["q_heads"], case["dim"], case["page"], s["requests"]
    gh, k_scale, v_scale = hq // hk, *_scales(case)
    starts, shared, length = s["starts"].long(), s["shared"].long(), s["lengths"].long()
    group = torch.searchsorted(starts[1:].contiguous(), torch.arange(n, device="cuda"), right=True)

    def keys_values(rows, position, inside):
        """[rows, kv_heads, positions, dim] in 32 bits, zeros where there is nothing."""
        position = torch.where(inside, position, 0)
        at, token = s["table"].long()[rows[:, None], position // page], position % page
        take = lambda cache, scale: torch.where(inside[..., None, None], cache[at, :, token].float() * scale, 0.0).transpose(1, 2)  # noqa: E731
        return take(s["k_cache"], k_scale), take(s["v_cache"], v_scale)

    def weights(scores, distance, seen):
        """Of scores [..., kv_heads, group, positions], with distance and seen [..., 1, 1, positions]."""
        if case["softcap"]:
            scores = case["softcap"] * torch.tanh(scores / case["softcap"])
        if case["slopes"]:
            scores = scores - s["slopes"].view(hk, gh, 1) * distance.float()
        if case["window"]:
            seen = seen & (distance < case["window"])
        scores = torch.where(seen, scores, -math.inf)
        top = scores.amax(-1, keepdim=True)
        w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
        return top, w, w.sum(-1, keepdim=True)

    # the shared tokens: the first member's pages, queries [groups, kv_heads, members * group, dim]
    t = torch.arange(s["most_shared"], device="cuda")
    k, v = keys_values(starts[:-1], t[None, :].expand(len(shared), -1), t[None, :] < shared[:, None])
    members = s["members"]
    of = (starts[:-1, None] + torch.arange(members, device="cuda")).clamp_max(n - 1)
    q = s["q"].float().view(n, hk, gh, dim)
    x = torch.matmul(q[of].permute(0, 2, 1, 3, 4).reshape(len(shared), hk, -1, dim), k.transpose(-1, -2)) * s["scale"]
    x = x.view(len(shared), hk, members, gh, -1).transpose(1, 2)
    distance = (length[of][..., None] - 1 - t)[:, :, None, None]
    top, w, total = weights(x, distance, (distance >= 0) & (t < shared[:, None])[:, None, None, None])
    o = torch.matmul(w.transpose(1, 2).reshape(len(shared), hk, members * gh, -1), v).view(len(shared), hk, members, gh, dim).transpose(1, 2)
    member = torch.arange(n, device="cuda") - starts[group]
    top, total, o = (y[group, member] for y in (top, total, o))
    # each request's own
    u = torch.arange(s["most_own"], device="cuda")
    position = shared[group][:, None] + u
    k, v = keys_values(torch.arange(n, device="cuda"), position, position < length[:, None])
    x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    distance = (length[:, None] - 1 - position)[:, None, None]
    top2, w, total2 = weights(x, distance, distance >= 0)
    o2 = torch.matmul(w, v)
    # both together
    both = torch.maximum(top, top2)
    at = torch.where(both == -math.inf, 0.0, both)
    f, f2 = torch.exp(top - at), torch.exp(top2 - at)
    total = total * f + total2 * f2
    out = (o * f + o2 * f2) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(n, hq, dim).to(TORCH[case["dtype"]]), "lse": (both + torch.log(total)).reshape(n, hq)}


# ---- what cannot be done without ------------------------------------------------------------

def work(case):
    if case["op"] == "select":
        rows, n = case["groups"] * case["beams"], case["groups"] * case["picks"]
        size = rows * case["vocab"]
        # on the average half of the longest history, read and written
        return {"bytes": size * BYTES[case["dtype"]] + 5 * rows + 13 * n + 4 * n * case["history"], "flops": 4 * size}
    if case["op"] == "fork":
        before, common, first = _fork_rows(case)
        have = _pages_of(before, case["page"])
        alone = torch.where(torch.arange(case["requests"]) == first, have, (have - common).clamp_min(0))
        # the tables' entries read and written, every page's count too, and what is there once per row
        return {"bytes": 8 * int(have.sum()) + 8 * int(alone.sum()) + 32 * case["requests"], "flops": 0}
    if case["op"] == "copy":
        tokens = _copy_tokens(case)
        if case["kind"] == "last":
            tokens = tokens[torch.arange(case["pairs"]) % 4 != 3]
        return {"bytes": 4 * int(tokens.sum()) * case["kv_heads"] * case["dim"] * BYTES[case["cache"]] + 12 * case["pairs"], "flops": 0}
    count, common, group, length = _shared_rows(case)
    dim, hq, hk, w = case["dim"], case["q_heads"], case["kv_heads"], case["window"]
    first = (length - w).clamp_min(0) if w else torch.zeros_like(length)  # of the tokens that a request sees
    pairs = int((length - first).sum())
    mine = (length - torch.maximum(first, common[group])).clamp_min(0)
    keys = int(mine.sum())
    end = torch.minimum(length, common[group])
    for g in range(case["groups"]):
        sees = (group == g) & (end > first)
        if bool(sees.any()):
            keys += int(end[sees].max() - first[sees].min())
    n = len(group)
    return {"bytes": 2 * keys * hk * dim * BYTES[case["cache"]] + 2 * n * hq * dim * BYTES[case["dtype"]] + 4 * n * hq,
            "flops": 4 * pairs * hq * dim}


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "select":
        return _exact_select(case, prepare(case, seed))
    if case["op"] == "shared":
        return _exact_shared(case, prepare(case, seed))
    if case["op"] == "copy":
        return _exact_copy(case, prepare(case, seed))
    return None  # whole numbers: the plain form is exact


def _exact_copy(case, s):
    """Pair by pair."""
    out = {}
    for name in ("k_cache", "v_cache"):
        cache = s[name].double()
        for source, target, tokens in zip(s["from"].tolist(), s["to"].tolist(), s["tokens"].tolist()):
            if source >= 0:
                cache[target, :, :tokens] = s[name][source, :, :tokens].double()
        out[name] = cache
    return out


def _exact_select(case, s):
    """The scores; the other results are whole numbers."""
    rows = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[:, None]
    if case["ended"]:
        rows[s["ended"] != 0] = -math.inf
        rows[:, s["end_token"]] = torch.where(s["ended"] != 0, s["scores"].double(), rows[:, s["end_token"]])
    rows = rows.view(case["groups"], -1)
    best = torch.full((case["groups"], case["picks"]), -math.inf, dtype=torch.float64, device="cuda")
    n = min(case["picks"], rows.shape[1])
    best[:, :n] = torch.topk(rows, n, dim=-1).values
    out = {"scores_out": best.reshape(-1), "tokens": None, "parents": None}
    if case["ended"]:
        out["ended_out"] = None
    if case["history"]:
        out["history_out"] = None
    return out


def _exact_shared(case, s):
    """Request by request and head by head."""
    hk, group, dim, page = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"], case["page"]
    starts, shared, lengths = s["starts"].tolist(), s["shared"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    k_scale, v_scale = _scales(case)
    for g in range(case["groups"]):
        for r in range(starts[g], starts[g + 1]):
            length, common = lengths[r], min(shared[g], lengths[r])
            first = max(0, length - case["window"]) if case["window"] else 0
            t = torch.arange(first, length, device="cuda")
            if not len(t):
                continue
            row = torch.where(t < common, starts[g], r)
            at = s["table"][row, t // page].long()
            for h in range(hk):
                k = s["k_cache"][at, h, t % page].double() * k_scale
                v = s["v_cache"][at, h, t % page].double() * v_scale
                heads = slice(h * group, (h + 1) * group)
                x = s["q"][r, heads].double() @ k.T * s["scale"]
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if case["slopes"]:
                    x = x - s["slopes"][heads, None].double() * (length - 1 - t)
                z = torch.logsumexp(x, -1)
                lse[r, heads] = z
                out[r, heads] = torch.exp(x - z[:, None]) @ v
    return {"out": out, "lse": lse}
