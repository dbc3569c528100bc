"""Serving operators over a paged key-value cache, as measurable cases.

Four operators that a decoder's step is made of, in the order in which a step
runs them:

  pages    block tables and slot maps from the requests' lengths
  rotary   rotary positions of queries and keys, keys and values written to
           their pages (or, without pages, the rotation and its gradient)
  decode   attention of one new token per request over its pages
  prefill  attention of each request's new tokens over its pages, its own
           tokens among them

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
BASE = 10000.0
E4M3_MAX = 448.0
# What an FP8 cache is stored with: values are codes times these.
K_SCALE, V_SCALE = 0.0625, 0.03125


def listed():
    return [
        # one decode step of a small batch: every request gets one token
        {"name": "pages_step", "op": "pages", "requests": 64, "page": 16, "width": 512, "kind": "step", "longest": 8000},
        # a scheduler's large step: prompts of up to 1024 tokens beside decodes, requests that end and return their pages
        {"name": "pages_prompts", "op": "pages", "requests": 1021, "page": 16, "width": 640, "kind": "mixed", "longest": 1024},
        # a decode step's queries and keys, bf16 cache
        {"name": "rotary_step_bf16", "op": "rotary", "tokens": 8, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "dtype": "bf16", "cache": "bf16", "page": 16, "interleaved": False, "inverse": False, "longest": 8192},
        # a long prompt into an FP8 cache, adjacent pairs in half of the head
        {"name": "rotary_prompt_e4m3", "op": "rotary", "tokens": 16381, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "dtype": "bf16", "cache": "e4m3", "page": 32, "interleaved": True, "inverse": False, "longest": 131072},
        # the rotation's gradient in training, f32, no cache
        {"name": "rotary_gradient_f32", "op": "rotary", "tokens": 4095, "q_heads": 32, "kv_heads": 32, "dim": 96, "rot": 96,
         "dtype": "f32", "cache": "", "page": 0, "interleaved": False, "inverse": True, "longest": 4096},
        # one user, a short context: latency alone
        {"name": "decode_one_bf16", "op": "decode", "requests": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "cache": "bf16", "page": 16, "longest": 1021, "ragged": False, "softcap": 0.0, "window": 0, "slopes": False},
        # a batch of very different lengths, one of them empty, FP8 cache, capped scores
        {"name": "decode_ragged_e4m3", "op": "decode", "requests": 48, "q_heads": 32, "kv_heads": 4, "dim": 128, "dtype": "bf16",
         "cache": "e4m3", "page": 32, "longest": 16384, "ragged": True, "softcap": 30.0, "window": 0, "slopes": False},
        # two users with very long contexts, wide heads, distance bias
        {"name": "decode_long_f16", "op": "decode", "requests": 2, "q_heads": 16, "kv_heads": 2, "dim": 256, "dtype": "f16",
         "cache": "f16", "page": 64, "longest": 131071, "ragged": False, "softcap": 0.0, "window": 0, "slopes": True},
        # a full batch: the bandwidth of the card
        {"name": "decode_batch_bf16", "op": "decode", "requests": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "cache": "bf16", "page": 16, "longest": 8192, "ragged": False, "softcap": 0.0, "window": 0, "slopes": False},
        # short prompts of several users, narrow heads, distance bias
        {"name": "prefill_short_f16", "op": "prefill", "requests": 5, "fresh": 161, "past": 0, "q_heads": 12, "kv_heads": 12,
         "dim": 64, "dtype": "f16", "cache": "f16", "page": 16, "ragged": True, "softcap": 0.0, "window": 0, "slopes": True,
         "prefix": False},
        # one long prompt: the matrix cores
        {"name": "prefill_prompt_bf16", "op": "prefill", "requests": 1, "fresh": 8192, "past": 0, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "ragged": False, "softcap": 0.0, "window": 0,
         "slopes": False, "prefix": False},
        # chunks of prompts over what is cached of them in FP8, a prefix that every token sees, capped scores
        {"name": "prefill_chunk_e4m3", "op": "prefill", "requests": 4, "fresh": 512, "past": 7000, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 32, "ragged": True, "softcap": 30.0, "window": 0,
         "slopes": False, "prefix": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 6, 8, 16]), kv


def draw(rng):
    op = rng.choice(["pages", "rotary", "decode", "prefill"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128, 256])
    if op == "pages":
        page, requests = max(page, 8), _log(rng, 1, 1021)
        longest = _log(rng, 1, min(8000, 522752 // requests))
        return {"op": op, "requests": requests, "page": page, "width": (2 * longest + 600) // page + 2,
                "kind": rng.choice(["step", "mixed"]), "longest": longest}
    dtype = rng.choice(["bf16", "f16"])
    cache = rng.choice([dtype, dtype, "e4m3"])
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256])
    if op == "rotary":
        paged = rng.random() < 0.6
        if not paged:
            dtype, cache = rng.choice(["bf16", "f16", "f32"]), ""
        tokens = _log(rng, 1, 16381 * 5120 // ((q_heads + 2 * kv_heads) * dim * (2 if dtype == "f32" else 1)))
        return {"op": op, "tokens": min(tokens, 32768), "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2]), "dtype": dtype, "cache": cache,
                "page": page if paged else 0, "interleaved": rng.random() < 0.5,
                "inverse": not paged and rng.random() < 0.5, "longest": _log(rng, 16, 1 << 20)}
    softcap = rng.choice([0.0, 0.0, 30.0])
    slopes = rng.random() < 0.3
    if op == "decode":
        requests = _log(rng, 1, 200)
        longest = _log(rng, 1, min(200000, (1 << 29) // (requests * kv_heads * dim), (1 << 28) // (requests * q_heads)))
        return {"op": op, "requests": requests, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
                "cache": cache, "page": page, "longest": longest, "ragged": rng.random() < 0.6, "softcap": softcap,
                "window": rng.choice([0, 0, _log(rng, 1, longest)]), "slopes": slopes}
    requests = _log(rng, 1, 24)
    fresh = _log(rng, 1, min(4096, 24000 // requests))
    past = rng.choice([0, _log(rng, 1, 16384)])
    most = 1 << 30  # scores of the padded batch
    past = min(past, max(0, most // (requests * q_heads * fresh) - fresh), (1 << 27) // (requests * kv_heads * dim))
    fresh = min(fresh, math.isqrt(most // (requests * q_heads)))
    return {"op": op, "requests": requests, "fresh": fresh, "past": past, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "cache": cache, "page": page, "ragged": rng.random() < 0.6, "softcap": softcap,
            "window": rng.choice([0, 0, _log(rng, 1, fresh + past)]), "slopes": slopes, "prefix": rng.random() < 0.3}


# ---- lengths: from the case alone, so that `work` knows them ----------------------------

def _spread(case):
    """Per request: (tokens cached before the call, new tokens), of the case alone."""
    n, op = case["requests"], case["op"]
    gen = torch.Generator().manual_seed(sum(v * (i + 3) for i, v in enumerate(v for v in case.values() if isinstance(v, int))))
    u = torch.rand(n, generator=gen, dtype=torch.float64)
    w = torch.rand(n, generator=gen, dtype=torch.float64)
    if op == "pages":
        longest = case["longest"]
        past = (u * longest).long()
        if case["kind"] == "step":
            return past, torch.ones(n, dtype=torch.int64)
        # of ten requests five have a new prompt, three decode, one goes back by a few tokens, one ends
        of = torch.arange(n) % 10
        fresh = torch.where(of < 5, (w * longest).long() + 1, torch.where(of < 8, 1, -torch.minimum(past, torch.tensor(5))))
        return torch.where(of < 5, 0, past), torch.where(of == 9, -past, fresh)
    if op == "decode":
        most = case["longest"]
        if not case["ragged"]:
            return torch.full((n,), most - 1), torch.ones(n, dtype=torch.int64)
        total = (torch.exp(u * math.log(most)) + 0.5).long().clamp(1, most)
        total[w.argmax()] = most
        if n > 2:
            total[w.argmin()] = 0
        return total - (total > 0).long(), (total > 0).long()
    past, fresh = case["past"], case["fresh"]
    if not case["ragged"]:
        return torch.full((n,), past), torch.full((n,), fresh)
    new = (torch.exp(u * math.log(max(fresh, 1))) + 0.5).long().clamp(1, fresh)
    new[w.argmax()] = fresh
    if n > 2:
        new[w.argmin()] = 0
    return (w * past).long(), new


def _pages_of(lengths, page):
    return (lengths + page - 1) // page


# ---- inputs -----------------------------------------------------------------------------

def _normal(gen, shape, dtype, std=1.0):
    if dtype == torch.float8_e4m3fn:
        return _normal(gen, shape, torch.bfloat16, std).clamp_(-E4M3_MAX, E4M3_MAX).to(dtype)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _int(values):
    return values.to(torch.int32).cuda()


def _cache(case, gen, pages):
    """Keys and values [pages + 1, kv_heads, page, dim]; the last page is spare and in no table."""
    shape = (pages + 1, case["kv_heads"], case["page"], case["dim"])
    fp8 = case["cache"] == "e4m3"
    return (_normal(gen, shape, TORCH[case["cache"]], 1 / K_SCALE if fp8 else 1.0),
            _normal(gen, shape, TORCH[case["cache"]], 1 / V_SCALE if fp8 else 1.0))


def _table(gen, lengths, page, pages):
    """Block tables over shuffled pages; entries past a request's pages are -1."""
    need = _pages_of(lengths, page)
    width = max(1, int(need.max()))
    order = torch.randperm(pages, generator=gen, device="cuda")
    first = (need.cumsum(0) - need).cuda()[:, None]
    col = torch.arange(width, device="cuda")[None, :]
    at = torch.where(col < need.cuda()[:, None], first + col, 0)
    return torch.where(col < need.cuda()[:, None], order[at], -1).to(torch.int32).contiguous()


def _scales(case):
    return (K_SCALE, V_SCALE) if case["cache"] == "e4m3" else (1.0, 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] == "pages":
        _prepare_pages(case, gen, s)
    elif case["op"] == "rotary":
        _prepare_rotary(case, gen, s)
    else:
        _prepare_attention(case, gen, s)
    if own:
        _handles(case, s)
    return s


def _prepare_pages(case, gen, s):
    past, fresh = _spread(case)
    page, width, n = case["page"], case["width"], case["requests"]
    after = past + fresh
    have, want = _pages_of(past, page), _pages_of(after, page)
    held, taken = int(have.sum()), int((want - have).clamp_min(0).sum())
    pages = held + taken + taken // 4 + 7
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    col = torch.arange(width)[None, :]
    at = torch.where(col < have[:, None], (have.cumsum(0) - have)[:, None] + col, 0).cuda()
    s["before"], s["after"] = _int(past), _int(after)
    s["table"] = torch.where((col < have[:, None]).cuda(), order[at], -1).to(torch.int32).contiguous()
    # the free pages in a ring that has turned a few times
    free = pages - held
    head = int(torch.randint(0, 4 * pages, (1,), generator=gen, device="cuda"))
    s["ring"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    s["ring"][(head + torch.arange(free, device="cuda")) % pages] = order[held:]
    s["ring_state"] = torch.tensor([head, head + free], dtype=torch.int64, device="cuda")
    s["tokens"] = int(fresh.clamp_min(0).sum()) + 3  # a captured step's batch is padded
    s["ring_state_out"] = torch.empty_like(s["ring_state"])
    s["slots"] = torch.empty(s["tokens"], dtype=torch.int64, device="cuda")
    s["positions"] = torch.empty(s["tokens"], dtype=torch.int32, device="cuda")
    s["starts"] = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    s["lengths"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["status"] = torch.empty(n, dtype=torch.int32, device="cuda")


def _prepare_rotary(case, gen, s):
    n, dim, dtype = case["tokens"], case["dim"], TORCH[case["dtype"]]
    hq, hk, half = case["q_heads"], case["kv_heads"], case["rot"] // 2
    s["q"] = _normal(gen, (n, hq, dim), dtype)
    s["k"] = _normal(gen, (n, hk, dim), dtype)
    s["v"] = _normal(gen, (n, hk, dim), dtype)
    s["positions"] = torch.randint(0, case["longest"], (n,), generator=gen, device="cuda", dtype=torch.int32)
    s["frequencies"] = BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(half, 1))
    s["q_out"] = torch.empty_like(s["q"])
    if not case["cache"]:
        s["k_out"] = torch.empty_like(s["k"])
        return
    pages = n // case["page"] + 5
    s["pages"] = pages
    s["k_cache"], s["v_cache"] = _cache(case, gen, pages)
    s["slots"] = torch.randperm(pages * case["page"], generator=gen, device="cuda")[:n].contiguous()
    if n > 4:
        s["slots"][n // 3] = -1  # a token that has no place


def _prepare_attention(case, gen, s):
    past, fresh = _spread(case)
    total = past + fresh
    page, n, dtype = case["page"], case["requests"], TORCH[case["dtype"]]
    pages = int(_pages_of(total, page).sum()) + 3
    s["pages"], s["fresh"], s["total"] = pages, int(fresh.sum()), int(total.max())
    s["most_fresh"] = int(fresh.max())
    s["k_cache"], s["v_cache"] = _cache(case, gen, pages)
    s["table"] = _table(gen, total, page, pages)
    s["lengths"] = _int(total)
    rows = n if case["op"] == "decode" else s["fresh"]
    s["q"] = _normal(gen, (rows, case["q_heads"], case["dim"]), dtype, 1.5)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((rows, case["q_heads"]), dtype=torch.float32, device="cuda")
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    h = torch.arange(1, case["q_heads"] + 1, dtype=torch.float32, device="cuda")
    s["slopes"] = torch.exp2(-8.0 * h / case["q_heads"]) if case["slopes"] else None
    if case["op"] == "prefill":
        s["starts"] = _int(torch.cat([torch.zeros(1, dtype=torch.int64), fresh.cumsum(0)]))
        s["prefix"] = _int(total // 3) if case["prefix"] else None


# ---- the library's calls ------------------------------------------------------------------

def _handles(case, s):
    """What a program keeps between the library's calls: descriptors and a workspace."""
    import manifesto_amd as M
    from manifesto_amd import attention as A
    M.init(torch.cuda.current_device())
    code = {"f32": M.FLOAT32, "f16": M.FLOAT16, "bf16": M.BFLOAT16, "e4m3": M.F8E4M3}
    s["A"] = A
    if case["op"] == "pages":
        return
    if case["cache"]:
        k_scale, v_scale = _scales(case)
        s["cache"] = A.KVCache(code[case["cache"]], case["page"], case["kv_heads"], case["dim"], s["pages"],
                               k_scale=k_scale, v_scale=v_scale)
    if case["op"] == "rotary":
        s["rotary"] = A.Rotary(code[case["dtype"]], case["q_heads"], case["kv_heads"], case["dim"], case["rot"],
                               interleaved=case["interleaved"], inverse=case["inverse"])
        return
    s["attention"] = A.Attention(code[case["dtype"]], case["q_heads"], s["scale"], softcap=case["softcap"],
                                 window=case["window"])
    if case["op"] == "decode":
        need = A.paged_decode_workspace(s["attention"], s["cache"], case["requests"], s["total"])
    else:
        need = A.paged_prefill_workspace(s["attention"], s["cache"], case["requests"], s["fresh"], s["most_fresh"], s["total"])
    s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def _ptr(t):
    return t.data_ptr() if t is not None else 0


def _run_own(s):
    A, case = s["A"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    op = case["op"]
    if op == "pages":
        A.page_plan(_ptr(s["before"]), _ptr(s["after"]), case["requests"], case["page"], _ptr(s["table"]), case["width"],
                    _ptr(s["ring"]), s["ring"].numel(), _ptr(s["ring_state"]), _ptr(s["ring_state_out"]),
                    _ptr(s["slots"]), _ptr(s["positions"]), s["tokens"], _ptr(s["starts"]), _ptr(s["lengths"]),
                    _ptr(s["status"]), stream=stream)
        return {k: s[k] for k in ("table", "ring", "ring_state_out", "slots", "positions", "starts", "lengths", "status")}
    if op == "rotary":
        if not case["cache"]:
            A.rotary(s["rotary"], case["tokens"], _ptr(s["q"]), _ptr(s["q_out"]), _ptr(s["k"]), _ptr(s["k_out"]),
                     _ptr(s["positions"]), _ptr(s["frequencies"]), stream=stream)
            return {"q": s["q_out"], "k": s["k_out"]}
        A.rotary_append(s["rotary"], s["cache"], case["tokens"], _ptr(s["q"]), _ptr(s["q_out"]), _ptr(s["k"]), _ptr(s["v"]),
                        _ptr(s["positions"]), _ptr(s["slots"]), _ptr(s["frequencies"]), _ptr(s["k_cache"]),
                        _ptr(s["v_cache"]), stream=stream)
        return {"q": s["q_out"], "k_cache": s["k_cache"][:-1], "v_cache": s["v_cache"][:-1]}
    if op == "decode":
        A.paged_decode(s["attention"], s["cache"], case["requests"], _ptr(s["q"]), _ptr(s["k_cache"]), _ptr(s["v_cache"]),
                       _ptr(s["table"]), s["table"].shape[1], _ptr(s["lengths"]), s["total"], _ptr(s["slopes"]),
                       _ptr(s["out"]), _ptr(s["lse"]), _ptr(s["workspace"]), s["workspace"].numel(), stream=stream)
    else:
        A.paged_prefill(s["attention"], s["cache"], case["requests"], s["fresh"], s["most_fresh"], _ptr(s["q"]),
                        _ptr(s["k_cache"]), _ptr(s["v_cache"]), _ptr(s["table"]), s["table"].shape[1], _ptr(s["starts"]),
                        _ptr(s["lengths"]), s["total"], _ptr(s["prefix"]), _ptr(s["slopes"]), _ptr(s["out"]),
                        _ptr(s["lse"]), _ptr(s["workspace"]), s["workspace"].numel(), stream=stream)
    return {"out": s["out"], "lse": s["lse"]}


# ---- the plain forms ------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"pages": _plain_pages, "rotary": _plain_rotary, "decode": _plain_decode, "prefill": _plain_prefill}[s["case"]["op"]](s)


def _plain_pages(s):
    """A request grows from `before` to `after` tokens, or shrinks.  New pages come from the ring's head in the
    requests' order, returned ones go to its tail.  A request whose table row or whose tokens do not fit, or
    for which no pages are left, keeps its length, and its tokens get the slot -1."""
    case, page, width, n, tokens = s["case"], s["case"]["page"], s["case"]["width"], s["case"]["requests"], s["tokens"]
    b, a = s["before"].long().clamp_min(0), s["after"].long().clamp_min(0)
    have, want = (b + page - 1) // page, (a + page - 1) // page
    fresh = (a - b).clamp_min(0)
    end = fresh.cumsum(0)
    wide = (have > width) | (want > width) | (s["before"] < 0) | (s["after"] < 0)
    late = end > tokens
    may = ~wide & ~(late & (fresh > 0))
    need = torch.where(may, (want - have).clamp_min(0), 0)
    head, tail, size = s["ring_state"][0], s["ring_state"][1], s["ring"].numel()
    given_up = need.cumsum(0) > tail - head
    ok = may & ~(given_up & (need > 0))
    status = torch.where(wide, 2, torch.where(late & (fresh > 0), 3, torch.where(ok, 0, 1)))
    take = torch.where(ok, need, 0)
    take_at = take.cumsum(0) - take
    give = torch.where(ok, (have - want).clamp_min(0), 0)
    give_end = give.cumsum(0)
    # the block tables with their new pages
    col = torch.arange(width, device="cuda")[None, :]
    new = (col >= have[:, None]) & (col < (have + take)[:, None])
    at = torch.where(new, (head + take_at[:, None] + col - have[:, None]) % size, 0)
    table = torch.where(new, s["ring"][at], s["table"])
    # a slot for each new token
    t = torch.arange(tokens, device="cuda")
    r = torch.searchsorted(end, t, right=True)
    inside = r < n
    r = r.clamp_max(n - 1)
    position = b[r] + t - (end - fresh)[r]
    row = (position // page).clamp(0, width - 1)
    held = table[r, row].long()
    slots = torch.where(inside & ok[r] & (held >= 0), held * page + position % page, -1)
    # what comes back, behind the ring's tail
    k = (torch.arange(size, device="cuda") - tail) % size
    g = torch.searchsorted(give_end, k, right=True).clamp_max(n - 1)
    back = (want[g] + k - (give_end - give)[g]).clamp(0, width - 1)
    ring = torch.where(k < give_end[-1], s["table"][g, back], s["ring"])
    return {"table": table, "ring": ring, "ring_state_out": torch.stack([head + take.sum(), tail + give_end[-1]]),
            "slots": slots, "positions": torch.where(inside, position, -1).to(torch.int32),
            "starts": torch.cat([end.new_zeros(1), end]).clamp_max(tokens).to(torch.int32),
            "lengths": torch.where(ok, a, b).to(torch.int32), "status": status.to(torch.int32)}


def _turn(x, cos, sin, rot, interleaved):
    x = x.float()
    rest = x[..., rot:]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    case = s["case"]
    # the phase of a late token has more digits than 32 bits hold: it is taken into one turn before it is rounded to them
    angle = torch.remainder(s["positions"].double()[:, None] * s["frequencies"], 2 * math.pi).float()[:, None, :]
    cos, sin = angle.cos(), angle.sin()
    if case["inverse"]:
        sin = -sin
    dtype = TORCH[case["dtype"]]
    q = _turn(s["q"], cos, sin, case["rot"], case["interleaved"]).to(dtype)
    k = _turn(s["k"], cos, sin, case["rot"], case["interleaved"])
    if not case["cache"]:
        return {"q": q, "k": k.to(dtype)}
    v = s["v"].float()
    slots = torch.where(s["slots"] < 0, s["pages"] * case["page"], s["slots"])  # into the spare page
    at, row = slots // case["page"], slots % case["page"]
    fp8 = case["cache"] == "e4m3"
    for cache, x, scale in ((s["k_cache"], k, K_SCALE), (s["v_cache"], v, V_SCALE)):
        x = (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype).view(torch.uint8) if fp8 else x.to(cache.dtype)
        (cache.view(torch.uint8) if fp8 else cache)[at, :, row] = x
    return {"q": q, "k_cache": s["k_cache"][:-1], "v_cache": s["v_cache"][:-1]}


def _gather(s):
    """Keys and values of every request as [requests, kv_heads, longest, dim] in 32 bits, zeros past its length."""
    case = s["case"]
    t = torch.arange(s["total"], device="cuda")
    inside = t[None, :] < s["lengths"][:, None]
    pages = s["table"][:, t // case["page"]].clamp_min(0).long()
    k_scale, v_scale = _scales(case)
    take = lambda cache, scale: torch.where(inside[:, None, :, None], (cache[pages, :, t % case["page"]].float() * scale).transpose(1, 2), 0.0)  # noqa: E731
    return take(s["k_cache"], k_scale), take(s["v_cache"], v_scale)


def _attend(s, q, k, v, seen, distance):
    """q [requests, kv_heads, group, rows, dim], k and v [requests, kv_heads, 1, longest, dim]; seen and distance
    [requests, 1, 1, rows, longest].  A row that sees nothing gives zeros and -inf."""
    case = s["case"]
    scores = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    if case["slopes"]:
        scores = scores - s["slopes"].view(1, case["kv_heads"], -1, 1, 1) * distance.abs().float()
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / torch.where(total == 0, 1.0, total)
    return out, (top + torch.log(total)).squeeze(-1)


def _plain_decode(s):
    case = s["case"]
    k, v = _gather(s)
    n, hk = case["requests"], case["kv_heads"]
    q = s["q"].float().view(n, hk, -1, 1, case["dim"])
    distance = (s["lengths"][:, None] - 1 - torch.arange(s["total"], device="cuda"))[:, None, None, None, :]
    seen = distance >= 0
    if case["window"]:
        seen = seen & (distance < case["window"])
    out, lse = _attend(s, q, k.unsqueeze(2), v.unsqueeze(2), seen, distance)
    return {"out": out.reshape(n, case["q_heads"], case["dim"]).to(TORCH[case["dtype"]]), "lse": lse.reshape(n, case["q_heads"])}


def _plain_prefill(s):
    case = s["case"]
    k, v = _gather(s)
    n, hk, hq, dim = case["requests"], case["kv_heads"], case["q_heads"], case["dim"]
    starts = s["starts"].long()
    fresh = starts[1:] - starts[:-1]
    i = torch.arange(s["most_fresh"], device="cuda")
    row = (starts[:-1, None] + i[None, :]).clamp_max(s["fresh"] - 1)
    q = s["q"].float()[row].view(n, -1, hk, hq // hk, dim).permute(0, 2, 3, 1, 4)
    position = (s["lengths"].long() - fresh)[:, None] + i[None, :]
    key = torch.arange(s["total"], device="cuda")
    distance = (position[:, :, None] - key)[:, None, None]
    seen = distance >= 0
    if case["window"]:
        seen = seen & (distance < case["window"])
    if case["prefix"]:
        seen = seen | (key < s["prefix"][:, None, None, None, None])
    seen = seen & (key < s["lengths"][:, None, None, None, None])
    out, lse = _attend(s, q, k.unsqueeze(2), v.unsqueeze(2), seen, distance)
    # the padded rows back into the tokens' order
    t = torch.arange(s["fresh"], device="cuda")
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    out = out.permute(0, 3, 1, 2, 4)[r, t - starts[r]].reshape(s["fresh"], hq, dim)
    lse = lse.permute(0, 3, 1, 2)[r, t - starts[r]].reshape(s["fresh"], hq)
    return {"out": out.to(TORCH[case["dtype"]]), "lse": lse}


# ---- what cannot be done without ------------------------------------------------------------

def work(case):
    if case["op"] == "pages":
        past, fresh = _spread(case)
        page, n = case["page"], case["requests"]
        moved = int((_pages_of(past + fresh, page) - _pages_of(past, page)).abs().sum())
        # lengths in, lengths, status and starts out; 8 + 4 bytes a token; a page's number read and written
        return {"bytes": 20 * n + 36 + 12 * (int(fresh.clamp_min(0).sum()) + 3) + 8 * moved, "flops": 0}
    if case["op"] == "rotary":
        n, dim, hq, hk = case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
        size = BYTES[case["dtype"]]
        turned = 3 * n * (hq + hk) * case["rot"]
        if not case["cache"]:
            return {"bytes": 2 * n * (hq + hk) * dim * size + 4 * n, "flops": turned}
        return {"bytes": n * dim * ((2 * hq + 2 * hk) * size + 2 * hk * BYTES[case["cache"]]) + 12 * n, "flops": turned}
    past, fresh = _spread(case)
    total = past + fresh
    dim, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    w = case["window"]
    if case["op"] == "decode":
        seen = total.clamp_max(w) if w else total
        keys, pairs, rows = int(seen.sum()), int(seen.sum()), case["requests"]
    else:
        rows = int(fresh.sum())
        prefix = total // 3 if case["prefix"] else torch.zeros_like(total)
        pairs = keys = 0
        for p, f, x in zip(past.tolist(), fresh.tolist(), prefix.tolist()):
            if not f:
                continue
            at = torch.arange(p, p + f)
            low = (at - w + 1).clamp_min(0) if w else torch.zeros_like(at)
            causal = at + 1 - low  # keys low..at, and those of the prefix that are not among them
            extra = torch.minimum(low, torch.tensor(x)) + (x - at - 1).clamp_min(0)
            pairs += int((causal + extra).sum())
            keys += p + f - (max(0, int(low[0]) - x) if w else 0)
    return {"bytes": 2 * keys * hk * dim * BYTES[case["cache"]] + 2 * rows * hq * dim * BYTES[case["dtype"]] + 4 * rows * hq,
            "flops": 4 * pairs * hq * dim}


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None  # whole numbers: the plain form is exact
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_attention(case, s)


def _exact_rotary(case, s):
    rot, half = case["rot"], case["rot"] // 2
    angle = s["positions"].double()[:, None] * s["frequencies"] * (-1.0 if case["inverse"] else 1.0)
    first = torch.arange(half, device="cuda") * 2 if case["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if case["interleaved"] else half)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]

    def turned(x):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(s["q"]), turned(s["k"])
    if not case["cache"]:
        return {"q": q, "k": k}
    if case["cache"] == "e4m3":
        return {"q": q, "k_cache": None, "v_cache": None}  # eight bits: a rounding, not a value
    caches = {}
    keep = s["slots"] >= 0
    for name, x in (("k_cache", k), ("v_cache", s["v"].double())):
        flat = s[name][:-1].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        flat[s["slots"][keep]] = x[keep]
        caches[name] = flat.view(-1, case["page"], case["kv_heads"], case["dim"]).transpose(1, 2).contiguous()
    return {"q": q, **caches}


def _exact_attention(case, s):
    """Request by request and head by head."""
    hk, group, dim, page = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"], case["page"]
    lengths = s["lengths"].tolist()
    starts = s["starts"].tolist() if case["op"] == "prefill" else list(range(len(lengths) + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    k_scale, v_scale = _scales(case)
    for r, length in enumerate(lengths):
        rows = starts[r + 1] - starts[r]
        if not length or not rows:
            continue
        pages = s["table"][r, : -(-length // page)].long()
        position = torch.arange(length - rows, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        seen = key <= position
        if case["window"]:
            seen = seen & (key > position - case["window"])
        if case["op"] == "prefill" and case["prefix"]:
            seen = seen | (key < s["prefix"][r])
        for h in range(hk):
            k = s["k_cache"][pages, h].double().reshape(-1, dim)[:length] * k_scale
            v = s["v_cache"][pages, h].double().reshape(-1, dim)[:length] * v_scale
            for g in range(h * group, (h + 1) * group):
                x = s["q"][starts[r]: starts[r + 1], g].double() @ k.T * s["scale"]
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if case["slopes"]:
                    x = x - s["slopes"][g].double() * (position - key).abs()
                x = x.masked_fill(~seen, -math.inf)
                z = torch.logsumexp(x, -1)
                lse[starts[r]: starts[r + 1], g] = z
                out[starts[r]: starts[r + 1], g] = torch.exp(x - z[:, None]) @ v
    return {"out": out, "lse": lse}
