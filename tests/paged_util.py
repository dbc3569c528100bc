"""Plain 64-bit forms of the paged-cache operators, and inputs for their tests."""
from __future__ import annotations

import math

import numpy as np
import torch

import manifesto_amd as M
from manifesto_amd import attention as A

TORCH = {M.BFLOAT16: torch.bfloat16, M.FLOAT16: torch.float16, M.FLOAT32: torch.float32, M.F8E4M3: torch.float8_e4m3fn}
# Half a step of the type, relative to the value; and its smallest half step.
HALF_STEP = {M.BFLOAT16: 2.0 ** -8, M.FLOAT16: 2.0 ** -11, M.FLOAT32: 2.0 ** -24, M.F8E4M3: 2.0 ** -4}
SMALLEST = {M.BFLOAT16: 2.0 ** -134, M.FLOAT16: 2.0 ** -25, M.FLOAT32: 2.0 ** -150, M.F8E4M3: 2.0 ** -10}


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def ptr(t) -> int:
    return t.data_ptr() if t is not None else 0


def plan_oracle(before, after, page, table, width, ring, head, tail, tokens):
    """mfh_page_plan, request by request."""
    table, ring, size = table.copy(), ring.copy(), len(ring)
    slots, positions = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int32)
    starts, lengths, status = [0], [], []
    taken = given = asked = 0
    for r, (b0, a0) in enumerate(zip(before.tolist(), after.tolist())):
        b, a = max(b0, 0), max(a0, 0)
        have, want, fresh = -(-b // page), -(-a // page), max(a - b, 0)
        start, end = starts[-1], starts[-1] + fresh
        state = 2 if have > width or want > width or b0 < 0 or a0 < 0 else 3 if fresh and end > tokens else 0
        need = max(want - have, 0) if state == 0 else 0
        asked += need
        if need and asked > tail - head:
            state = 1
        if state == 0:
            for j in range(have, want):
                table[r, j] = ring[(head + taken) % size]
                taken += 1
            for j in range(want, have):
                ring[(tail + given) % size] = table[r, j]
                given += 1
        for t in range(start, min(end, tokens)):
            position = b + t - start
            positions[t] = np.int64(position).astype(np.int32)
            if state == 0:
                held = table[r, position // page]
                slots[t] = held * page + position % page if held >= 0 else -1
        starts.append(end)
        lengths.append(a if state == 0 else b)
        status.append(state)
    return {"table": table, "ring": ring, "ring_state": np.array([head + taken, tail + given]), "slots": slots,
            "positions": positions, "starts": np.minimum(starts, tokens).astype(np.int32),
            "lengths": np.array(lengths, np.int32), "status": np.array(status, np.int32)}


def attention_oracle(q, keys, values, positions, scale, softcap=0.0, window=0, slopes=None, prefix=0):
    """q [n, heads, dim], keys and values [length, kv_heads, dim], all f64 on the CPU; positions of the n rows.
    Returns out, lse, and sum p |v| with the largest sum |q k| for the error bounds."""
    n, heads, dim = q.shape
    group = heads // max(1, keys.shape[1])
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros(n, heads, dtype=torch.float64)
    key = torch.arange(keys.shape[0])
    for i in range(n):
        seen = key <= positions[i]
        if window:
            seen &= key > positions[i] - window
        seen |= key < prefix
        if not bool(seen.any()):
            continue
        for h in range(heads):
            k, v = keys[seen, h // group], values[seen, h // group]
            s = k @ q[i, h] * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * (positions[i] - key[seen]).abs()
            z = torch.logsumexp(s, 0)
            p = torch.exp(s - z)
            lse[i, h], out[i, h], spread[i, h] = z, p @ v, p @ v.abs()
            reach[i, h] = (k.abs() @ q[i, h].abs()).max() * abs(scale)
    return out, lse, spread, reach


def check_attention(got, got_lse, want, dtype, dim, softcap=0.0, slope_reach=0.0):
    """Bounds: the result's rounding and that of every weight to `dtype`; scores to within the rounding of a sum of
    `dim` products in f32 (and of the cap and the bias), as a relative error of every weight."""
    out, lse, spread, reach = want
    got, got_lse = got.double().cpu(), got_lse.double().cpu()
    empty = torch.isinf(lse) & (lse < 0)
    assert torch.equal(torch.isinf(got_lse) & (got_lse < 0), empty)
    assert (got[empty] == 0).all()
    u = HALF_STEP[dtype]
    score = reach * (dim + 8) * 2.0 ** -23 + (softcap + slope_reach + 16.0) * 2.0 ** -21
    bound = u * out.abs() * 1.02 + spread * (1.02 * u + 4 * score[..., None]) + 2 * SMALLEST[dtype]
    assert torch.isfinite(got).all()
    assert ((got - out).abs() <= bound).all(), float(((got - out).abs() / bound).max())
    fine = ~empty
    off = (got_lse - lse)[fine].abs()
    assert (off <= 2 * score[fine] + lse[fine].abs() * 2.0 ** -22).all(), float(off.max())


class Cache:
    """Key and value pages filled with NaN but for the tokens that are put there."""

    def __init__(self, dtype, page, kv_heads, dim, pages, order="head", seed=0, k_scale=1.0, v_scale=1.0, gap=0):
        self.dtype, self.page, self.kv_heads, self.dim, self.pages = dtype, page, kv_heads, dim, pages
        self.k_scale, self.v_scale = k_scale, v_scale
        row = dim + gap  # unused elements between rows
        if order == "head":  # [pages, kv_heads, page, dim]
            strides = (kv_heads * page * row, row, page * row)
        else:  # [pages, page, kv_heads, dim]
            strides = (kv_heads * page * row, kv_heads * row, row)
        n = pages * kv_heads * page * row
        self.gen = torch.Generator().manual_seed(seed)
        self.buffers = []
        for _ in range(2):
            self.buffers.append(torch.full((n,), math.nan, dtype=torch.float32).to(TORCH[dtype]).cuda())
        self.views = [torch.as_strided(b.view(torch.uint8) if dtype == M.F8E4M3 else b, (pages, page, kv_heads, dim),
                                       (strides[0], strides[1], strides[2], 1)) for b in self.buffers]
        self.desc = A.KVCache(dtype, page, kv_heads, dim, pages, page_stride=strides[0], token_stride=strides[1],
                              head_stride=strides[2], k_scale=k_scale, v_scale=v_scale)
        self.free = torch.randperm(pages, generator=self.gen).tolist()

    def random(self, n, std):
        x = torch.randn(n, self.kv_heads, self.dim, generator=self.gen) * std
        return x.clamp(-448, 448).to(TORCH[self.dtype])

    def put(self, length, table_row, k_std=1.0, v_std=1.0):
        """Fills `length` tokens into free pages of a request; returns its keys and values as f64 on the CPU."""
        ks, vs = self.random(length, k_std), self.random(length, v_std)
        for j in range(-(-length // self.page)):
            table_row[j] = self.free.pop()
        if length:
            t = torch.arange(length)
            pages, rows = table_row[t // self.page].long().cuda(), (t % self.page).cuda()
            for view, x in zip(self.views, (ks, vs)):
                view[pages, rows] = (x.view(torch.uint8) if self.dtype == M.F8E4M3 else x).cuda()
        return ks.double() * self.k_scale, vs.double() * self.v_scale
