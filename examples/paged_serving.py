"""One attention layer served over a paged key-value cache.

    python3 examples/paged_serving.py [--e4m3] [--steps N]

Prompts of different lengths come in, their tokens are computed in one call,
and every request then answers token by token until it ends and its pages go
back.  A step is page_plan, rotary_append and paged_prefill or paged_decode;
the steps of one token each are one captured graph that is replayed, since all
that changes between them (lengths, pages, slots) is on the device.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import manifesto_amd as M  # noqa: E402
from manifesto_amd import attention as A  # noqa: E402


class PagedAttention:
    """The layer's weights, its cache, and what the steps share; bf16, on the current device."""

    def __init__(self, requests: int, longest: int, q_heads: int = 16, kv_heads: int = 4, head_dim: int = 128,
                 hidden: int = 1024, page_size: int = 16, cache_dtype: int = M.BFLOAT16, window: int = 0,
                 pages: int | None = None, seed: int = 0):
        M.init(torch.cuda.current_device())
        self.requests, self.longest, self.head_dim = requests, longest, head_dim
        self.q_heads, self.kv_heads, self.page_size = q_heads, kv_heads, page_size
        self.width = -(-longest // page_size)
        pages = requests * self.width if pages is None else pages
        gen = torch.Generator("cuda").manual_seed(seed)
        self.weight = (torch.randn(hidden, (q_heads + 2 * kv_heads) * head_dim, generator=gen, device="cuda") * hidden ** -0.5).bfloat16()
        scale = 1.0 if cache_dtype == M.BFLOAT16 else 2.0 ** -6  # |k|, |v| up to 7 in codes up to 448
        self.cache = A.KVCache(cache_dtype, page_size, kv_heads, head_dim, pages, k_scale=scale, v_scale=scale)
        kind = torch.bfloat16 if cache_dtype == M.BFLOAT16 else torch.float8_e4m3fn
        self.keys, self.values = (torch.empty(pages, kv_heads, page_size, head_dim, dtype=kind, device="cuda") for _ in range(2))
        # q, k and v are slices of the projection's rows
        row = (q_heads + 2 * kv_heads) * head_dim
        self.rotary = A.Rotary(M.BFLOAT16, q_heads, kv_heads, head_dim, q_strides=(row, head_dim), k_strides=(row, head_dim),
                               v_strides=(row, head_dim))
        self.frequencies = torch.tensor(A.rotary_frequencies(head_dim), dtype=torch.float64, device="cuda")
        self.attention = A.Attention(M.BFLOAT16, q_heads, head_dim ** -0.5, window=window)

        def ints(*shape, dtype=torch.int32):
            return torch.zeros(*shape, dtype=dtype, device="cuda")

        self.table = torch.full((requests, self.width), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.arange(pages, dtype=torch.int32, device="cuda")  # every page is free
        self.ring_state, self.ring_state_out = torch.tensor([0, pages], device="cuda"), ints(2, dtype=torch.int64)
        self.lengths, self.after, self.next = ints(requests), ints(requests), ints(requests)
        self.starts, self.status = ints(requests + 1), ints(requests)
        need = A.paged_decode_workspace(self.attention, self.cache, requests, longest)
        self.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")

    def step(self, x: torch.Tensor, most_fresh: int):
        """Rows of x are the new tokens, request after request; self.after says how long each request becomes.
        Returns the attention's rows, and the queries as they were turned."""
        p = torch.Tensor.data_ptr
        tokens, stream = x.shape[0], torch.cuda.current_stream().cuda_stream
        slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        positions = torch.empty(tokens, dtype=torch.int32, device="cuda")
        A.page_plan(p(self.lengths), p(self.after), self.requests, self.page_size, p(self.table), self.width, p(self.ring),
                    self.ring.numel(), p(self.ring_state), p(self.ring_state_out), p(slots), p(positions), tokens,
                    p(self.starts), p(self.next), p(self.status), stream=stream)
        self.ring_state.copy_(self.ring_state_out)
        self.lengths.copy_(self.next)
        qkv = x @ self.weight
        q = torch.empty(tokens, self.q_heads, self.head_dim, dtype=torch.bfloat16, device="cuda")
        out, at_k = torch.empty_like(q), self.q_heads * self.head_dim * 2
        A.rotary_append(self.rotary, self.cache, tokens, p(qkv), p(q), p(qkv) + at_k,
                        p(qkv) + at_k + self.kv_heads * self.head_dim * 2, p(positions), p(slots), p(self.frequencies),
                        p(self.keys), p(self.values), stream=stream)
        if most_fresh == 1 and tokens == self.requests:
            A.paged_decode(self.attention, self.cache, self.requests, p(q), p(self.keys), p(self.values), p(self.table),
                           self.width, p(self.lengths), self.longest, 0, p(out), 0, p(self.workspace),
                           self.workspace.numel(), stream=stream)
        else:
            need = A.paged_prefill_workspace(self.attention, self.cache, self.requests, tokens, most_fresh, self.longest)
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            A.paged_prefill(self.attention, self.cache, self.requests, tokens, most_fresh, p(q), p(self.keys), p(self.values),
                            p(self.table), self.width, p(self.starts), p(self.lengths), self.longest, 0, 0, p(out), 0,
                            p(workspace), need, stream=stream)
        return out, q

    def prompts(self, x: torch.Tensor, lengths):
        """The prompts' tokens, in one call."""
        self.after.copy_(self.lengths + torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        result = self.step(x, max(lengths))
        refused = self.status.nonzero().flatten().tolist()
        if refused:
            raise RuntimeError(f"no pages for the requests {refused}: {self.status.tolist()}")
        return result

    def capture(self, x: torch.Tensor):
        """A graph of one more token per request, read from x; returns it with its result and queries."""
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x @ self.weight  # the library's first call chooses its kernel
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            torch.add(self.lengths, 1, out=self.after)
            out, q = self.step(x, 1)
        return graph, out, q

    def end(self, request: int):
        """Returns the request's pages; the others keep theirs."""
        self.after.copy_(self.lengths)
        self.after[request] = 0
        p, none = torch.Tensor.data_ptr, 0
        A.page_plan(p(self.lengths), p(self.after), self.requests, self.page_size, p(self.table), self.width, p(self.ring),
                    self.ring.numel(), p(self.ring_state), p(self.ring_state_out), none, none, 0, p(self.starts), p(self.next),
                    p(self.status), stream=torch.cuda.current_stream().cuda_stream)
        self.ring_state.copy_(self.ring_state_out)
        self.lengths.copy_(self.next)

    def free_pages(self) -> int:
        head, tail = self.ring_state.tolist()
        return tail - head


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--e4m3", action="store_true", help="keep keys and values in 8 bits")
    parser.add_argument("--steps", type=int, default=64)
    args = parser.parse_args()
    prompts = [1, 37, 512, 1900, 64, 1023, 333, 4000]
    layer = PagedAttention(len(prompts), max(prompts) + args.steps, cache_dtype=M.F8E4M3 if args.e4m3 else M.BFLOAT16)
    x = torch.randn(sum(prompts), layer.weight.shape[0], device="cuda").bfloat16()
    layer.prompts(x, prompts)
    torch.cuda.synchronize()
    print(f"{len(prompts)} prompts, {sum(prompts)} tokens: {layer.free_pages()} of {layer.ring.numel()} pages are free")
    token = x[: len(prompts)].clone()
    graph, out, _ = layer.capture(token)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(args.steps):
        graph.replay()
        token.copy_(out.reshape(len(prompts), -1)[:, : token.shape[1]])
    torch.cuda.synchronize()
    micros = (time.perf_counter() - start) / args.steps * 1e6
    print(f"{args.steps} steps of one token each: {micros:.0f} us a step; lengths {layer.lengths.tolist()}")
    for request in range(len(prompts)):
        layer.end(request)
    print(f"all requests ended: {layer.free_pages()} pages are free")


if __name__ == "__main__":
    main()
