"""Beam search over one attention layer and a vocabulary, served from a paged key-value cache.

    python3 examples/beam_search.py [--beams N] [--steps N]

Prompts of different lengths come in and are computed once, in the row of each
request's first beam; a fork makes the other beams share its pages.  A step
then attends with the prompt's pages read once for all beams of a request,
selects the best continuations, and brings block tables, pages that are written
next and histories into the beams' new order.  Steps are one captured graph,
for all that changes between them is on the device.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import manifesto_amd as M  # noqa: E402
from manifesto_amd import attention as A, beams as B  # noqa: E402

_spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
_paged = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_paged)
p = torch.Tensor.data_ptr


class BeamSearch(_paged.PagedAttention):
    """The layer and its cache, an embedding and a vocabulary, and the beams' state; row g * beams + b is beam b of request g."""

    def __init__(self, requests: int, beams: int, longest: int, vocab: int = 4096, end_token: int = -1, **layer):
        rows = requests * beams
        super().__init__(rows, longest, **layer)
        self.groups, self.beams, self.vocab = requests, beams, vocab
        hidden = self.weight.shape[0]
        gen = torch.Generator("cuda").manual_seed(99)
        self.embedding = torch.randn(vocab, hidden, generator=gen, device="cuda").bfloat16()
        self.to_vocab = (torch.randn(self.q_heads * self.head_dim, vocab, generator=gen, device="cuda") * 0.2).bfloat16()
        pages = self.ring.numel()

        def ints(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device="cuda")

        # what forks read and write
        self.table_out, self.shares = torch.full_like(self.table, -1), ints(pages)
        self.copy_from, self.copy_to, self.copy_tokens = ints(rows), ints(rows), ints(rows)
        self.fork_space = torch.empty(A.page_fork_workspace(rows, pages), dtype=torch.uint8, device="cuda")
        # the selection's
        self.shape = B.Beams(M.BFLOAT16, beams, beams, vocab, end_token=end_token, history_stride=longest)
        self.scores, self.tokens, self.parents = torch.zeros(rows, device="cuda"), ints(rows), ints(rows)
        self.next_scores = torch.zeros(rows, device="cuda")
        self.ended, self.next_ended = (torch.zeros(rows, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.with_end = end_token >= 0
        self.history, self.next_history, self.known = ints(rows, longest), ints(rows, longest), ints(requests)
        self.select_space = torch.empty(B.beam_select_workspace(self.shape, requests), dtype=torch.uint8, device="cuda")
        # the shared attention's: beams of a request, and the whole pages of its prompt
        self.group_starts = torch.arange(0, rows + 1, beams, dtype=torch.int32, device="cuda")
        self.shared, self.most_shared, self.most_own = ints(requests), longest, longest
        need = A.paged_decode_shared_workspace(self.attention, self.cache, rows, requests, longest, longest)
        self.shared_space = torch.empty(need, dtype=torch.uint8, device="cuda")

    def fork(self, parents: torch.Tensor):
        """Row r becomes a copy of row parents[r]; the pages that grow next are copied."""
        stream = torch.cuda.current_stream().cuda_stream
        A.page_fork(p(parents), p(self.lengths), 0, self.requests, self.page_size, p(self.table), p(self.table_out), self.width,
                    p(self.shares), p(self.shares), self.ring.numel(), p(self.ring), self.ring.numel(), p(self.ring_state),
                    p(self.ring_state_out), p(self.next), p(self.status), p(self.copy_from), p(self.copy_to), p(self.copy_tokens),
                    p(self.fork_space), self.fork_space.numel(), stream=stream)
        A.page_copy(self.cache, self.requests, p(self.copy_from), p(self.copy_to), p(self.copy_tokens), p(self.keys),
                    p(self.values), stream=stream)
        self.table.copy_(self.table_out)
        self.ring_state.copy_(self.ring_state_out)
        self.lengths.copy_(self.next)

    def select(self, logits: torch.Tensor):
        """The best continuations of every request's beams, and the beams in their order."""
        B.beam_select(self.shape, self.groups, p(logits), p(self.scores), p(self.ended) if self.with_end else 0, p(self.next_scores),
                      p(self.tokens), p(self.parents), p(self.next_ended), p(self.history), p(self.known), p(self.next_history),
                      p(self.select_space), self.select_space.numel(), stream=torch.cuda.current_stream().cuda_stream)
        self.scores.copy_(self.next_scores)
        self.ended.copy_(self.next_ended)
        self.history.copy_(self.next_history)
        self.known.add_(1)
        self.fork(self.parents)

    def begin(self, prompts):
        """Computes the prompts (lists of tokens) and selects each request's first beams."""
        lengths = [len(prompts[r // self.beams]) if r % self.beams == 0 else 0 for r in range(self.requests)]
        text = torch.tensor([t for prompt in prompts for t in prompt], device="cuda")
        out, _ = self.prompts(self.embedding[text], lengths)
        for g, prompt in enumerate(prompts):
            self.history[g * self.beams, : len(prompt)] = torch.tensor(prompt, dtype=torch.int32, device="cuda")
        self.known.copy_(torch.tensor([len(x) for x in prompts], dtype=torch.int32))
        self.shared.copy_(self.known // self.page_size * self.page_size)
        self.most_shared = int(self.shared.max())
        # what does not fill a page of the prompt, and the steps that the longest prompt leaves
        self.most_own = min(self.page_size - 1 + self.longest - max(len(x) for x in prompts), self.longest)
        # of each request only the first beam is there yet
        self.scores.fill_(float("-inf"))
        self.scores[:: self.beams] = 0.0
        logits = torch.zeros(self.requests, self.vocab, dtype=torch.bfloat16, device="cuda")
        last = torch.tensor(lengths[:: self.beams], device="cuda").cumsum(0) - 1
        logits[:: self.beams] = out.flatten(1)[last] @ self.to_vocab
        self.select(logits)

    def advance(self):
        """One more token for every beam; returns the attention's rows and the queries as they were turned."""
        stream, n = torch.cuda.current_stream().cuda_stream, self.requests
        slots = torch.empty(n, dtype=torch.int64, device="cuda")
        positions = torch.empty(n, dtype=torch.int32, device="cuda")
        torch.add(self.lengths, 1, out=self.after)
        A.page_plan(p(self.lengths), p(self.after), n, self.page_size, p(self.table), self.width, p(self.ring), self.ring.numel(),
                    p(self.ring_state), p(self.ring_state_out), p(slots), p(positions), n, p(self.starts), p(self.next), p(self.status),
                    stream=stream)
        self.ring_state.copy_(self.ring_state_out)
        self.lengths.copy_(self.next)
        qkv = self.embedding[self.tokens.clamp_min(0)] @ self.weight
        q = torch.empty(n, self.q_heads, self.head_dim, dtype=torch.bfloat16, device="cuda")
        out, at_k = torch.empty_like(q), self.q_heads * self.head_dim * 2
        A.rotary_append(self.rotary, self.cache, n, p(qkv), p(q), p(qkv) + at_k, p(qkv) + at_k + self.kv_heads * self.head_dim * 2,
                        p(positions), p(slots), p(self.frequencies), p(self.keys), p(self.values), stream=stream)
        A.paged_decode_shared(self.attention, self.cache, n, self.groups, p(q), p(self.keys), p(self.values), p(self.table), self.width,
                              p(self.group_starts), p(self.shared), self.most_shared, p(self.lengths), self.most_own, 0,
                              p(out), 0, p(self.shared_space), self.shared_space.numel(), stream=stream)
        return out, q

    def capture_search(self):
        """A graph of one step: a token more for every beam, and the selection behind it."""
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # the library's first calls choose their kernels
            x = self.embedding[self.tokens.clamp_min(0)]
            x @ self.weight
            torch.zeros(self.requests, self.to_vocab.shape[0], dtype=torch.bfloat16, device="cuda") @ self.to_vocab
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, q = self.advance()
            self.select(out.flatten(1) @ self.to_vocab)
        return graph, out, q


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--beams", type=int, default=4)
    parser.add_argument("--steps", type=int, default=64)
    args = parser.parse_args()
    lengths = [1, 37, 512, 1900, 64, 1023, 333, 4000]
    search = BeamSearch(len(lengths), args.beams, max(lengths) + args.steps + 1, vocab=32000, end_token=2)
    gen = torch.Generator().manual_seed(1)
    search.begin([torch.randint(3, 32000, (n,), generator=gen).tolist() for n in lengths])
    torch.cuda.synchronize()
    print(f"{len(lengths)} prompts, {args.beams} beams each: {search.free_pages()} of {search.ring.numel()} pages are free")
    graph, _, _ = search.capture_search()
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(args.steps):
        graph.replay()
    torch.cuda.synchronize()
    micros = (time.perf_counter() - start) / args.steps * 1e6
    print(f"{args.steps} steps: {micros:.0f} us a step; {search.free_pages()} pages are free")
    best = search.scores.view(len(lengths), -1)[:, 0].tolist()
    print("best scores", [round(s, 2) for s in best])
    search.fork(torch.full((search.requests,), -1, dtype=torch.int32, device="cuda"))
    print(f"all requests ended: {search.free_pages()} pages are free")


if __name__ == "__main__":
    main()
