"""A model's long context, answered through the index.

One attention layer over a document of --tokens tokens: its keys and values go
into a paged cache (rotary positions on a quarter of each head), an index is
built over the keys of every key head, and then, for every new token,

  1. the token's queries are turned and its key and value appended,
  2. its query heads search the index of their key head by inner product,
  3. retrieved_attention reads the first tokens, the latest ones and those
     found, decode_attention all of them.

The index holds the document; the tokens that came after it are all read, as the
window grows with them (a much longer answer would append them to an index of its
own). Two continuations share the document's pages (a fork). Printed: the share
of the full softmax's weight that the retrieved tokens carry, how far the output
is off, and the time of either attention and of the searches. The data are
synthetic: keys of --topics topics with noise, every new query near one of them.

    python examples/long_context.py --tokens 65536
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import jasper_amd  # noqa: E402


def build_indexes(cache, seq, exact):
    """A search (queries [heads, dim], k) -> ids per key head of the cache's layer 0."""
    searches = []
    for keys in cache.keys(0, seq):
        if exact:
            searches.append(lambda q, k, keys=keys: jasper_amd.bruteforce_knn(keys, q, k, distance="ip")[0])
        else:
            graph = jasper_amd.Graph.build(keys, n_neighbors=32, distance="ip")
            searches.append(lambda q, k, graph=graph: graph.search(q, k=k, beam_width=max(64, 2 * k))[0])
    return searches


def retrieve(searches, q, k):
    """The ids [sequences, heads, k] that each query head's search of its key head's index returns."""
    n, heads, dim = q.shape
    group = heads // len(searches)
    found = [search(q[:, h * group:(h + 1) * group].reshape(-1, dim), k).view(n, group, k)
             for h, search in enumerate(searches)]
    return torch.cat(found, dim=1).contiguous()


def timed(f, repeats=20):
    f()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(repeats):
        f()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) / repeats * 1e3


@torch.no_grad()
def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=32768)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--q-heads", type=int, default=8)
    ap.add_argument("--kv-heads", type=int, default=2)
    ap.add_argument("--dim", type=int, default=128)
    ap.add_argument("--k", type=int, default=100, help="tokens retrieved per query head")
    ap.add_argument("--first", type=int, default=4)
    ap.add_argument("--last", type=int, default=64, help="at least; all tokens after the document in any case")
    ap.add_argument("--topics", type=int, default=0, help="0: one per 64 tokens")
    ap.add_argument("--exact", action="store_true", help="search by brute force, not through a graph")
    ap.add_argument("--quiet", action="store_true")
    a = ap.parse_args(argv)
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    n_topics = a.topics or max(1, a.tokens // 64)
    topics = 1.8 * rand(n_topics, a.dim)

    def tokens(n, noise):  # keys of n tokens: a topic each, and the rest of the layer's projections
        topic = torch.randint(0, n_topics, (n, a.kv_heads), device="cuda", generator=g)
        k = (topics[topic] + noise * rand(n, a.kv_heads, a.dim)).half()
        q = topics[topic.repeat_interleave(a.q_heads // a.kv_heads, dim=1)] + noise * rand(n, a.q_heads, a.dim)
        return q.half(), k, rand(n, a.kv_heads, a.dim).half()

    cos, sin = jasper_amd.rotary_table(a.tokens + a.steps, a.dim // 4 // 2 * 2)
    pages = -(-(a.tokens + a.steps) // 16) + 8
    cache = jasper_amd.PagedCache(pages, n_layers=1, kv_heads=a.kv_heads, dim=a.dim, max_sequences=2)
    document = cache.new()
    step = cache.extend([document], a.tokens)
    q, k, v = tokens(a.tokens, 0.5)
    cache.append(0, step, None, k, v, cos, sin)
    searches = build_indexes(cache, document, a.exact)
    answers = [document, cache.fork(document)]

    weights, errors = [], []
    for _ in range(a.steps):
        step = cache.extend(answers, 1)
        q, k, v = tokens(len(answers), 0.5)
        q = cache.append(0, step, q, k, v, cos, sin)
        ids = retrieve(searches, q, a.k)
        last = max(a.last, step.max_len - a.tokens)  # what the index does not hold
        out, lse = cache.retrieved(0, step, q, ids, first=a.first, last=last, return_lse=True)
        full, full_lse = cache.decode(0, step, q, return_lse=True)
        weights.append(torch.exp(lse - full_lse).mean().item())
        errors.append(((out.float() - full.float()).norm() / full.float().norm()).item())
    us = [timed(lambda: cache.retrieved(0, step, q, ids, first=a.first, last=last)), timed(lambda: cache.decode(0, step, q)),
          timed(lambda: retrieve(searches, q, a.k))]
    if not a.quiet:
        print(f"{a.tokens} tokens, {a.first} + {a.k} + {last} read per query head: "
              f"{100 * sum(weights) / a.steps:.1f}% of the weight, output off by {100 * sum(errors) / a.steps:.2f}%; "
              f"attention {us[0]:.1f} us of the retrieved, after {us[2]:.1f} us of searches; {us[1]:.1f} us of all")
    cache.free(answers)
    return sum(weights) / a.steps, sum(errors) / a.steps


if __name__ == "__main__":
    main()
