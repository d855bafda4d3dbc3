"""Prompt passes on caches in 8 bits and under windows, recorded into a graph and replayed."""
import pytest
import torch

from page_cases import Book, close
from test_page_attention_gpu import prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("seen", [(None, 0), (37, 5)])
def test_recorded_prompts(ops, quant, seen):
    """A pass of several sequences, some of them behind pages that are there, recorded once (attention, rounding and tails; shares with their join) and replayed for other
    tokens, with other work, waits and another stream between."""
    starts, new = [32, 0, 1024], [40, 23, 64]
    book = Book(starts, 8, 2, 128, quant, seed=11, room=80)
    k, v = list(book.k), list(book.v)
    x, seqs, poss, q = book.append([0, 1, 2], new)
    x = x.clone()
    prompt(ops, book, x, seqs, poss, *seen)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt(ops, book, x, seqs, poss, *seen, longest=1100)
    for i in range(6):
        book.k, book.v, book.lens = list(k), list(v), list(starts)
        y, _, _, q = book.append([0, 1, 2], new)
        x.copy_(y)
        if i % 2:
            torch.cuda.synchronize()
            torch.randn((1000, 1000), device=book.dev).sum()
        if i % 3 == 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
        close(out, book.expect(q, seqs, poss, *seen))
        for b in range(3):
            book.same_pages(b)
