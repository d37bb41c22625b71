"""Document numbers of every size on the GPU: told apart as on the CPU, in any
order, over rows of any length, and in a graph."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import biased_attention
from neural_shift_cuda_amd import _C
from test_token_documents_cpu import PACKINGS, packed, tensors

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"


def first_places(docs):
    """Each number's first place in its row, -1 for negative ones."""
    out = []
    for row in docs.tolist():
        seen = {}
        out.append([seen.setdefault(x, j) if x >= 0 else -1 for j, x in enumerate(row)])
    return torch.tensor(out, dtype=torch.int32).view(docs.shape)


@pytest.mark.parametrize("name", list(PACKINGS))
def test_documents_are_told_apart(name):
    docs, small = packed(*PACKINGS[name])
    q, k, v = (t.to(DEV) for t in tensors())
    got = biased_attention(q, k, v, causal=True, documents=docs.to(DEV))
    assert torch.equal(got, biased_attention(q, k, v, causal=True, documents=small.to(DEV)))
    assert not torch.equal(got, biased_attention(q, k, v, causal=True))


@pytest.mark.parametrize("B,L,many", [(1, 1, 1), (3, 63, 5), (2, 64, 64), (5, 65, 3), (1, 257, 2),
                                      (2, 1000, 1000), (4, 5000, 7), (70, 129, 40)])
@pytest.mark.parametrize("order", ["packed", "mixed"])
def test_numbers_become_first_places(B, L, many, order):
    g = torch.Generator().manual_seed(L)
    numbers = torch.randint(-(1 << 40), 1 << 62, (many,), generator=g)
    docs = numbers[torch.randint(0, many, (B, L), generator=g)]
    if order == "packed":
        docs = docs.sort(1).values
    assert torch.equal(_C.document_ids(docs.to(DEV)).cpu(), first_places(docs))


def test_in_a_graph():
    q, k, v = (t.to(DEV) for t in tensors())
    docs = packed(*PACKINGS["int64"])[0].to(DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        biased_attention(q, k, v, documents=docs)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = biased_attention(q, k, v, documents=docs)
    for r in range(4):
        new = docs.roll(r + 1, 1)
        want = biased_attention(q, k, v, documents=new.clone())
        docs.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {r}"
