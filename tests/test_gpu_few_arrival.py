"""The few-token layer where the last workgroup to arrive sums the parts of its columns.

At most eight tokens, at most 16 parts (chosen experts times cuts of the hidden width) and
as many tiles as CUs: the one hand-over between the workgroups of a launch.
"""

import pytest
import torch

from nanotitan_amd.moe_ops import moe_few_tokens
from tests.test_gpu_few_tokens import TYPES, _check, _inputs

pytestmark = pytest.mark.gpu

SHAPES = [  # T, d, f, E, k: parts = min(T k, E) experts x cuts (a cut per 512 of f)
    (1, 512, 2048, 16, 2),  # 2 x 4
    (7, 512, 1365, 8, 2),   # 8 x 2
    (8, 100, 2000, 3, 1),   # 3 x 3, a last tile that reaches back
    (2, 33, 1024, 4, 1),    # 2 x 2, a single narrow tile
    (8, 257, 511, 16, 2),   # 16 x 1, a last tile of one column
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,d,f,E,k", SHAPES)
def test_parts_summed_by_the_last_arriver(ext, dtype, ffn, T, d, f, E, k):
    x, router, weights = _inputs(T, d, f, E, TYPES[dtype], ffn, T * d + E)
    _check(x, router, None, weights, k)


@pytest.mark.parametrize("dtype,T,d,f,E,k", [("bf16", *SHAPES[0]), ("fp32", *SHAPES[1]),
                                             ("fp16", *SHAPES[2])])
def test_two_streams_and_replays_with_other_routings(ext, dtype, T, d, f, E, k):
    """Every call, at once with another or replayed, gives the bits of a call alone."""
    x, _, weights = _inputs(T, d, f, E, TYPES[dtype], "swiglu", 3)
    g = torch.Generator().manual_seed(4)
    routes = [torch.randn(T, E, generator=g).cuda() for _ in range(6)]

    def call(logits):
        with torch.no_grad():
            return moe_few_tokens(x, weights, k, logits=logits)

    refs = [[t.clone() for t in call(r)] for r in routes]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for i in range(len(routes)):
            with torch.cuda.stream(side):
                got.append((i, call(routes[i])))
            j = (i + 1) % len(routes)
            got.append((j, call(routes[j])))
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, refs[i])), i
    static = routes[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = call(static), call(static)
    for i in (1, 2, 0, 3, 5, 4):
        static.copy_(routes[i])
        graph.replay()
        torch.cuda.synchronize()
        for captured in (first, second):
            assert all(torch.equal(a, b) for a, b in zip(captured, refs[i])), i
        call(routes[0])
