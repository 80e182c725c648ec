"""Differential attention: the order of sums goes by the sizes and by the scratch that a call finds. Behind an eager call of its own sizes a recorded one
has that call's bits; recorded where the arena has room for less, it adds in another order, within the same bounds."""
import pytest
import torch

from cgpt_amd import capi, ops
from tests.test_gpu_differential_attention import GRADS, backward, case, check, forward, inputs, options, reference
from tests.util import DTYPE_IDS, DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(1, 512, 512, 8, 2, 128), case(1, 8, 6000, 8, 2, 64)], ids=["keys", "queries"])
def test_recorded_where_the_scratch_is_small(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas, dout)
    small = case(1, 40, 40, 2, 1, c["d"])
    given = inputs(small, dtype, device)
    out, second, lse = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((2, *q.shape[:3]), device=device)
    grads = [torch.zeros_like(t) for t in (q, k, v, lambdas)]
    results = (out, second, lse, *grads)

    def both(stream=None):
        ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, stream, options(c))
        ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, stream, options(c))

    capi.call("cgptx_release_scratch")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        backward(small, *given, forward(small, *given[:3], given[4]))
    stream.synchronize()
    recorded = []
    for eager_before in (False, True):
        if eager_before:
            with torch.cuda.stream(stream):
                both()
            stream.synchronize()
            eager = [t.clone() for t in results]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            both()
        recorded.append(graph)
        for _ in range(3):
            for t in results:
                t.fill_(5.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for got, name in zip(results, ("out", "second", "lse", *GRADS)):
                check(got, want[name], want[name + "_err"], name)
            assert not eager_before or all(torch.equal(a, b) for a, b in zip(results, eager))
    recorded[0].replay()  # the block that it was recorded with is still there
    torch.cuda.synchronize()
    for got, name in zip(results, ("out", "second", "lse", *GRADS)):
        check(got, want[name], want[name + "_err"], name)
