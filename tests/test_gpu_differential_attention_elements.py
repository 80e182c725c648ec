"""Differential attention: a single value that is not finite in a key that some queries of a tile do not see reaches none of them, whichever of the
elements that a lane reads together holds it."""
import pytest
import torch

from tests.test_gpu_differential_attention import case, check, forward, inputs, reference
from tests.util import DTYPE_IDS, DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(1, 70, 70, 4, 2, 64), case(1, 200, 200, 2, 1, 128), case(2, 33, 33, 2, 2, 36)], ids=["64", "128", "36"])
def test_one_value_of_a_hidden_key(device, c, dtype):
    q, k, v, _, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas)
    key = c["ks"] - 6
    for column in range(c["d"] // 2, c["d"] // 2 + 8):
        for value in (float("nan"), float("inf")):
            broken = v.clone()
            broken[:, key, :, column] = value
            for got, name in zip(forward(c, q, k, broken, lambdas), ("out", "second")):
                check(got[:, :key], want[name][:, :key], want[name + "_err"][:, :key], f"{name}, column {column}")
                assert not torch.isfinite(got[:, key:, :, column]).any(), f"{name}: column {column}"
