"""Log probabilities where the logits leave the ordinary: rows of the type's lowest values."""
import pytest

import helpers as Hh
from test_logprobs_gpu import _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("N,V,top", [(3, 5000, 20), (2, 40001, 5), (300, 1033, 0)])
def test_minus_infinity_beside_the_lowest_values(N, V, top, dtype):
    """Rows masked by the type's lowest value whose padding is -inf: the padding has probability 0, whether the others are the
    lowest value, near it or few."""
    import torch
    Hh.need_cuda()
    x, tokens = _logits(N, V, dtype, seed=V)
    low = torch.finfo(x.dtype).min
    x[:, ::3] = -float("inf")
    x[0, torch.arange(V, device="cuda") % 3 > 0] = low
    x[1, 1::3] = low
    x[1, 2::3] = low * (1 - 2 * torch.finfo(x.dtype).eps)     # four steps above it: these have all the probability
    if N > 2:
        x[2] = -float("inf")
        x[2, V - 1] = low
    tokens[0], tokens[1] = 1, 3
    got = _check(x, tokens, top)
    assert got[0][1] == -float("inf") and got[0].isfinite()[0]
