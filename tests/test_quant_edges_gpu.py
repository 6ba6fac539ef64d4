"""Attention over a 4-bit cache where its inputs leave the ordinary: queries and scores of any size, NaN among the values,
small scales, long units beside others, every number of query rows; the write's scales over all of fp16."""
import numpy as np
import pytest

import helpers as Hh
from oracle import quant_oracle as Q
from test_quant_decode_gpu import SCALE, _close, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len,G", [(1, 4), (40, 4), (200, 2)])
def test_a_call_behind_a_stalled_one(q_len, G):
    """A call whose bounded waits run out ends with its loads landed and its products done: the one behind it in the stream,
    on the same SMs, is right."""
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    q, kc, vc, table, qs, lens = _inputs([3000] * 20, [q_len] * 20, 2, G, 64, seed=31)
    want = Hh.ops().cascade_quant_decode(q, kc, vc, table, qs, lens, q_len, SCALE, True)
    outs = [(torch.empty_like(want[0]), torch.empty_like(want[1])) for _ in range(2)]
    for _ in range(3):
        for flags, (out, lse) in zip((C.FLAG_DEBUG_STALL, 0), outs):
            d = C.quant_desc(q, kc, vc, table, None, lens, q_len, SCALE, flags=flags)
            ws = torch.zeros(C.quant_decode_workspace_size(d), dtype=torch.uint8, device="cuda")
            C.quant_decode(d, out, lse, ws)
        assert torch.equal(outs[1][0], want[0]) and torch.equal(outs[1][1], want[1])
        assert C.device_error() == 1
