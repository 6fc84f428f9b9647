"""GPU: parts of a unit that many warps leave and the last one joins, over and over: the joined rows are the same bit by bit whichever
warp comes last, and those of the oracle. (That every lane's reads of the parts come after the arrivals is shown by reading.)"""

from __future__ import annotations

import pytest
import torch

from test_kv_q4_gpu import _check_chunk, _chunk_inputs

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("Hq,Hkv,hd", [(16, 4, 128), (12, 1, 128), (6, 2, 64)])
def test_joins_repeat_bit_for_bit(zb, Hq, Hkv, hd):
    gen = torch.Generator().manual_seed(Hq)
    x = _chunk_inputs(gen, [1, 1], [30000, 8000], Hq, Hkv, hd, 64)
    first = _check_chunk(zb, *x, max_new=1)
    x = [t.to(DEV) for t in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(60):  # beside another stream's, so that the order of arrival changes
        with torch.cuda.stream(side):
            outs.append(zb.ops.gqa_chunk_q4(*x, max_new=1))
        outs.append(zb.ops.gqa_chunk_q4(*x, max_new=1))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
