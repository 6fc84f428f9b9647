"""GPU: batches marked as decode whose requests bring more than one token (drafts), or none, over a pool of 4 bits: every row is what it
is in the same batch not marked so."""

from __future__ import annotations

import pytest
import torch

from test_kv_q4_model_gpu import DEV, _model, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 3, 1], [2, 1, 0], [0, 0, 9]])
def test_decode_batches_with_drafts(zb, news):
    model = _model(zb, 4)
    layer = model.layers.op_list[3].attention
    pool = model.allocate_caches(4, 40 * 16, DEV, kv_bits=4)
    zb.core.get_global_ctx().attn_backend = pool
    gen = torch.Generator().manual_seed(7)
    table = _table(gen, 3, 9, 40)
    lengths = [70, 33, 100]
    layer.prepare()
    old = torch.randn(sum(lengths), 512, generator=gen).bfloat16().to(DEV)
    n = sum(news)
    x = torch.randn(n, 512, generator=gen).bfloat16().to(DEV)

    def run(x, news, keys, is_decode):
        cu = torch.tensor([0, *news], dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
        meta = zb.core.AttnMetadata(None, None, table, torch.tensor(keys, dtype=torch.int32, device=DEV), cu)
        reqs = [zb.core.Req(b, 1) for b in range(3)]  # what the host said of the batch when it made it
        with zb.core.forward_batch(zb.core.Batch(reqs=reqs, is_decode=is_decode, attn_metadata=meta)):
            return layer.forward(x)

    run(old, lengths, lengths, False)
    keys = [a + b for a, b in zip(lengths, news)]
    expected = run(x, news, keys, False)
    junk = [torch.full_like(expected, float("nan")) for _ in range(64)]  # what an unwritten row would hold
    del junk
    got = run(x, news, keys, True)
    assert zb.ops.device_status() == 0
    if news == [1, 1, 1]:
        assert got.isfinite().all()
    assert torch.allclose(got.float(), expected.float(), rtol=0, atol=3e-2 * float(expected.abs().max()))
