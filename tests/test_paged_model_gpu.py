"""GPU: the whole model over the paged operators (a device-side cu_seqlens_q), against the oracle LM (oracle/lm.py, pinned
to the reference Zonos3LM) and against the module's own torch prefill.

The reduced model of tests/test_model_gpu.py (hidden 512, 4 layers in the 3:1 pattern, GQA 8 / 2 heads of 128). Ragged
prompts arrive in chunks while other streams decode, over a paged pool of 16-token pages and over the slot pool.

Bars as in tests/test_model_gpu.py: soft-capped logits against the oracle's (bf16 activations vs fp32) at cosine >= 0.999
for a prompt's rows, none below 0.995 for decode rows (a token whose router logits sit one bf16 step from a top-k tie can
take another expert). The module alone, paged against torch prefill: both round q and k to bf16 (the torch path after each
of up to three steps) and probabilities and outputs once, so their outputs differ by a few bf16 units: 3e-2 of the largest
value."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from conftest import max_rel_err
from oracle import lm as olm
from test_model_gpu import _configs

pytestmark = pytest.mark.gpu

TEXT_VOCAB = 1024
MAX_LEN = 96


def _model(zb, seed):
    oc, mc = _configs(zb)
    w = olm.random_weights(oc, seed=seed)
    model = zb.model.Zonos3ForCausalLM(mc)
    model.load_state_dict(dict(w))
    model.to(torch.device("cuda"), torch.bfloat16)
    return oc, w, model


@pytest.mark.parametrize("page_size", [None, 16])
def test_chunked_prefill_beside_decode_matches_oracle_lm(zb, page_size):
    dev = torch.device("cuda")
    oc, w, model = _model(zb, 3)
    streams = 5
    pool = model.allocate_caches(streams, streams * MAX_LEN, dev, page_size=page_size)
    page = page_size or 1
    per = -(-MAX_LEN // page)
    gen = torch.Generator().manual_seed(5)
    table = torch.randperm(streams * per, generator=gen).view(streams, per).to(torch.int32).to(dev)
    lengths = [40, 9, 61, 17, 30]
    rows = [torch.cat([torch.randint(0, 4096, (n, 10), generator=gen), torch.randint(0, TEXT_VOCAB, (n, 1), generator=gen)], 1)
            for n in lengths]
    caches = [olm.Cache() for _ in range(streams)]
    ref = [olm.forward(oc, w, r, c) for r, c in zip(rows, caches)]  # every row's logits, in one go
    # new tokens a step and stream: chunks of prompts, single tokens and pauses side by side
    steps = [[7, 9, 30, 0, 1], [1, 0, 1, 16, 1], [20, 0, 29, 1, 27], [12, 0, 1, 0, 1]]
    done = [0] * streams
    zb.core.get_global_ctx().attn_backend = pool
    for news in steps:
        live = [b for b in range(streams) if news[b]]
        cu = [0]
        for b in live:
            cu.append(cu[-1] + news[b])
        ids = torch.cat([rows[b][done[b]:done[b] + news[b]] for b in live]).to(torch.int32).to(dev)
        meta = zb.core.AttnMetadata(positions=None, out_loc=None, page_table=table[live].contiguous(),
                                    cache_seqlens=torch.tensor([done[b] + news[b] for b in live], dtype=torch.int32, device=dev),
                                    cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device=dev))
        batch = zb.core.Batch(reqs=[zb.core.Req(b, news[b], done[b], uid=b) for b in live], is_decode=False, input_ids=ids,
                              attn_metadata=meta)
        with zb.core.forward_batch(batch):
            got = model.forward().float().cpu()
        for i, b in enumerate(live):
            part = ref[b][done[b]:done[b] + news[b]]
            cos = F.cosine_similarity(got[cu[i]:cu[i + 1]].flatten(1), part.flatten(1), dim=1)
            assert cos.min() >= 0.995 and cos.median() >= 0.999, f"stream {b} at {done[b]}: {cos.min():.5f}, {cos.median():.5f}"
            done[b] += news[b]
    assert done == lengths
    assert zb.ops.device_status() == 0


def test_attention_module_paged_against_torch_prefill(zb):
    """The same prefill through the module's host-list path and its device-tensor path, then a decode step through either:
    outputs and cache contents."""
    dev = torch.device("cuda")
    _, _, model = _model(zb, 4)
    layer = model.layers.op_list[3].attention
    lengths, width = [20, 1, 77], 80
    n = sum(lengths)
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(n, 512, generator=gen).bfloat16().to(dev)
    table = torch.randperm(3 * width, generator=gen).view(3, width).to(torch.int32).to(dev)
    cu = [0, 20, 21, 98]
    seqlens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    positions = torch.cat([torch.arange(k) for k in lengths]).to(torch.int32).to(dev)
    out_loc = torch.cat([table[b, :k] for b, k in enumerate(lengths)]).contiguous()
    results = []
    for paged in (False, True):
        pool = zb.attention.SlotKVPool([3], 3 * width, 2, 128, dev)
        zb.core.get_global_ctx().attn_backend = pool
        meta = zb.core.AttnMetadata(None if paged else positions, None if paged else out_loc, table, seqlens,
                                    torch.tensor(cu, dtype=torch.int32, device=dev) if paged else cu)
        reqs = [zb.core.Req(b, k) for b, k in enumerate(lengths)]
        with zb.core.forward_batch(zb.core.Batch(reqs=reqs, is_decode=False, attn_metadata=meta)):
            first = layer.forward(x)
        meta = zb.core.AttnMetadata(seqlens, table[torch.arange(3), seqlens.long()].contiguous(), table, seqlens + 1,
                                    torch.arange(4, dtype=torch.int32, device=dev) if paged else None)
        with zb.core.forward_batch(zb.core.Batch(reqs=reqs, is_decode=True, attn_metadata=meta)):
            second = layer.forward(x[:3].contiguous())
        results.append((first, second, pool.k_buffer.clone(), pool.v_buffer.clone()))
    for a, b in zip(results[0][:3], results[1][:3]):
        assert max_rel_err(b, a) <= 3e-2
    assert torch.equal(results[0][3], results[1][3])


def test_a_paged_pool_asks_for_device_lengths(zb):
    dev = torch.device("cuda")
    _, _, model = _model(zb, 4)
    layer = model.layers.op_list[3].attention
    zb.core.get_global_ctx().attn_backend = zb.attention.PagedKVPool([3], 4, 16, 2, 128, dev)
    one = torch.ones(1, dtype=torch.int32, device=dev)
    meta = zb.core.AttnMetadata(one - 1, one - 1, one[None] - 1, one, [0, 1])
    for decode in (False, True):
        with zb.core.forward_batch(zb.core.Batch(reqs=[zb.core.Req(0, 1)], is_decode=decode, attn_metadata=meta)):
            with pytest.raises(RuntimeError, match="device tensor"):
                layer.forward(torch.zeros(1, 512, device=dev, dtype=torch.bfloat16))
