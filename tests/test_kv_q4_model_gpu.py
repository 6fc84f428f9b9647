"""GPU: the attention module, the whole model and its captured decode step over a KV cache of 4 bits, and windows with first tokens
kept, through the module.

The module against the oracles on its own projection: queries from oracle.paged.append, keys and values as the pool stands for
them. Bar as between the module's other paths (tests/test_paged_model_gpu.py): q, the weights, the output and its product round to
bf16 a few times, 3e-2 of the largest value. A captured step against the same step run eagerly: the same kernels, equal bit by bit."""

from __future__ import annotations

import dataclasses

import pytest
import torch
import torch.nn.functional as F

from conftest import max_rel_err
from oracle import lm as olm
from oracle import paged, paged_q4
from test_model_gpu import _configs

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _model(zb, seed, **change):
    oc, mc = _configs(zb)
    model = zb.model.Zonos3ForCausalLM(dataclasses.replace(mc, **change))
    model.load_state_dict(dict(olm.random_weights(oc, seed=seed)))
    model.to(torch.device(DEV), torch.bfloat16)
    return model


def _table(gen, streams, pages, total):
    return torch.randperm(total, generator=gen)[: streams * pages].view(streams, pages).to(torch.int32).to(DEV)


@pytest.mark.parametrize("bits,change", [(4, {}), (4, dict(attention_window=24, attention_sinks=3)),
                                         (16, dict(attention_window=24, attention_sinks=3))])
def test_attention_module_matches_oracle(zb, bits, change):
    """A ragged batch of prompts, then one of single tokens, then one that mixes them."""
    model = _model(zb, 4, **change)
    layer = model.layers.op_list[3].attention
    pool = model.allocate_caches(4, 40 * 16, DEV, page_size=16, kv_bits=bits)
    zb.core.get_global_ctx().attn_backend = pool
    gen = torch.Generator().manual_seed(7)
    table = _table(gen, 3, 9, 40)
    lengths = [0, 0, 0]
    for news in ([20, 1, 77], [1, 1, 1], [30, 1, 0]):
        n = sum(news)
        lengths = [a + b for a, b in zip(lengths, news)]
        cu = torch.tensor([0, news[0], news[0] + news[1], n], dtype=torch.int32)
        seqlens = torch.tensor(lengths, dtype=torch.int32)
        x = torch.randn(n, 512, generator=gen).bfloat16().to(DEV)
        meta = zb.core.AttnMetadata(None, None, table, seqlens.to(DEV), cu.to(DEV))
        batch = zb.core.Batch(reqs=[zb.core.Req(b, k) for b, k in enumerate(news)], is_decode=max(news) == 1, attn_metadata=meta)
        with zb.core.forward_batch(batch):
            got = layer.forward(x)
        p = F.linear(x, layer._proj).cpu()
        if bits == 4:
            k, v = paged_q4.read(pool.kv(3).cpu())
        else:
            k, v = pool.k(3).cpu().double(), pool.v(3).cpu().double()
        q = paged.append(p, k.clone(), v.clone(), table.cpu(), seqlens, cu, heads=8, kv_heads=2, temp=layer._temp.cpu())[0]
        out = paged.chunk(q, k, v, table.cpu(), seqlens, cu, window=change.get("attention_window", 0),
                          sinks=change.get("attention_sinks", 0), gate=p[:, 12 * 128:])[0]
        assert max_rel_err(got, out.flatten(1) @ layer.wo.weight.double().cpu().t()) <= 3e-2
    assert zb.ops.device_status() == 0


@pytest.mark.parametrize("change", [{}, dict(attention_window=20, attention_sinks=2)])
@pytest.mark.parametrize("bits", [4, 16])
def test_captured_decode_step_is_the_eager_one(zb, bits, change):
    """Replays of the captured step over a pool of 4 bits (and over a slot pool with a window) against the step run eagerly, from
    the same streams; lengths advance and stop at what the table has pages for."""
    model = _model(zb, 5, **change)
    streams, tokens = 6, 64
    page = 16 if bits == 4 else 1
    pool = model.allocate_caches(streams, streams * tokens, DEV, kv_bits=bits)
    gen = torch.Generator().manual_seed(8)
    table = _table(gen, streams, tokens // page, streams * tokens // page)
    sampling = zb.model.SamplingConfig(temperature=0.0, repetition_window=0, repetition_penalty=1.0)
    graph = zb.model.DecodeGraph(model, pool, streams, table, sampling=sampling)
    graph.capture()
    caches = [pool.buffer] if bits == 4 else [pool.k_buffer, pool.v_buffer]
    states = caches + [t for g in model.gdn_layers() for t in (g._recurrent_state, g._conv_state)]
    lengths = torch.tensor([1, 9, 33, 40, 63, 64], dtype=torch.int32, device=DEV)
    ids = torch.cat([torch.randint(0, 4096, (streams, 10), generator=gen), torch.randint(0, 1024, (streams, 1), generator=gen)], 1)
    ids = ids.to(torch.int32).to(DEV)
    out_loc = table[torch.arange(streams), ((lengths - 1) // page).long()] if bits == 16 else lengths - 1
    if bits == 4:  # keys and values in every page
        rows = torch.randn(streams * tokens, 4 * 128, generator=gen).bfloat16().to(DEV)
        full = torch.full((streams,), tokens, dtype=torch.int32, device=DEV)
        cu = (torch.arange(streams + 1) * tokens).to(torch.int32).to(DEV)
        zb.ops.gqa_append_q4(rows, pool.kv(3), table, full, cu, heads=0, kv_heads=2)
    else:
        for t in caches:
            t.copy_(torch.randn(t.shape, generator=gen))
    start = [t.clone() for t in states]
    results = []
    for replay in (True, False):
        for t, s in zip(states, start):
            t.copy_(s)
        graph.reset()
        graph.load(ids, lengths - 1, lengths, out_loc.contiguous())
        steps = []
        for _ in range(3):
            if replay:
                graph.replay()
            else:
                with graph._context():
                    graph._body()
            steps.append([graph.logits.clone(), graph.codes.clone(), graph.cache_seqlens.clone(), *(t.clone() for t in states)])
        results.append(steps)
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert results[0][2][2].tolist() == [4, 12, 36, 43, 64, 64]
    assert not torch.equal(results[0][0][3], start[0]) and zb.ops.device_status() == 0


def test_what_asks_for_device_lengths_says_so(zb):
    model = _model(zb, 4)
    layer = model.layers.op_list[3].attention
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    meta = zb.core.AttnMetadata(one - 1, one - 1, one[None] - 1, one, [0, 1])
    x = torch.zeros(1, 512, device=DEV, dtype=torch.bfloat16)
    windowed = _model(zb, 4, attention_window=9).layers.op_list[3].attention
    for attention, pool in ((layer, zb.attention.QuantKVPool([3], 4, 16, 2, 128, DEV)),
                            (windowed, zb.attention.SlotKVPool([3], 64, 2, 128, DEV))):
        zb.core.get_global_ctx().attn_backend = pool
        for decode in (False, True):
            with zb.core.forward_batch(zb.core.Batch(reqs=[zb.core.Req(0, 1)], is_decode=decode, attn_metadata=meta)):
                with pytest.raises(RuntimeError, match="device tensor"):
                    attention.forward(x)
    with pytest.raises(ValueError, match="kv_bits"):
        model.allocate_caches(1, 64, DEV, kv_bits=8)
