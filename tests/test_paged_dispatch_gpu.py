"""GPU: which kernels the attention module takes for a batch's metadata. A batch that the module ran before it knew paged
batches keeps its kernels, so its results are equal bit by bit, whatever form its ``cu_seqlens_q`` comes in."""

from __future__ import annotations

import pytest
import torch

from conftest import max_rel_err
from test_paged_model_gpu import _model

pytestmark = pytest.mark.gpu

LENGTHS, WIDTH = [20, 1, 77], 80


@pytest.fixture(scope="module")
def layer(zb):
    return _model(zb, 4)[2].layers.op_list[3].attention


def _prefill(zb, layer, form):
    """Output and caches of a prefill of LENGTHS, its bounds in the given form, over the slot pool."""
    dev = torch.device("cuda")
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(sum(LENGTHS), 512, generator=gen).bfloat16().to(dev)
    table = torch.randperm(3 * WIDTH, generator=gen).view(3, WIDTH).to(torch.int32).to(dev)
    positions = torch.cat([torch.arange(k) for k in LENGTHS]).to(torch.int32).to(dev)
    out_loc = torch.cat([table[b, :k] for b, k in enumerate(LENGTHS)]).contiguous()
    pool = zb.attention.SlotKVPool([3], 3 * WIDTH, 2, 128, dev)
    zb.core.get_global_ctx().attn_backend = pool
    seqlens = torch.tensor(LENGTHS, dtype=torch.int32, device=dev)
    meta = zb.core.AttnMetadata(positions, out_loc, table, seqlens, form([0, 20, 21, 98]))
    reqs = [zb.core.Req(b, k) for b, k in enumerate(LENGTHS)]
    with zb.core.forward_batch(zb.core.Batch(reqs=reqs, is_decode=False, attn_metadata=meta)):
        return layer.forward(x), pool, table, seqlens, reqs, x


@pytest.mark.parametrize("form", [lambda cu: torch.tensor(cu, dtype=torch.int32), lambda cu: torch.tensor(cu),
                                  lambda cu: torch.tensor(cu, device="cuda"), tuple])
def test_prefill_bounds_in_other_forms_take_the_host_path(zb, layer, form):
    expected, pool, *_ = _prefill(zb, layer, list)
    got, pool2, *_ = _prefill(zb, layer, form)
    assert torch.equal(got, expected)
    assert torch.equal(pool2.k_buffer, pool.k_buffer) and torch.equal(pool2.v_buffer, pool.v_buffer)


@pytest.mark.parametrize("form", [list, lambda cu: torch.tensor(cu, dtype=torch.int32),
                                  lambda cu: torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                  lambda cu: torch.tensor(cu, device="cuda")])
def test_decode_with_bounds_keeps_the_decode_kernels(zb, layer, form):
    """A decode batch over the slot pool, its slots and positions given: bounds beside them change nothing."""
    results = []
    for bounds in (None, form([0, 1, 2, 3])):
        _, pool, table, seqlens, reqs, x = _prefill(zb, layer, list)
        loc = table[torch.arange(3), seqlens.long()].contiguous()
        meta = zb.core.AttnMetadata(seqlens, loc, table, seqlens + 1, bounds)
        with zb.core.forward_batch(zb.core.Batch(reqs=reqs, is_decode=True, attn_metadata=meta)):
            results.append((layer.forward(x[:3].contiguous()), pool.k_buffer))
    assert torch.equal(results[1][0], results[0][0]) and torch.equal(results[1][1], results[0][1])


def test_decode_without_slots_runs_the_paged_operators(zb, layer):
    """With device bounds alone (no positions, no slots) a decode batch is a batch like any other; q and k are rounded once
    instead of up to three times, so outputs differ by a few bf16 units (3e-2 of the largest, as between the prefills)."""
    outs = []
    for paged in (False, True):
        _, _, table, seqlens, reqs, x = _prefill(zb, layer, list)
        loc = table[torch.arange(3), seqlens.long()].contiguous()
        bounds = torch.arange(4, dtype=torch.int32, device="cuda")
        meta = zb.core.AttnMetadata(*((None, None) if paged else (seqlens, loc)), table, seqlens + 1, bounds)
        with zb.core.forward_batch(zb.core.Batch(reqs=reqs, is_decode=True, attn_metadata=meta)):
            outs.append(layer.forward(x[:3].contiguous()))
    assert max_rel_err(outs[1], outs[0]) <= 3e-2
