"""GPU: edges of the paged-cache operators: values near the ends of bf16's range, workspaces that several calls share,
batches whose bounds are wrong, arguments past 32 bits.

Tolerances are those of tests/test_gqa_paged_gpu.py. Where scores are tens of nats large their own error counts beside
the roundings to bf16: a score is off by at most hd 2^-23 scale sum_d |q_d k_d| (``size`` of the oracle) and 2^-15 for its
exponential, and it moves both a weight and the sum that divides it."""

from __future__ import annotations

import pytest
import torch

from oracle import paged
from test_gqa_paged_gpu import DEV, _chunk_inputs, _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news, caches", [([1, 1], [700, 130]), ([40, 200], [300, 0]), ([300], [600]), ([1], [6000])])
@pytest.mark.parametrize("offset", [-60.0, -20.0, 0.0, 20.0, 60.0])
@pytest.mark.parametrize("binade", [-100, 0, 100])
def test_chunk_values_of_any_size(zb, news, caches, offset, binade):
    """Values of 2^100 and 2^-100 under scores around ``offset`` nats: the output is a mean of them, so it is neither
    infinite nor 0."""
    gen = torch.Generator().manual_seed(int(offset) + binade + len(news))
    hd = 64 if len(news) == 1 else 128
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, news, caches, 8, 2, hd, 16)
    if offset:  # one dim adds the offset to every score
        q[..., 0] = 8.0
        k[..., 0] = offset * hd ** 0.5 / 8.0
    v = (v.float() * 2.0 ** binade).bfloat16()
    lse = torch.empty(q.shape[:2], device=DEV)
    out = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), lse=lse)
    ref, spread, ref_lse, size = paged.chunk(q, k, v, table, seqlens, cu)
    score = hd * 2.0 ** -23 * size + 2.0 ** -15
    _close(out, ref, spread * (2.0 ** -7 * (1 + 2.0 ** -4) + 2 * score[..., None]))
    _close(lse, ref_lse, score)
    assert zb.ops.device_status() == 0
