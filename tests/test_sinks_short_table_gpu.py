"""GPU: a window with first keys kept where the page table ends before the window begins: the first keys alone are seen, all of them
that the table holds, in whatever tile they lie (the window would begin in the last of theirs). Tolerances: those of
tests/test_gqa_paged_gpu.py and tests/test_kv_q4_gpu.py."""

from __future__ import annotations

import pytest
import torch

import test_gqa_paged_gpu as bf16
import test_kv_q4_gpu as q4

pytestmark = pytest.mark.gpu


def _cut(x, columns, keys):
    """The same pages in a table of ``columns``; requests of ``keys`` keys."""
    *head, table, seqlens, cu = x
    return *head, table[:, :columns].contiguous(), torch.tensor(keys, dtype=torch.int32), cu


# what the table holds, the requests' keys, window, first keys; rows of the first two requests stand behind the table's end
CASES = [(144, [300, 330, 150], 60, 140), (272, [300, 500, 200], 20, 259), (144, [161, 400, 144], 3, 150), (400, [700, 450, 90], 30, 399),
         (128, [200, 260, 130], 40, 100)]


@pytest.mark.parametrize("held,keys,window,sinks", CASES)
@pytest.mark.parametrize("news", [[1, 3, 1], [20, 40, 1]])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_first_keys_alone(zb, held, keys, window, sinks, news, hd):
    gen = torch.Generator().manual_seed(held + window)
    x = q4._chunk_inputs(gen, news, [held] * 3, 8, 2, hd, 16)
    q4._check_chunk(zb, *_cut(x, held // 16, keys), window=window, sinks=sinks)
    for page in (1, 8, 16):
        x = bf16._chunk_inputs(gen, news, [held] * 3, 8, 2, hd, page)
        bf16._check_chunk(zb, *_cut(x, held // page, keys), window=window, sinks=sinks)
