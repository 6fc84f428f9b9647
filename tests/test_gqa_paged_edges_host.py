"""What the paged-cache entry points and the model refuse before any launch, and what they say (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from test_gqa_paged_host import SHARED, _append, _chunk


def test_decode_graph_refuses_a_paged_pool(zb):
    """Before it changes the model: the layers' static mode is set up after the check."""
    model = SimpleNamespace(attention_layer_ids=lambda: [3])
    pool = zb.attention.PagedKVPool([3], 4, 16, 2, 128, "cpu")
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="page size 1"):
        zb.model.DecodeGraph(model, pool, 2, table)


@pytest.mark.parametrize("change", SHARED)
def test_errors_name_their_entry_point(zb, change):
    lib = zb._lib.load()
    for call, name in ((_chunk, "gqa_chunk"), (_append, "gqa_append")):
        assert call(lib, **change) == 1
        assert name in zb._lib.last_error()
