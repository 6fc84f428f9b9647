"""What the paged-cache entry points and the model refuse before any launch, and what they say (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


def test_decode_graph_refuses_a_paged_pool(zb):
    """Before it changes the model: the layers' static mode is set up after the check."""
    model = SimpleNamespace(attention_layer_ids=lambda: [3])
    pool = zb.attention.PagedKVPool([3], 4, 16, 2, 128, "cpu")
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="page size 1"):
        zb.model.DecodeGraph(model, pool, 2, table)
