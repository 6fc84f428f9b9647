"""The decode step's bookkeeping takes one page-table row for all streams, and a decode graph over 4 bits keeps no table of slots for
each stream."""

from __future__ import annotations

import ctypes

import torch

from test_window_config_host import _graph

P, N = ctypes.c_void_p(256), None


def test_a_decode_graph_over_4_bits_keeps_one_row(zb):
    pool = zb.attention.QuantKVPool([3], 8, 16, 2, 128, "cpu")
    graph = _graph(zb, zb.config.ModelConfig(512, num_layers=4, num_qo_heads=4, num_kv_heads=2), pool)
    assert graph._slot_table.shape == (3, 8 * 16) and graph._slot_table.untyped_storage().nbytes() == 8 * 16 * 4


def test_table_strides(zb):
    """0 or at least a row's length; nothing is launched for no streams."""
    lib = zb._lib.load()

    def call(stride):
        return lib.zb_decode_advance(P, 11, P, 11, N, 0, 0, N, P, P, P, P, P, stride, 64, 0, N)

    assert call(0) == 0 and call(64) == 0 and call(63) == 1 and call(-1) == 1
