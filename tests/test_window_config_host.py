"""The window's fields of ModelConfig take nothing from callers that do not know them: positional arguments keep their places, and a
config object without the fields is one of layers that see all keys."""

from __future__ import annotations

import dataclasses
import types

import torch


def test_positional_arguments_keep_their_places(zb):
    """The fields from before the window's, in their order."""
    order = ["hidden_size", "num_layers", "rms_norm_eps", "gdn_num_heads", "gdn_head_dim", "moe_n_experts", "moe_topk",
             "moe_intermediate_size", "moe_alpha", "norm_topk_prob", "moe_router_type", "moe_balancing_strategy", "moe_router_use_eda",
             "moe_start_from_layer", "use_training_router_weights", "attention_pattern", "num_qo_heads", "num_kv_heads", "head_dim",
             "rope_theta", "intermediate_size", "n_codebooks", "codebook_size", "text_vocab", "text_extra_tokens", "audio_pad_id",
             "loss_softcap"]
    fields = [f.name for f in dataclasses.fields(zb.config.ModelConfig)]
    assert fields[: len(order)] == order
    values = list(dataclasses.astuple(zb.config.ModelConfig(512)))[: len(order)]
    values[order.index("intermediate_size")] = 4096
    config = zb.config.ModelConfig(*values)
    assert config.intermediate_size == 4096 and config.attention_window == config.attention_sinks == 0
