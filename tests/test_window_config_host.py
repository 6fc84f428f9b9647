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


def _graph(zb, config, pool):
    """A decode graph that is not captured: its buffers, on the CPU."""
    model = zb.model.Zonos3ForCausalLM(zb.config.ModelConfig(512, num_layers=4, moe_n_experts=4, moe_topk=2, moe_intermediate_size=64,
                                                             num_qo_heads=4, num_kv_heads=2))
    model._config = config
    return zb.model.DecodeGraph(model, pool, 3, torch.zeros(3, 8, dtype=torch.int32))


def test_a_config_without_the_fields_decodes(zb):
    whole = zb.config.ModelConfig(512, num_layers=4, num_qo_heads=4, num_kv_heads=2)
    known = {f.name: getattr(whole, f.name) for f in dataclasses.fields(whole) if not f.name.startswith("attention_window")}
    known.pop("attention_sinks")
    config = types.SimpleNamespace(**known, audio_vocab_size=whole.audio_vocab_size)
    pool = zb.attention.SlotKVPool([3], 64, 2, 128, "cpu")
    assert _graph(zb, config, pool).bounds is None
    config.attention_window = 9
    assert _graph(zb, config, pool).bounds.tolist() == [0, 1, 2, 3]
