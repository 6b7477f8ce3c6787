"""Model configurations are given by position too: fields keep their places, new ones go to the end."""
import dataclasses

from transformerengine_b200.models.llama import LlamaConfig
from transformerengine_b200.models.mistral import MistralConfig
from transformerengine_b200.models.qwen import Qwen3Config

FIELDS = ["vocab_size", "hidden_size", "num_layers", "num_heads", "num_kv_heads", "ffn_hidden_size", "rms_eps", "rope_theta", "init_std",
          "params_dtype", "recompute", "quantize_lm_head", "head_dim", "activation", "zero_centered_gamma", "embedding_scale",
          "tie_embeddings", "sliding_window", "qk_norm", "qk_norm_eps"]


def test_fields_keep_their_positions():
    for cls in (LlamaConfig, MistralConfig, Qwen3Config):
        assert [f.name for f in dataclasses.fields(cls)][:len(FIELDS)] == FIELDS
    by_place = LlamaConfig(*[getattr(LlamaConfig(), n) for n in FIELDS[:-2]], True, 1e-5)
    assert by_place.qk_norm is True and by_place.qk_norm_eps == 1e-5 and by_place.sink_tokens == 0
