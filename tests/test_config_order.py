"""``Config`` by position: a field that came later stands behind those that were there."""
import json


def test_fields_by_position(tmp_path):
    from jacobiforcing_amd.config import Config
    (tmp_path / "config.json").write_text(json.dumps(dict(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                                          rms_norm_eps=1e-6, rope_theta=1e4, max_position_embeddings=1024, eos_token_id=511, pad_token_id=510)))
    c = Config(str(tmp_path), 1024, 8, 512, 0.5, 1, True, None, -1, -1, 512, 40, "paged", "float32", False, 32, 3, 0.25, 0.5, 6, 99)
    assert (c.max_num_batched_tokens, c.max_num_seqs, c.max_model_len, c.gpu_memory_utilization, c.enforce_eager, c.kvcache_block_size, c.num_kvcache_blocks) == (1024, 8, 512, 0.5, True, 512, 40)
    assert (c.kv_cache_layout, c.dtype) == ("paged", "float32")
    assert (c.jacobi_enabled, c.jacobi_block_len, c.jacobi_max_blocks, c.jacobi_spawn_ratio, c.jacobi_lookahead_start_ratio, c.jacobi_n_gram_pool_size, c.jacobi_max_iterations) == (False, 32, 3, 0.25, 0.5, 6, 99)
    assert c.quantization is None
