"""Checkpoints whose matrices are 8-bit values beside scales are refused before anything of them is taken: the loaders read no scales, and the values alone are other weights."""
import pytest
import torch


def state(cfg, dtype):
    H, I, hd, g = cfg.hidden_size, cfg.intermediate_size, cfg.head_dim, torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g) * 0.02
    sd = {"model.embed_tokens.weight": rnd(cfg.vocab_size, H), "model.norm.weight": torch.ones(H), "lm_head.weight": rnd(cfg.vocab_size, H)}
    for i in range(cfg.num_hidden_layers):
        pre = f"model.layers.{i}."
        for n, heads in (("q", cfg.num_attention_heads), ("k", cfg.num_key_value_heads), ("v", cfg.num_key_value_heads)):
            sd[pre + f"self_attn.{n}_proj.weight"], sd[pre + f"self_attn.{n}_proj.bias"] = rnd(heads * hd, H).to(dtype), rnd(heads * hd)
        sd[pre + "self_attn.o_proj.weight"] = rnd(H, cfg.num_attention_heads * hd).to(dtype)
        sd[pre + "mlp.gate_proj.weight"], sd[pre + "mlp.up_proj.weight"], sd[pre + "mlp.down_proj.weight"] = rnd(I, H).to(dtype), rnd(I, H).to(dtype), rnd(H, I).to(dtype)
        sd[pre + "input_layernorm.weight"], sd[pre + "post_attention_layernorm.weight"] = torch.ones(H), torch.ones(H)
    return sd


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("files", [False, True])
def test_loaders(tmp_path, dtype, files):
    from safetensors.torch import save_file
    from jacobiforcing_amd.modeling.qwen2 import Qwen2Config, Qwen2Weights
    cfg = Qwen2Config.tiny()
    sd, w = state(cfg, dtype), Qwen2Weights(cfg, "cpu", dtype=torch.float32)
    before, w.fp8 = w.embed, True
    if files:
        save_file(sd, str(tmp_path / "model.safetensors"))
    load = (lambda: w.load_safetensors(str(tmp_path), cfg)) if files else (lambda: w.load_state_dict(sd, cfg))
    if dtype.itemsize == 1:
        with pytest.raises(ValueError, match="8-bit"):
            load()
        assert w.embed is before and w.fp8              # as they were
    else:
        load()
        assert not w.fp8 and torch.equal(w.layers[1]["wd"], sd["model.layers.1.mlp.down_proj.weight"].float())
