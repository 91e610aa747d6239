"""Weights with norms of queries and keys per head for models without them, and the other way round."""
import numpy as np
import pytest

from denograd_amd import synthetic
from denograd_amd.llama3 import MODEL_PARAMS, Llama3
from denograd_amd.state import safe_save
from tests.test_gpu_paged_model import cache_for, logits

CFG = synthetic.config("tiny16")


def named(qk_norm):
    """A model of these args as far as load_weights looks before it asks for a device."""
    llm = Llama3.__new__(Llama3)
    llm.params = {"n_layers": CFG["n_layers"], **({} if qk_norm is None else {"qk_norm": qk_norm})}
    return llm


def test_norms_that_the_model_does_not_have():
    """A checkpoint with them, loaded by default settings, would answer without its norms."""
    with pytest.raises(KeyError, match="layers.0.attention.k_norm.weight: .*qk_norm=True"):
        named(None).load_weights(synthetic.random_state_dict(dict(CFG, qk_norm=True), seed=1))
    with pytest.raises(KeyError, match="layers.3.attention.q_norm.weight"):
        named(None).load_weights({"layers.3.attention.q_norm.weight": np.ones(64, np.float16)}, quantized=True)
    assert not any("qk_norm" in MODEL_PARAMS[size]["args"] for size in MODEL_PARAMS)


def test_norms_that_the_weights_do_not_have():
    sd = synthetic.random_state_dict(dict(CFG, qk_norm=True), seed=1)
    del sd["layers.1.attention.k_norm.weight"]
    with pytest.raises(KeyError, match="layers.1.attention.k_norm.weight missing"):
        named(True).load_weights(sd)
    with pytest.raises(KeyError, match="layers.0.attention.k_norm.weight missing"):
        named(True).load_weights(synthetic.random_state_dict(CFG, seed=1))


@pytest.mark.gpu
def test_a_file_with_norms(hip, tmp_path):
    """In Hugging Face names: refused where nothing is said of norms, loaded with and without them where it is; the rotate-half order is undone for projections and norms alike."""
    cfg = dict(CFG, qk_norm=True, max_context=256)
    sd, rng, hd = synthetic.random_state_dict(cfg, seed=3, std=0.05), np.random.default_rng(1), 64
    half = np.concatenate([np.arange(0, hd, 2), np.arange(1, hd, 2)])                # rotate-half from interleaved
    names = {"wq": "q_proj", "wk": "k_proj", "wv": "v_proj", "wo": "o_proj", "w1": "gate_proj", "w2": "down_proj", "w3": "up_proj", "q_norm": "q_norm", "k_norm": "k_norm"}
    file = {"model.embed_tokens.weight": sd["tok_embeddings.weight"], "model.norm.weight": sd["norm.weight"], "lm_head.weight": sd["output.weight"].copy()}
    for k in list(sd):
        if not k.startswith("layers."):
            continue
        _, l, part, *rest = k.split(".")
        if "q_norm" in k or "k_norm" in k:
            sd[k] = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float16)
            file[f"model.layers.{l}.self_attn.{rest[0]}.weight"] = sd[k][half]
        elif part in ("attention", "feed_forward"):
            w = sd[k]
            if rest[0] in ("wq", "wk"):
                w = w.reshape(-1, hd, w.shape[1])[:, half].reshape(w.shape)
            file[f"model.layers.{l}.{'self_attn' if part == 'attention' else 'mlp'}.{names[rest[0]]}.weight"] = w
        else:
            file[f"model.layers.{l}.{ {'attention_norm': 'input_layernorm', 'ffn_norm': 'post_attention_layernorm'}[part] }.weight"] = sd[k]
    fn = str(tmp_path / "model.safetensors")
    safe_save({k: np.ascontiguousarray(v) for k, v in file.items()}, fn)
    toks, out = [np.arange(9, dtype=np.int32)], []
    with pytest.raises(KeyError, match="qk_norm=True"):
        Llama3.from_config({k: v for k, v in cfg.items() if k != "qk_norm"}).load(fn)
    for llm in (Llama3.from_config(cfg).load(fn), Llama3.from_config(cfg).load_weights(sd), Llama3.from_config(dict(cfg, qk_norm=False)).load(fn)):
        cache = cache_for(llm, 4)
        llm.model.forward_paged(cache, [cache.add()], toks)
        out.append(logits(llm.model, 1))
    assert np.array_equal(out[0], out[1]) and np.abs(out[2] - out[0]).max() > 0.05 * np.abs(out[0]).max()
