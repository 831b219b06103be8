"""The decode products (k_gemv) of matrices whose rows are no multiple of a wave's rows: the LM head of a
model without layers, logits = out . (rmsnorm(x) * output_norm), against 64 bits."""
import numpy as np
import pytest

import gmoe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 129, 130, 131, 132])
def test_lm_head_of_any_vocabulary(vocab):
    cfg = dict(dim=64, hidden_dim=64, n_layers=1, n_heads=1, vocab_size=vocab, q_lora_rank=64, kv_lora_rank=64, rope_dim=16,
               qk_nope_dim=32, head_k_dim=48, v_head_dim=32, group_size=32, cache_cap=4, attn_layers=0, has_l0_ffn=0, max_batch=1)
    g, _ = gmoe.synth_model_weights(cfg, vocab)
    weights = {n: (g[n + "_q"].reshape(vocab, 2, 32) * g[n + "_s"].astype(np.float64)[..., None]).reshape(vocab, 64) for n in ("tok", "out")}
    print(f"[case] {vocab} rows", flush=True)
    model = gmoe.Model(cfg)
    try:
        model.upload(g)
        for token in {0, vocab - 1}:
            x = weights["tok"][token]
            h = x / np.sqrt((x * x).mean() + 1e-5) * g["output_norm"]
            got = model.forward_token(token, 0)
            # 64 products and 70 sums and factors, each rounded by 2^-24 of the terms' magnitudes
            assert (np.abs(got - weights["out"] @ h) <= 140 * 2.0 ** -24 * (np.abs(weights["out"]) @ np.abs(h))).all()
    finally:
        model.close()
