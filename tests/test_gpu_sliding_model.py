"""A patched Hugging Face model whose layers have a sliding window: prefill and decoding against eager attention."""
import json

import pytest
import torch

from shareprefill_b200 import SharePrefill
from shareprefill_b200.workloads import synthetic_lookup

pytestmark = pytest.mark.gpu

WINDOW = 70


def _tiny_qwen(dtype):
    from transformers import Qwen2Config, Qwen2ForCausalLM
    cfg = Qwen2Config(vocab_size=128, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=4096, use_sliding_window=True, sliding_window=WINDOW,
                      max_window_layers=1, attn_implementation="eager")
    assert cfg.layer_types == ["full_attention", "sliding_attention", "sliding_attention"]
    torch.manual_seed(0)
    return Qwen2ForCausalLM(cfg).to(dtype).cuda().eval()


def _patched(model, tmp_path):
    p = tmp_path / "l.json"
    p.write_text(json.dumps(synthetic_lookup(3, 4, 2, group_size=2)))
    return SharePrefill(model_name="tiny", sharing_lookup_path=str(p), block_size=64, min_budget=4096)(model)


def test_prefill_with_windowed_layers_matches_eager(tmp_path):
    model = _tiny_qwen(torch.bfloat16)
    ids = torch.randint(0, 128, (1, 700), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        want = model(ids).logits.float()
        got = _patched(model, tmp_path)(ids).logits.float()
    # three layers of bf16 activations whose roundings (2^-8 each) differ between two orders of summation, as in the
    # test of the dense layers
    err = (got - want).abs()
    assert err.max() < 0.15 and err.mean() < 0.01, (err.max().item(), err.mean().item())


def test_decoding_behind_a_sliding_cache_matches_eager(tmp_path):
    model = _tiny_qwen(torch.bfloat16)
    ids = torch.randint(0, 128, (1, 150), generator=torch.Generator().manual_seed(2)).cuda()
    steps = torch.randint(0, 128, (6,), generator=torch.Generator().manual_seed(3)).tolist()

    def logits(m):
        out, cache = [], None
        with torch.no_grad():
            r = m(ids, use_cache=True)
            for t in steps:
                out.append(r.logits[:, -1].float())
                cache = r.past_key_values
                r = m(torch.tensor([[t]], device="cuda"), past_key_values=cache, use_cache=True)
        return torch.stack(out + [r.logits[:, -1].float()])

    want = logits(model)
    got = logits(_patched(model, tmp_path))
    err = (got - want).abs()
    assert err.max() < 0.15 and err.mean() < 0.01, (err.max().item(), err.mean().item())


@pytest.mark.parametrize("prompt,cached,refused", [(150, "static", False), (30, "static", True), (30, "dynamic", False), (1, "static", True), (1, "dynamic", False)])
def test_caches_of_a_fixed_size_are_served_when_full_and_refused_before(tmp_path, prompt, cached, refused):
    from transformers import DynamicCache, Qwen2Config, Qwen2ForCausalLM, StaticCache

    from shareprefill_b200 import native
    cfg = Qwen2Config(vocab_size=128, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=4096, use_sliding_window=True, sliding_window=WINDOW,
                      max_window_layers=0, attn_implementation="eager")
    assert set(cfg.layer_types) == {"sliding_attention"}
    torch.manual_seed(0)
    model = Qwen2ForCausalLM(cfg).to(torch.bfloat16).cuda().eval()
    ids = torch.randint(0, 128, (1, prompt + 5), generator=torch.Generator().manual_seed(4)).cuda()

    def logits():
        cache = StaticCache(config=cfg, max_cache_len=400) if cached == "static" else DynamicCache(config=cfg)
        with torch.no_grad():
            out = [model(ids[:, :prompt], past_key_values=cache).logits[:, -1].float()]
            for i in range(prompt, prompt + 5):
                out.append(model(ids[:, i:i + 1], None, None, cache).logits[:, -1].float())      # (also by position)
        return torch.stack(out)

    want = logits()
    p = tmp_path / "l.json"
    p.write_text(json.dumps(synthetic_lookup(2, 4, 2, group_size=2)))
    model = SharePrefill(model_name="tiny", sharing_lookup_path=str(p), block_size=64, min_budget=4096)(model)
    if refused:
        # a prompt of 30 tokens meets 70 keys; one token could pass for a step behind 69
        with pytest.raises((NotImplementedError, native.SpfError), match="sliding window"):
            logits()
        return
    err = (logits() - want).abs()
    assert err.max() < 0.15 and err.mean() < 0.01, (err.max().item(), err.mean().item())
    assert model.attention_sharing.tokens_so_far is None          # a call of the decoder by itself is not measured by it
    with torch.no_grad():
        assert torch.isfinite(model.model(torch.zeros(1, 400, dtype=torch.int64, device="cuda")).last_hidden_state).all()
