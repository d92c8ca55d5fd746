"""The generator's beam mode with a tokenizer of two end tokens, and logits without a number."""
import pytest

from dtree_hip.adapters import load_target_model
from dtree_hip.api import DFlashGenerator
from dtree_hip.config import tiny_qwen3, tiny_qwen35

pytestmark = pytest.mark.gpu


class Tokenizer:
    def __init__(self, ends):
        self.eos_token_ids = ends

    def encode(self, text):
        return [3 + ord(c) % 50 for c in text]

    def decode(self, tokens, skip_special_tokens=False):
        return ",".join(map(str, tokens))


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
def test_a_tokenizer_with_two_end_tokens(gpu_device, family):
    target = load_target_model(tiny_qwen3() if family == "qwen3" else tiny_qwen35(), seed=0, max_past=200, norm_jitter=0.1,
                               kv_bits=8)
    gen = DFlashGenerator(target_model=target, draft_model=object())
    prompt = Tokenizer(()).encode("a prompt of some characters")
    free = gen.generate_from_tokens(prompt, max_new_tokens=12, decode_mode="beam", num_beams=1).generated_tokens
    end = free[5]
    gen.target.tokenizer = Tokenizer({end, target.model.args.vocab_size - 1})
    with pytest.raises(ValueError, match="stop_token_ids"):
        gen.generate("a prompt of some characters", max_new_tokens=12, decode_mode="beam", num_beams=1)
    res = gen.generate("a prompt of some characters", max_new_tokens=12, decode_mode="beam", num_beams=1, stop_token_ids={end})
    assert res.generated_tokens == free[:free.index(end) + 1]
    assert res.metrics["hypotheses"][0].finished and res.text == ",".join(map(str, res.generated_tokens))


def test_logits_of_nan(gpu_device):
    target = load_target_model(tiny_qwen3(), seed=0, max_past=200, kv_bits=8)
    target.model.weights.final_norm.fill_(float("nan"))
    gen = DFlashGenerator(target_model=target, draft_model=object())
    with pytest.raises(RuntimeError, match="no token continues"):
        gen.generate_from_tokens([5, 6, 7], max_new_tokens=4, decode_mode="beam", num_beams=3)
