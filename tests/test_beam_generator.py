"""What the generator's decode_mode "beam" hands to the search, refuses and returns. CPU
only: the searches themselves are in test_gpu_beam_generate.py."""
from types import SimpleNamespace

import pytest

from dtree_hip import api
from dtree_hip.adapters import LoadedTargetModel
from dtree_hip.beam import BeamHypothesis


class Tokenizer:
    eos_token_ids = {7, 9}

    def encode(self, text):
        return [len(w) for w in text.split()]

    def decode(self, tokens, skip_special_tokens=False):
        return " ".join(map(str, tokens))


@pytest.fixture
def generator(monkeypatch):
    target = LoadedTargetModel("random:custom", None, SimpleNamespace(args=None), None, SimpleNamespace(family="qwen3"))
    gen = api.DFlashGenerator(target_model=target, draft_model=object(), tokenizer=Tokenizer())
    gen.calls, gen.found = [], [BeamHypothesis([3, 7], -1.0, True)]

    def search(target, prompts, **kw):
        gen.calls.append(kw)
        return [gen.found], {"num_input_tokens": len(prompts[0])}

    monkeypatch.setattr(api, "beam_generate", search)
    return gen


def test_one_of_the_tokenizers_stop_tokens(generator):
    with pytest.raises(ValueError, match=r"\[7, 9\].*stop_token_ids"):
        generator.generate("a bb ccc", decode_mode="beam")
    assert not generator.calls
    res = generator.generate("a bb ccc", decode_mode="beam", num_beams=3, length_penalty=0.5, max_new_tokens=6,
                             stop_token_ids=[7])
    assert generator.calls == [dict(num_beams=3, max_new_tokens=6, stop_token_ids={7}, length_penalty=0.5)]
    assert res.output_tokens == [1, 2, 3, 3, 7] and res.generated_tokens == [3, 7] and res.text == "3 7"
    generator.generate_from_tokens([1], decode_mode="beam", stop_token_ids=())
    assert generator.calls[-1]["stop_token_ids"] == set()
    generator.target.tokenizer = None
    generator.generate_from_tokens([1], decode_mode="beam")
    assert generator.calls[-1]["stop_token_ids"] == set()


@pytest.mark.parametrize("mode", ["dflash", "dtree"])
def test_the_other_modes_take_any_number(generator, monkeypatch, mode):
    got = []

    def decode(target, draft, prompt_tokens, stop_token_ids, **kw):
        got.append(stop_token_ids)
        return [1], {"num_input_tokens": 1}

    monkeypatch.setattr(api, mode + "_generate", decode)
    generator.generate_from_tokens([1], decode_mode=mode)
    generator.generate_from_tokens([1], decode_mode=mode, stop_token_ids=[4, 5, 6])
    assert got == [{7, 9}, {4, 5, 6}]


def test_a_temperature_is_refused(generator):
    with pytest.raises(ValueError, match="temperature"):
        generator.generate("a", decode_mode="beam", temperature=0.7, stop_token_ids=[7])
    assert not generator.calls


def test_no_continuation(generator):
    generator.found = []
    with pytest.raises(RuntimeError, match="no token continues"):
        generator.generate("a", decode_mode="beam", stop_token_ids=[7])
