"""How the engine's steps choose their rows' tokens, captured and launched one by one, against the plain model."""

import pytest

from tests.helpers import TINY, make_model_folder, random_tokens
from tests.plain import llama
from tests.test_choices_gpu import check_answer, engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [262144, 262145])
@pytest.mark.parametrize("graphs", [False, True])
def test_top_p_on_either_side_of_the_kernels_largest_vocabulary(tmp_path, vocab, graphs):
    """A row that top-p cuts beside a greedy one and one that is drawn from all (logits of some 0.11 from token to token: low temperatures,
    so that no draw falls among tokens that weigh a millionth each)."""
    from tesseract_b200 import SamplingParams

    folder = make_model_folder(str(tmp_path), {**TINY["a"], "num_hidden_layers": 1, "hidden_size": 32, "intermediate_size": 64,
                                               "vocab_size": vocab}, "bfloat16", 3)
    config, tensors = llama.load_folder(folder)
    same = dict(max_tokens=4, ignore_eos=True)
    kinds = [SamplingParams(temperature=0.03, top_p=0.15, seed=8, **same), SamplingParams(temperature=0.0, **same),
             SamplingParams(temperature=0.02, seed=7, **same)]
    prompts = [random_tokens(vocab, n, seed=n) for n in (41, 3, 40)]
    outs = engine(folder, cuda_graphs=graphs).generate(prompts, kinds)
    for prompt, params, out in zip(prompts, kinds, outs):
        assert out.finish_reason == "length" and len(out.token_ids) == 4, out.error
        check_answer(config, tensors, prompt, params, out.token_ids)
