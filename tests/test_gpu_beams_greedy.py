"""One beam is greedy generation: the same ids, whatever penalty, and a score that is the sum of their log probabilities."""
import pytest
import torch

from conftest import small_cfg
from seedplane_amd.qwen_engine import Qwen2Engine
from seedplane_amd.synth import make_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    cfg, w = make_weights(small_cfg(), 'q8', seed=3)
    return Qwen2Engine(config=cfg, tensors=w, max_tokens=16)


@pytest.mark.parametrize('n,steps,penalty', [(1, 1, 1.0), (9, 8, 1.0), (40, 20, 0.0), (16, 5, 0.7)])
def test_one_beam_is_greedy(gpu_device, engine, n, steps, penalty):
    prompt = torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    want = list(engine.generate(prompt, steps))
    got = engine.generate_beams(prompt, beams=1, max_new_tokens=steps, length_penalty=penalty)
    assert [ids for ids, _ in got] == [want]
    logits = engine.forward(prompt + want[:-1], all_logits=True)[0].double().cpu()[n - 1:]
    score = sum(float(torch.log_softmax(row, -1)[t]) for row, t in zip(logits, want)) / steps ** penalty
    # (fp16 activations: logits of the wide pass and of single steps within 2e-2 of each other, so log probabilities within 4e-2)
    assert abs(got[0][1] - score) <= 4e-2 * steps / steps ** penalty
