"""GPU: the runners' own stream against work that the caller's stream still has to do."""
import pytest
import torch

from slang_b200 import paged, runner, synth

pytestmark = pytest.mark.gpu


def _busy(dev):
    """A few tenths of a second of work for the current stream."""
    a = torch.full((8192, 8192), 1e-4, device=dev)
    for _ in range(16):
        a = a @ a
    return a


@pytest.fixture(scope="module")
def model(cuda):
    return runner.DeviceModel(synth.random_model(synth.small_config(), seed=81), cuda, 96)


PROMPTS = [synth.prompt_tokens(n, 2048, seed=n) for n in (21, 5, 13)]
SAMPLING = dict(temperature=[0.9, 1.2, 0.8], top_k=[0, 50, 0], top_p=[0.9, 1.0, 0.95], seeds=[3, 4, 5])


def _paged(dm):
    return paged.PagedRunner(dm, 3, n_pages=24, page_size=8)


def test_paged_runner_made_behind_a_busy_stream(cuda, model):
    """The runner's buffers are ready before its own stream uses them, however late the caller's stream is."""
    want = _paged(model).generate(PROMPTS, 8, **SAMPLING)
    _busy(cuda)  # loads what it needs
    torch.cuda.synchronize()
    _busy(cuda)
    assert _paged(model).generate(PROMPTS, 8, **SAMPLING) == want
    torch.cuda.synchronize()


def test_sampling_settings_from_a_busy_stream(cuda, model):
    """Settings may be tensors that the caller's stream is still to write."""
    r = _paged(model)
    want = r.generate(PROMPTS, 8, **SAMPLING)
    late = {k: torch.as_tensor(v, device=cuda) for k, v in SAMPLING.items()}
    mine = {k: torch.zeros_like(v) for k, v in late.items()}
    torch.cuda.synchronize()
    _busy(cuda)
    for k, v in late.items():
        mine[k].copy_(v)
    assert r.generate(PROMPTS, 8, **mine) == want
    torch.cuda.synchronize()


def test_runner_made_behind_a_busy_stream(cuda, model):
    def run():
        r = runner.Runner(model, 1)
        first = r.prefill(PROMPTS[0])
        return [first] + r.decode(7)[0].tolist()

    want = run()
    torch.cuda.synchronize()
    _busy(cuda)
    assert run() == want
    torch.cuda.synchronize()
