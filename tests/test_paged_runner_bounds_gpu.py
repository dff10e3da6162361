"""GPU: what PagedRunner refuses once its sequences reach the end of their room."""
import pytest
import torch

from slang_b200 import paged, runner, synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda):
    return runner.DeviceModel(synth.random_model(synth.small_config(), seed=82), cuda, 32)


def _prompts(*lens):
    return [synth.prompt_tokens(n, 2048, seed=n) for n in lens]


def test_steps_past_the_reserved_pages(cuda, model):
    """decode_step ends where decode does: at the first token without a page, nothing changed."""
    r = paged.PagedRunner(model, 2, n_pages=8, page_size=4)
    first = r.prefill(_prompts(6, 3), steps=2)
    r.decode_step()
    r.decode_step()  # positions 6 and 7: the last of the pages
    torch.cuda.synchronize()
    pos = r.pos.tolist()
    for more in (r.decode_step, lambda: r.decode(1)):
        with pytest.raises(ValueError):
            more()
    torch.cuda.synchronize()
    assert r.pos.tolist() == pos
    # the steps taken one by one are those of a run
    whole = paged.PagedRunner(model, 2, n_pages=8, page_size=4)
    assert whole.prefill(_prompts(6, 3), steps=2) == first
    rest = whole.decode(2)
    history = r.history.cpu()
    assert [history[b, n + 1:n + 3].tolist() for b, n in enumerate((6, 3))] == rest


def test_steps_past_max_seq(cuda, model):
    r = paged.PagedRunner(model, 1, n_pages=8, page_size=8)
    r.prefill(_prompts(30), steps=2)
    r.decode_step()
    with pytest.raises(ValueError):
        r.decode_step()


def test_nothing_prefilled(cuda, model):
    r = paged.PagedRunner(model, 1, n_pages=8, page_size=4)
    for early in (r.decode_step, lambda: r.decode(1)):
        with pytest.raises(ValueError):
            early()


def test_bad_step_counts(cuda, model):
    r = paged.PagedRunner(model, 1, n_pages=8, page_size=4)
    with pytest.raises(ValueError):
        r.prefill(_prompts(9), steps=-8)  # fewer pages than the prompt itself takes
    with pytest.raises(ValueError):
        r.generate(_prompts(9), 0)
    with pytest.raises(ValueError):
        r.generate(_prompts(9), -1)
    r.prefill(_prompts(9), steps=2)
    with pytest.raises(ValueError):
        r.decode(-1)


def test_refused_settings_change_nothing(cuda, model):
    r = paged.PagedRunner(model, 2, n_pages=8, page_size=4)
    r.set_sampling(temperature=0.5, top_k=7)
    for bad in (dict(temperature=0.9, top_p=[0.1, 0.2, 0.3]), dict(temperature=0.9, seeds=[[1], [2]])):
        with pytest.raises(ValueError):
            r.set_sampling(**bad)
    torch.cuda.synchronize()
    assert r.temperature.tolist() == [0.5, 0.5] and r.top_k.tolist() == [7, 7]


def test_tokens_outside_the_vocabulary(cuda, model):
    """They would be read from past the embedding table: refused before anything is changed."""
    r = paged.PagedRunner(model, 2, n_pages=8, page_size=4)
    first = r.prefill(_prompts(6, 3), steps=4)
    for bad in (2048, -1, 2 ** 31, 2 ** 40, -2 ** 31):
        with pytest.raises(ValueError):
            r.prefill([[1, 2, bad], [3]], steps=4)
    again = paged.PagedRunner(model, 2, n_pages=8, page_size=4)
    assert again.prefill(_prompts(6, 3), steps=4) == first and again.decode(3) == r.decode(3)
