"""GPU: several sequences served over paged caches, against the reference's and the oracle's runs."""
import os

import numpy as np
import pytest

from oracle import decoder as odec
from slang_b200 import manifest, paged, runner, synth
from tests._util import first_divergence

pytestmark = pytest.mark.gpu
TOL = 5e-2  # softcapped logits where the GEMMs carry f16 activations and the caches f16 (the reference: f32)


def _oracle(model, prompt, steps, max_seq):
    """Greedy tokens and top-2 margins of the softcapped logits."""
    dec = odec.OracleDecoder(model, max_seq)
    for p, t in enumerate(prompt):
        logits = dec.forward(int(t), p)
    toks, margins, pos = [], [], len(prompt)
    for _ in range(steps):
        top = np.sort(logits)[-2:]
        toks.append(int(np.argmax(logits)))
        margins.append(float(top[1] - top[0]))
        logits = dec.forward(toks[-1], pos)
        pos += 1
    return toks, margins


def test_matches_the_reference_in_a_batch(cuda, golden):
    """The reference's own prompt and tokens, served next to two other prompts."""
    model = synth.random_model(synth.small_config(), seed=77)
    prompt = [int(t) for t in golden["dec_small_prompt"]]
    others = [synth.prompt_tokens(n, 2048, seed=n) for n in (1, 37)]
    r = paged.PagedRunner(runner.DeviceModel(model, cuda, 96), 3, n_pages=24, page_size=8)
    got = r.generate([others[0], prompt, others[1]], 16)
    first_divergence(got[1], golden["dec_small_tokens"], golden["dec_small_margins"], TOL, "paged, the reference's prompt")
    for b, p in ((0, others[0]), (2, others[1])):
        ref, margins = _oracle(model, p, 16, 96)
        first_divergence(got[b], ref, margins, TOL, f"paged, sequence {b}")


@pytest.mark.parametrize("batch", [1, 11])
def test_batches_and_pages(cuda, batch):
    """The GEMV and the GEMM lm_head, pages of one token and of many, a second batch on the same pages."""
    model = synth.random_model(synth.small_config(), seed=78)
    dm = runner.DeviceModel(model, cuda, 64)
    for page in (1, 16):
        r = paged.PagedRunner(dm, batch, n_pages=64 * batch // page, page_size=page)
        for seed in (5, 6):
            prompts = [synth.prompt_tokens(3 + 2 * b, 2048, seed=seed * 100 + b) for b in range(batch)]
            got = r.generate(prompts, 6)
            for b in range(0, batch, 5):
                ref, margins = _oracle(model, prompts[b], 6, 64)
                first_divergence(got[b], ref, margins, TOL, f"batch {batch}, page {page}, sequence {b}")


def test_windows_and_shared_kv(cuda):
    """A sliding window on two layers, one of which reads another layer's keys and values."""
    model = synth.random_model(synth.small_config(), seed=80)
    cfg = dict(model["config"], sliding_window=6)
    specs = [dict(sp, sliding=i in (1, 3), kv_source=1 if i == 3 else i) for i, sp in enumerate(runner.layer_specs(cfg))]
    cfg["layer_specs"] = specs
    model = dict(model, config=cfg)
    dm = runner.DeviceModel(model, cuda, 64)
    prompts = [synth.prompt_tokens(n, 2048, seed=n) for n in (29, 7)]
    got = paged.PagedRunner(dm, 2, n_pages=20, page_size=4).generate(prompts, 8)
    for b, p in enumerate(prompts):
        ref, margins = _oracle(model, p, 8, 64)
        first_divergence(got[b], ref, margins, TOL, f"windows, sequence {b}")


def test_sampled_runs_follow_their_seeds(cuda):
    """A sequence's sampled tokens depend on its own prompt, settings and seed, not on its place in
    the batch or on its neighbours; temperature 0 and top-k 1 are greedy."""
    model = synth.random_model(synth.small_config(), seed=79)
    dm = runner.DeviceModel(model, cuda, 64)
    prompts = [synth.prompt_tokens(n, 2048, seed=n) for n in (9, 4, 17)]
    kw = dict(temperature=[0.9, 1.3, 0.7], top_k=[0, 40, 0], top_p=[0.9, 1.0, 0.8], min_p=[0.0, 0.0, 0.02])
    r = paged.PagedRunner(dm, 3, n_pages=24, page_size=8)
    one = r.generate(prompts, 10, seeds=[11, 22, 33], **kw)
    assert one == r.generate(prompts, 10, seeds=[11, 22, 33], **kw)
    turned = r.generate(prompts[::-1], 10, seeds=[33, 22, 11], **{k: v[::-1] for k, v in kw.items()})
    assert turned[::-1] == one
    assert r.generate(prompts, 10, seeds=[12, 23, 34], **kw) != one
    greedy = r.generate(prompts, 10)
    assert r.generate(prompts, 10, temperature=1.0, top_k=1, seeds=5) == greedy
    assert all(0 <= t < 2048 for row in one + greedy for t in row)


def test_refusals(cuda):
    model = synth.random_model(synth.small_config(), seed=79)
    dm = runner.DeviceModel(model, cuda, 32)
    r = paged.PagedRunner(dm, 2, n_pages=4, page_size=8)
    with pytest.raises(ValueError):  # one prompt for two sequences
        r.generate([[1, 2]], 4)
    with pytest.raises(ValueError):  # an empty prompt
        r.generate([[1, 2], []], 4)
    with pytest.raises(ValueError):  # past max_seq
        r.generate([[1] * 30, [2]], 8)
    with pytest.raises(ValueError):  # more pages than there are
        r.generate([[1] * 20, [2] * 20], 4)
    with pytest.raises(ValueError):  # past the reserved pages
        r.prefill([[1] * 8, [2] * 5], steps=2)
        r.decode(20)
    with pytest.raises(ValueError):
        r.set_sampling(temperature=[1.0, 1.0, 1.0])
    with pytest.raises(ValueError):
        paged.PagedRunner(dm, 0, n_pages=4)
    export = manifest.read(os.path.join(os.path.dirname(__file__), "golden", "export_arch"))
    with pytest.raises(ValueError):  # per-layer embeddings
        paged.PagedRunner(runner.DeviceModel(export, cuda, 32), 1, n_pages=4)
    with pytest.raises(ValueError):  # head_dim 512
        paged.PagedRunner(runner.DeviceModel({k: v for k, v in export.items() if k != "ple"}, cuda, 32), 1, n_pages=4)
