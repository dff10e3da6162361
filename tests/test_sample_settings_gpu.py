"""GPU: sampling settings at and past the ends of their ranges, the softcap, nuclei of very small weights."""
import math

import numpy as np
import pytest
import torch

from slang_b200 import kernels as kern
from tests.test_sample_gpu import RESOLVED, reference

pytestmark = pytest.mark.gpu


def _rows(cuda, rows, vocab, seed):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x = 2.5 * torch.randn(rows, vocab, generator=gen, device=cuda)
    seeds = torch.randint(-2 ** 62, 2 ** 62, (rows,), generator=gen, device=cuda)
    return x, seeds, torch.arange(rows, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("vocab", [1, 700, 40000])
@pytest.mark.parametrize("floor", [1.5, 1.0078125, 1e30, math.inf, math.nan])
@pytest.mark.parametrize("rules", [{}, {"top_k": 5}, {"top_p": 0.7}, {"top_k": 2000, "top_p": 0.9}])
def test_min_p_above_one_keeps_the_largest(cuda, vocab, floor, rules):
    """No weight reaches a min_p above 1 (or one that is not a number): the largest logit, the first of
    equal ones, always stays."""
    x, seeds, pos = _rows(cuda, 24, vocab, 5)
    x[8:16, ::7] = x[8:16].amax(1, keepdim=True)  # many equal ones, index 0 among them
    x[16:, 0], x[16:, vocab // 2:] = -math.inf, x[16:].amax() + 1  # and an upper half of equal ones
    kw = {k: torch.full((24,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=cuda)
          for k, v in rules.items()}
    got = kern.sample(x, seeds, pos, min_p=torch.full((24,), floor, device=cuda), **kw)
    want = [int((row == row.max()).nonzero()[0]) for row in x]
    assert got.tolist() == want


@pytest.mark.parametrize("rules", [{}, {"top_k": 3}, {"top_p": 0.4}])
def test_min_p_of_one_keeps_equal_ones(cuda, rules):
    """min_p of 1 keeps what weighs as much as the largest: the draw is among equal logits."""
    n = 64
    x = torch.tensor([[2.0, 1.0, 2.0, -1.0, 2.0, 0.0]], device=cuda).repeat(n, 1)
    seeds, pos = torch.arange(n, device=cuda) * 7919 + 3, torch.zeros(n, dtype=torch.int32, device=cuda)
    kw = {k: torch.full((n,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=cuda)
          for k, v in rules.items()}
    got = kern.sample(x, seeds, pos, min_p=torch.ones(n, device=cuda), **kw).tolist()
    names = {"top_p": "p", "top_k": "k"}
    want = [reference(x[r].cpu().numpy(), int(seeds[r]), 0, floor=1.0, **{names[k]: v for k, v in rules.items()})[0]
            for r in range(n)]
    assert got == want and len(set(got)) > 1


@pytest.mark.parametrize("top_k", [0, 4, 3000])
def test_top_p_that_is_not_a_number_is_off(cuda, top_k):
    x, seeds, pos = _rows(cuda, 16, 9000, 6)
    k = torch.full((16,), top_k, dtype=torch.int32, device=cuda)
    got = kern.sample(x, seeds, pos, top_k=k, top_p=torch.full((16,), math.nan, device=cuda))
    assert torch.equal(got, kern.sample(x, seeds, pos, top_k=k))


def test_nucleus_of_very_small_weights(cuda):
    """One token weighs 1, 800000 others 2^-33 each, and top_p ends half way through those: what is
    drawn of them lies in the first half.  (Their masses are lost to sums in units of 2^-31.)"""
    vocab, rows, w = 800000, 100, 2.0 ** -33
    x = torch.full((1, vocab), math.log(w), device=cuda)
    x[0, 0] = 0.0
    x = x.repeat(rows, 1)
    w = math.exp(float(x[0, 1]))
    total = 1 + (vocab - 1) * w
    p = torch.full((rows,), (1 + 0.5 * vocab * w) / total, device=cuda)
    # tokens 1 .. last are in; the sums resolve 2^-23 of the total, 1024 such tokens, and p 2^-24
    last, slack = int((float(p[0]) * total - 1) / w) + 1, 2048
    pos = torch.zeros(rows, dtype=torch.int32, device=cuda)
    drawn = []
    for call in range(1500):
        seeds = torch.arange(rows, device=cuda) + call * rows
        got = kern.sample(x, seeds, pos, top_p=p)
        drawn.append(got[got != 0])
    drawn = torch.cat(drawn).tolist()
    # 150000 draws, each with a chance of 4.7e-5 of one of them: 7 expected, none with a chance of e^-7
    assert drawn and max(drawn) <= last + slack, (last, drawn)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1000, 50001])
@pytest.mark.parametrize("softcap", [5.0, 30.0])
def test_softcap(cuda, dtype, vocab, softcap):
    """The draw is that of softcap * tanh(x / softcap), in every rule."""
    rows = 48
    x, seeds, pos = _rows(cuda, rows, vocab, vocab)
    x = (0.24 * softcap * x).to(dtype)  # up to about 2.5 times the cap
    x[1, ::3] = -math.inf
    u = torch.rand(3, rows, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    kind = torch.arange(rows, device=cuda) % 6
    temp = torch.where(kind == 0, 0.0, 0.5 + u[0])
    k = torch.where((kind == 2) | (kind == 4), 1 + (300 * u[1]).int(), 0).to(torch.int32)
    p = torch.where((kind == 1) | (kind == 4), 0.3 + 0.6 * u[2], 1.0)
    floor = torch.where((kind == 3) | (kind == 4), 0.2 * u[0], 0.0)
    got = kern.sample(x, seeds, pos, temperature=temp, top_k=k, top_p=p, min_p=floor, softcap=softcap).tolist()
    plain = kern.sample(x, seeds, pos, temperature=temp, top_k=k, top_p=p, min_p=floor).tolist()
    checked = 0
    for r in range(rows):
        v = x[r].double().cpu().numpy()
        capped = np.where(np.isinf(v), v, softcap * np.tanh(v / softcap))
        args = [int(seeds[r]), int(pos[r]), float(temp[r]), int(k[r]), float(p[r]), float(floor[r])]
        want, gap = reference(capped, *args)
        # the cap is computed in f32, a few 2^-22 off: values closer than that may change places
        top = np.sort(capped)[::-1]
        edges = [0] if kind[r] == 0 else [int(k[r]) - 1] if k[r] > 0 else []
        for at in edges:
            gap = min(gap, math.inf if top[at] == top[at + 1] else top[at] - top[at + 1])
        if gap > 4 * RESOLVED:  # 2^-14: steps of 2^-18 at 30, twice, over temperatures from 0.5
            checked += 1
            assert got[r] == want, (r, args)
    assert checked >= 0.75 * rows and got != plain


@pytest.mark.parametrize("rules", [{"top_p": 0.3}, {"top_k": 100, "top_p": 0.5}, {"min_p": 0.5}, {}])
def test_infinite_temperature(cuda, rules):
    """Every finite logit weighs 1, however far apart they lie."""
    rows, vocab = 32, 700
    x, seeds, pos = _rows(cuda, rows, vocab, 8)
    x = x * 1e37
    x[:, ::5] = -math.inf
    kw = {k: torch.full((rows,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=cuda)
          for k, v in rules.items()}
    got = kern.sample(x, seeds, pos, temperature=torch.full((rows,), math.inf, device=cuda), **kw).tolist()
    names = {"top_p": "p", "top_k": "k", "min_p": "floor"}
    for r in range(rows):
        want, gap = reference(x[r].cpu().numpy(), int(seeds[r]), int(pos[r]), 1e300, **{names[k]: v for k, v in rules.items()})
        assert gap <= RESOLVED or got[r] == want, r
