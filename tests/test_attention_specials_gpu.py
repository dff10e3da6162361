"""GPU: scores that are not finite, in the packed-prompt and the paged decode attention."""
import math

import pytest
import torch

from slang_b200 import kernels as kern

pytestmark = pytest.mark.gpu
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


def _reference(q, k, v, scale):
    """Causal attention of one sequence and head in 64 bits, and sum p |v|; rows whose scores are all -inf give 0."""
    s = scale * q.double() @ k.double().T
    s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
    p = torch.softmax(s, -1)
    p[torch.all(s == -math.inf, -1)] = 0
    return p @ v.double(), p @ v.double().abs()


def _check(got, want, mass, dtype):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    tol = EPS[dtype] * (want.abs() + mass) + 2.0 ** -16 * mass + 1e-7
    bad = ~torch.isnan(want) & ~((got.double() - want).abs() <= tol)
    assert not bad.any()


def _prompt(cuda, hd, dtype, n, seed):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    q, k, v = (torch.randn(n, 2, hd, generator=gen, device=cuda).to(dtype) for _ in range(3))
    return q, k[:, :1].contiguous(), v[:, :1].contiguous()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_key_that_is_not_a_number(cuda, hd, dtype):
    """A NaN key reaches every query that sees it, wherever it lies in its block, and no other."""
    n, first = 400, 100  # queries from 200 on see whole blocks around it
    q, k, v = _prompt(cuda, hd, dtype, n, 1)
    plan = kern.PackedPlan([n], 2, 1, hd, device=cuda)
    clean = kern.attn_prefill_packed(q, k, v, plan, scale=0.2)
    for at in range(first, first + 64):
        bad = k.clone()
        bad[at, 0, at % hd] = math.nan
        got = kern.attn_prefill_packed(q, bad, v, plan, scale=0.2)
        assert torch.equal(got[:at], clean[:at])
        assert torch.isnan(got[at:]).all(), f"key {at}"


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinite_scores(cuda, hd, dtype):
    """A score of -inf has no weight, one of +inf leaves no number, as the formula has it."""
    n = 400
    q, k, v = _prompt(cuda, hd, dtype, n, 2)
    plan = kern.PackedPlan([n], 2, 1, hd, device=cuda)
    q[:, :, 0] = torch.where(torch.arange(n, device=cuda) % 3 == 0, 1.0, -1.0)[:, None].to(dtype)
    for at in (0, 5, 64, 67, 101, 127, 130, 250):
        bad = k.clone()
        bad[at, 0, 0] = math.inf  # its score: -inf for two queries of three, +inf for the third
        got = kern.attn_prefill_packed(q, bad, v, plan, scale=0.2)
        for h in range(2):
            want, mass = _reference(q[:, h], bad[:, 0], v[:, 0], 0.2)
            _check(got[:, h], want, mass, dtype)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_score_minus_infinity(cuda, hd, dtype):
    n = 300
    q, k, v = _prompt(cuda, hd, dtype, n, 3)
    q[:, :, 0], k[:, :, 0] = 1.0, -math.inf
    got = kern.attn_prefill_packed(q, k, v, kern.PackedPlan([n], 2, 1, hd, device=cuda), scale=0.2)
    assert torch.all(got == 0)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_decode_scores_that_are_not_finite(cuda, hd):
    """The paged decode: the last query of the same cases."""
    n, page = 400, 16
    q, k, v = _prompt(cuda, hd, torch.float16, n, 4)
    q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
    table = torch.arange(n // page, dtype=torch.int32, device=cuda)[None]
    pos = torch.tensor([n - 1], dtype=torch.int32, device=cuda)
    pages = lambda t: t.view(n // page, 1, page, hd)  # noqa: E731
    for at in (0, 15, 16, 77, 200, 399):
        for value in (math.nan, math.inf, -math.inf):
            bad = k.clone()
            bad[at, 0, 0] = value
            got = kern.attn_decode_paged(q[-1:], kern.PagedKV(pages(bad), pages(v)), table, pos, scale=0.2)
            for h in range(2):
                want, mass = _reference(q[:, h], bad[:, 0], v[:, 0], 0.2)
                _check(got[0, h], want[-1], mass[-1], torch.float16)
