"""GPU: many keys of very small weight beside one that dominates (an attention sink)."""
import math

import pytest
import torch

from slang_b200 import kernels as kern

pytestmark = pytest.mark.gpu
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


def _sink(cuda, n, hd, dtype, gap):
    """q . k is gap for key 0 and 0 for the others; v is 0 for key 0 and 1 for the others."""
    q = torch.zeros(n, 2, hd, dtype=dtype, device=cuda)
    k, v = (torch.zeros(n, 1, hd, dtype=dtype, device=cuda) for _ in range(2))
    q[..., 0], k[0, 0, 0], v[1:] = 1.0, gap, 1.0
    return q, k, v


def _tolerance(keys, want, dtype):
    """Rounding of the weights and of the output to the type, f32 terms and exponentials (2^-13), and f16's
    subnormals: weights below 2^-14 of what the type reaches (2^7 over the running maximum's weight) lie in
    steps of 2^-31 of that weight, an output below 2^-14 in steps of 2^-24; half a step each."""
    low, out = (2.0 ** -32, 2.0 ** -25) if dtype == torch.float16 else (0.0, 0.0)
    return (2 * EPS[dtype] + 2.0 ** -13) * want + keys * low + out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [9.0, 14.0, 17.6875, 19.0])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefill(cuda, hd, gap, dtype):
    n = 4500
    q, k, v = _sink(cuda, n, hd, dtype, gap)
    got = kern.attn_prefill_packed(q, k, v, kern.PackedPlan([n], 2, 1, hd, device=cuda)).double()
    others = torch.arange(n, device=cuda, dtype=torch.float64)  # keys besides 0 that a query sees
    mass = others * math.exp(-float(torch.tensor(gap).to(dtype)))
    want = (mass / (1 + mass))[:, None, None]
    assert torch.all((got - want).abs() <= _tolerance(others[:, None, None], want, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [9.0, 14.0, 17.6875, 19.0])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_decode(cuda, hd, gap, dtype):
    n, page = 24000, 64
    q, k, v = _sink(cuda, n, hd, dtype, gap)
    pages = lambda t: t.view(n // page, 1, page, hd)  # noqa: E731
    table = torch.arange(n // page, dtype=torch.int32, device=cuda)[None]
    pos = torch.tensor([n - 1], dtype=torch.int32, device=cuda)
    got = kern.attn_decode_paged(q[-1:].contiguous(), kern.PagedKV(pages(k), pages(v)), table, pos).double()
    mass = torch.tensor((n - 1) * math.exp(-float(torch.tensor(gap).to(dtype))), dtype=torch.float64, device=cuda)
    want = mass / (1 + mass)
    assert torch.all((got - want).abs() <= _tolerance(n - 1, want, dtype))
