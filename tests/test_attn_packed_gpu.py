"""Packed-prompt attention: its plan on the host, its results against 64 bits on the GPU."""
import math

import pytest
import torch

from slang_b200 import _lib
from slang_b200 import kernels as kern

# The output's rounding to its type moves it by at most eps / 2 of its size, the probabilities'
# rounding by at most that share of sum p |v|; f32 scores of a few units add some 2^-20 of that sum.
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


def _reference(q, k, v, q_lens, kv_lens, scale, window):
    nh, hd = q.shape[1:]
    group = nh // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    q0 = k0 = 0
    for ql, kl in zip(q_lens, kv_lens):
        pos = torch.arange(kl - ql, kl, device=q.device)[:, None]
        at = torch.arange(kl, device=q.device)[None]
        seen = (at <= pos) & ((at > pos - window) if window else torch.ones_like(at, dtype=torch.bool))
        some = seen.any(1)
        for h in range(nh):
            kk, vv = k[k0:k0 + kl, h // group].double(), v[k0:k0 + kl, h // group].double()
            s = (scale * q[q0:q0 + ql, h].double() @ kk.T).masked_fill(~seen, -math.inf)[some]
            p = torch.softmax(s, -1) if kl else s
            rows = torch.arange(q0, q0 + ql, device=q.device)[some]
            out[rows, h], mass[rows, h] = p @ vv, p @ vv.abs()
        q0, k0 = q0 + ql, k0 + kl
    return out, mass


def _check(got, want, mass, dtype):
    tol = EPS[dtype] * (want.abs() + mass) + 2.0 ** -16 * mass + 1e-7
    off = (got.double() - want).abs()
    assert not torch.isnan(got).any()
    assert torch.all(off <= tol), f"off by {float((off - tol).max()):.3g} over the bound"


def _inputs(tq, tk, nh, nkv, hd, dtype, seed, dev):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(t, h, hd, generator=gen, device=dev).to(dtype) for t, h in ((tq, nh), (tk, nkv), (tk, nkv))]


def test_plan_covers_every_query_once():
    """Each query of each sequence lies in one tile, with its sequence's keys and its own position."""
    lens, kv = [1, 0, 300, 17, 64], [1, 5, 300, 400, 20]
    for nh, nkv, hd, per in ((8, 1, 256, 32), (6, 2, 128, 84), (5, 1, 64, 50), (12, 1, 256, 20), (128, 1, 64, 2)):
        plan = kern.PackedPlan(lens, nh, nkv, hd, kv_lens=kv, window=9, device="cpu")
        seen = {}
        for q0, n, k0, kl, pos0 in plan.tiles[:, :5].tolist():
            assert 1 <= n <= per
            for i in range(n):
                assert q0 + i not in seen
                seen[q0 + i] = (k0, kl, pos0 + i)
        want, q0, k0 = {}, 0, 0
        for a, b in zip(lens, kv):
            want.update({q0 + i: (k0, b, b - a + i) for i in range(a)})
            q0, k0 = q0 + a, k0 + b
        assert seen == want and plan.total_q == sum(lens) and plan.total_k == sum(kv)
    long = kern.PackedPlan([100, 2000, 50], 8, 1, 256, device="cpu").tiles
    ends = (long[:, 4] + long[:, 1]).tolist()
    assert ends == sorted(ends, reverse=True)  # those that see the most keys first


def test_plan_refusals():
    for bad in (lambda: kern.PackedPlan([1, -1], 8, 1, 128, device="cpu"), lambda: kern.PackedPlan([4], 7, 2, 128, device="cpu"),
                lambda: kern.PackedPlan([4], 8, 1, 96, device="cpu"), lambda: kern.PackedPlan([4], 8, 1, 512, device="cpu"),
                lambda: kern.PackedPlan([4], 129, 1, 64, device="cpu"), lambda: kern.PackedPlan([4], 8, 1, 64, window=-1, device="cpu")):
        with pytest.raises(_lib.SlangError):
            bad()
    with pytest.raises(ValueError):
        kern.PackedPlan([4, 5], 8, 1, 64, kv_lens=[4], device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd,dtype,window,q_lens,kv_lens", [
    (8, 1, 256, torch.float16, 0, [1], None),
    (8, 1, 256, torch.float16, 0, [300], None),
    (8, 1, 256, torch.bfloat16, 0, [15, 16, 17, 0, 127, 128, 129, 1], None),
    (8, 1, 256, torch.float16, 100, [700, 99, 101], None),
    (4, 4, 256, torch.bfloat16, 0, [513, 2], None),
    (12, 1, 256, torch.float16, 33, [77, 130], None),
    (32, 8, 128, torch.bfloat16, 0, [64, 1, 257, 640], None),
    (8, 8, 128, torch.float16, 0, [1000], None),
    (7, 1, 128, torch.float16, 50, [345, 12], None),
    (6, 2, 64, torch.float16, 0, [129, 600], None),
    (5, 1, 64, torch.bfloat16, 128, [513], None),
    (16, 1, 64, torch.float16, 1, [40, 200], None),
    (96, 1, 128, torch.float16, 0, [5, 31], None),
    (8, 2, 128, torch.bfloat16, 0, [10, 64, 1, 3], [500, 64, 129, 1000]),  # a cached prefix
    (8, 1, 256, torch.float16, 0, [64, 5], [20, 0]),  # more queries than keys: rows that see nothing
    (4, 2, 64, torch.float16, 60, [200, 3], [130, 700]),
])
def test_attn_prefill_packed(cuda, nh, nkv, hd, dtype, window, q_lens, kv_lens):
    kv = kv_lens or q_lens
    q, k, v = _inputs(sum(q_lens), sum(kv), nh, nkv, hd, dtype, nh + hd + sum(q_lens), cuda)
    scale = 3.0 / math.sqrt(hd)
    plan = kern.PackedPlan(q_lens, nh, nkv, hd, kv_lens=kv_lens, window=window, device=cuda)
    want, mass = _reference(q, k, v, q_lens, kv, scale, window)
    got = kern.attn_prefill_packed(q, k, v, plan, scale=scale)
    kern.device_status()
    _check(got, want, mass, dtype)
    assert torch.equal(got, kern.attn_prefill_packed(q, k, v, plan, scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 256), (8, 2, 128), (4, 1, 64)])
def test_attn_prefill_packed_long(cuda, nh, nkv, hd):
    q, k, v = _inputs(3001, 3001, nh, nkv, hd, torch.float16, 5, cuda)
    plan = kern.PackedPlan([2500, 501], nh, nkv, hd, device=cuda)
    want, mass = _reference(q, k, v, [2500, 501], [2500, 501], 0.2, 0)
    _check(kern.attn_prefill_packed(q, k, v, plan, scale=0.2), want, mass, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 256), (8, 2, 128), (4, 1, 64)])
def test_attn_prefill_packed_other_sequences_garbage(cuda, nh, nkv, hd):
    """NaN and infinities in the next sequence's keys and values reach nothing."""
    q, k, v = _inputs(430, 430, nh, nkv, hd, torch.float16, 7, cuda)
    lens = [100, 200, 130]
    want, mass = _reference(q, k, v, lens, lens, 0.2, 0)
    k[100:300], v[100:300], q[100:300] = math.nan, math.inf, math.nan
    plan = kern.PackedPlan(lens, nh, nkv, hd, device=cuda)
    got = kern.attn_prefill_packed(q, k, v, plan, scale=0.2)
    for lo, hi in ((0, 100), (300, 430)):
        _check(got[lo:hi], want[lo:hi], mass[lo:hi], torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_prefill_packed_rising_scores(cuda, hd):
    """Scores that climb along the keys by tens per block: the running maximum is raised block
    after block.  Whole-number q and k, so that the scores up to ~6000 are exact in f32."""
    gen = torch.Generator(device=cuda).manual_seed(8)
    q, k, v = _inputs(900, 900, 4, 1, hd, torch.float16, 8, cuda)
    q = torch.randint(0, 3, q.shape, generator=gen, device=cuda).half()
    k = torch.randint(0, 3, k.shape, generator=gen, device=cuda).half() + (torch.arange(900, device=cuda) // 100)[:, None, None]
    plan = kern.PackedPlan([900], 4, 1, hd, device=cuda)
    want, mass = _reference(q, k, v, [900], [900], 0.125, 0)
    _check(kern.attn_prefill_packed(q, k, v, plan, scale=0.125), want, mass, torch.float16)


@pytest.mark.gpu
def test_attn_prefill_packed_strides_and_stream(cuda):
    """q, k and v as views of one packed q|k|v tensor, out into a wider one, on another stream."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    qkv = torch.randn(333, 12, 128, generator=gen, device=cuda).bfloat16()
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    wide = torch.zeros(333, 9, 128, dtype=torch.bfloat16, device=cuda)
    plan = kern.PackedPlan([111, 222], 8, 2, 128, device=cuda)
    want, mass = _reference(q, k, v, [111, 222], [111, 222], 0.25, 0)
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kern.attn_prefill_packed(q, k, v, plan, scale=0.25, out=wide[:, :8])
    torch.cuda.current_stream().wait_stream(side)
    _check(wide[:, :8], want, mass, torch.bfloat16)
    assert torch.all(wide[:, 8] == 0)


@pytest.mark.gpu
def test_attn_prefill_packed_matches_the_unpacked_kernel(cuda):
    """The single-prompt kernel of the prefill computes the same attention."""
    q, k, v = _inputs(500, 500, 8, 1, 256, torch.float16, 3, cuda)
    q *= 0.2
    one = kern.attn_prefill(q, k[:, 0].contiguous(), v[:, 0].contiguous())
    got = kern.attn_prefill_packed(q, k, v, kern.PackedPlan([500], 8, 1, 256, device=cuda))
    # both round p and the output once each
    assert torch.all((got.float() - one.float()).abs() <= 4 * EPS[torch.float16] * v.abs().max().float())


@pytest.mark.gpu
def test_attn_prefill_packed_refusals(cuda):
    q, k, v = _inputs(20, 20, 4, 2, 64, torch.float16, 3, cuda)
    plan = kern.PackedPlan([20], 4, 2, 64, device=cuda)
    for bad in (lambda: kern.attn_prefill_packed(q.float(), k, v, plan), lambda: kern.attn_prefill_packed(q, k.bfloat16(), v, plan)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kern.attn_prefill_packed(q[:19], k, v, plan), lambda: kern.attn_prefill_packed(q, k[:, :1], v[:, :1], plan),
                lambda: kern.attn_prefill_packed(q, k, v.transpose(0, 1).contiguous().transpose(0, 1), plan),
                lambda: kern.attn_prefill_packed(q, k, v, plan, out=q.float()),
                lambda: kern.attn_prefill_packed(q.cpu(), k, v, plan),
                lambda: kern.attn_prefill_packed(q, k, v, kern.PackedPlan([20], 4, 2, 64, device="cpu"))):
        with pytest.raises(ValueError):
            bad()
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(_lib.SlangError):
            kern.attn_prefill_packed(q, k, v, plan, scale=scale)
    odd = torch.zeros(20, 4, 68, dtype=torch.float16, device=cuda)[..., :64]
    with pytest.raises(_lib.SlangError) as e:
        kern.attn_prefill_packed(odd, k, v, plan)
    assert e.value.code == _lib.SB_ERR_ALIGN
    none = kern.attn_prefill_packed(q[:0], k[:0], v[:0], kern.PackedPlan([0], 4, 2, 64, device=cuda))
    assert none.shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd,lens", [(8, 1, 256, [500]), (16, 4, 128, [500, 300]), (6, 2, 64, [600, 100])])
def test_attn_prefill_packed_repeats(cuda, nh, nkv, hd, lens):
    """200 launches back to back give the same bits, each right: the kernel's roles hand over in order."""
    q, k, v = _inputs(sum(lens), sum(lens), nh, nkv, hd, torch.float16, 12, cuda)
    plan = kern.PackedPlan(lens, nh, nkv, hd, device=cuda)
    want, mass = _reference(q, k, v, lens, lens, 0.2, 0)
    outs = [kern.attn_prefill_packed(q, k, v, plan, scale=0.2) for _ in range(200)]
    _check(outs[0], want, mass, torch.float16)
    assert all(torch.equal(o, outs[0]) for o in outs)
