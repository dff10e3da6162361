"""GPU: sampling against a plain 64-bit implementation with a Philox of its own."""
import math

import numpy as np
import pytest
import torch

from slang_b200 import _lib
from slang_b200 import kernels as kern


def philox(seed: int, pos: int, n: int) -> np.ndarray:
    """Words [n] of Philox4x32-10 under key ``seed`` at counters (i / 4, pos, 0, 0)."""
    m = np.uint64(0xFFFFFFFF)
    key = [np.uint64(seed & 0xFFFFFFFF), np.uint64((seed >> 32) & 0xFFFFFFFF)]
    q = -(-n // 4)
    ctr = [np.arange(q, dtype=np.uint64), np.full(q, pos & 0xFFFFFFFF, np.uint64), np.zeros(q, np.uint64),
           np.zeros(q, np.uint64)]
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ key[0], b & m, (a >> np.uint64(32)) ^ ctr[3] ^ key[1], a & m]
        key = [(key[0] + np.uint64(0x9E3779B9)) & m, (key[1] + np.uint64(0xBB67AE85)) & m]
    return np.stack(ctr, 1).reshape(-1)[:n]


def reference(x, seed, pos, temp=1.0, k=0, p=1.0, floor=0.0):
    """(token, gap): the drawn token, and by what factor the runner-up or the nearest of the
    rules' edges missed it (a draw closer than f32 arithmetic resolves is no test)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(x.size), -x))
    if x[order[0]] == -np.inf:
        return -1, math.inf
    if temp <= 0 or p <= 0:
        return int(order[0]), math.inf
    if 0 < k < x.size:
        order = order[:k]
    with np.errstate(invalid="ignore"):
        d = np.where(x[order] == x[order[0]], 0.0, x[order] - x[order[0]])
    w = np.exp(d / temp)
    before = np.cumsum(w) - w
    keep = (w >= floor) & (w > 0) & ((before < p * w.sum()) if p < 1 else True)
    keep[0] = True
    u = np.minimum((philox(seed, pos, x.size)[order] + 0.5) * 2.0 ** -32, 1 - 2.0 ** -24)
    with np.errstate(divide="ignore"):
        time = np.where(keep, -np.log1p(-u) / w, np.inf)
        all_time = np.where(w > 0, -np.log1p(-u) / w, np.inf)
    best = time.min()
    token = int(order[time == best].min())
    rivals = np.sort(time)
    gap = rivals[1] / best - 1 if rivals.size > 1 else math.inf
    # tokens at an edge of the nucleus or of min-p that would win were they let in, or out
    edge = np.ones(w.size)
    if p < 1:
        edge = np.minimum(edge, np.abs(before / w.sum() - p))
    if floor > 0:
        edge = np.minimum(edge, np.abs(w / floor - 1))
    gap = min(gap, edge[all_time <= best].min())
    return token, gap


# f32 logits differ by steps of 2^-20 at sizes up to 16; the distance to the maximum over the
# temperature carries at most 2^-19, an exponential and a sum a few 2^-22 more
RESOLVED = 2.0 ** -16


def _check(logits, seeds, pos, tokens, temp=None, k=None, p=None, floor=None):
    x = logits.float().cpu().numpy()
    out, checked = tokens.tolist(), 0
    for r in range(x.shape[0]):
        at = lambda t, off: off if t is None else t[r].item()  # noqa: E731
        want, gap = reference(x[r], int(seeds[r]), int(pos[r]), at(temp, 1.0), at(k, 0), at(p, 1.0), at(floor, 0.0))
        if gap > RESOLVED:
            checked += 1
            assert out[r] == want, f"row {r}: drew {out[r]}, expected {want} (gap {gap:.3g})"
    assert checked >= 0.9 * x.shape[0]


def test_reference_philox_known_answer():
    """The published test vectors of Philox4x32-10 (key and counter zero)."""
    assert [hex(int(w)) for w in philox(0, 0, 4)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def _inputs(rows, vocab, dtype, seed, dev, spread=2.5):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=gen, device=dev)
    hot = torch.randint(0, vocab, (rows, 6), generator=gen, device=dev)
    x.scatter_add_(1, hot, 8 * torch.rand(rows, 6, generator=gen, device=dev))
    seeds = torch.randint(-2 ** 62, 2 ** 62, (rows,), generator=gen, device=dev)
    pos = torch.randint(0, 100000, (rows,), generator=gen, device=dev).to(torch.int32)
    return x.to(dtype), seeds, pos, torch.rand(4, rows, generator=gen, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 5, 1000, 1024, 1025, 4099, 32003, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sample_all_rules(cuda, vocab, dtype):
    rows = 48 if vocab < 100000 else 24
    x, seeds, pos, u = _inputs(rows, vocab, dtype, vocab, cuda)
    kind = torch.arange(rows, device=cuda) % 6
    temp = torch.where(kind == 0, 0.0, 0.5 + u[0])
    k = torch.where((kind == 2) | (kind == 4), 1 + (u[1] ** 3 * min(vocab, 400)).int(), 0).to(torch.int32)
    p = torch.where((kind == 1) | (kind == 4), 0.3 + 0.7 * u[2], 1.0)
    floor = torch.where((kind == 3) | (kind == 4), 0.2 * u[3] ** 2, 0.0)
    got = kern.sample(x, seeds, pos, temperature=temp, top_k=k, top_p=p, min_p=floor)
    _check(x, seeds, pos, got, temp, k, p, floor)
    assert torch.equal(got, kern.sample(x, seeds, pos, temperature=temp, top_k=k, top_p=p, min_p=floor))
    _check(x, seeds, pos, kern.sample(x, seeds, pos))  # every rule off
    # a row's draw does not depend on the batch it is in
    alone = torch.cat([kern.sample(x[r:r + 1], seeds[r:r + 1], pos[r:r + 1], temp[r:r + 1], k[r:r + 1], p[r:r + 1],
                                   floor[r:r + 1]) for r in range(0, rows, 5)])
    assert torch.equal(alone, got[::5])


@pytest.mark.gpu
def test_sample_ties_and_large_k(cuda):
    """Equal logits rank by index: the k-th place falls among thousands of equal values."""
    rows, vocab = 32, 50000
    gen = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randint(0, 3, (rows, vocab), generator=gen, device=cuda).float()
    x[1] = 0.25  # one value throughout
    seeds = torch.arange(rows, device=cuda) * 7919
    pos = torch.arange(rows, dtype=torch.int32, device=cuda)
    k = torch.tensor([1, 2, 17, 1000, 16000, 20000, 49999, 50000], dtype=torch.int32, device=cuda).repeat(rows // 8)
    got = kern.sample(x, seeds, pos, top_k=k)
    _check(x, seeds, pos, got, k=k)
    p = torch.linspace(0.01, 0.99, rows, device=cuda)
    _check(x, seeds, pos, kern.sample(x, seeds, pos, top_p=p), p=p)
    _check(x, seeds, pos, kern.sample(x, seeds, pos, top_k=k, top_p=p), k=k, p=p)


@pytest.mark.gpu
def test_sample_masked_rows(cuda):
    """-inf, the type's lowest value, NaN, +inf and rows without any token."""
    inf, low = math.inf, torch.finfo(torch.float32).min
    rows = [[-inf] * 9, [math.nan] * 9, [-inf] * 4 + [3.0] + [-inf] * 4, [low] * 9, [low] * 8 + [0.0],
            [math.nan] * 3 + [1.0] + [-inf] * 5, [inf, 1.0, inf, -inf, 0.0, 1.0, 2.0, inf, 3.0], [0.0, -0.0] * 4 + [-1.0],
            [-1000.0] * 9]
    x = torch.tensor(rows, device=cuda)
    n = x.shape[0]
    pos = torch.zeros(n, dtype=torch.int32, device=cuda)
    full = torch.ones(n, device=cuda)
    for seed in range(40):
        seeds = torch.full((n,), seed * 1000003, device=cuda)
        for kw in ({}, {"top_p": 0.5 * full}, {"min_p": 0.1 * full}, {"temperature": 0.3 * full},
                   {"top_k": torch.full((n,), 3, dtype=torch.int32, device=cuda)}, {"temperature": 0 * full}):
            got = kern.sample(x, seeds, pos, **kw)
            names = {"top_p": "p", "min_p": "floor", "temperature": "temp", "top_k": "k"}
            want = [reference(x[r].cpu().numpy(), seed * 1000003, 0, **{names[a]: b[r].item() for a, b in kw.items()})[0]
                    for r in range(n)]
            assert got.tolist() == want, kw
            assert got[0] == -1 and got[1] == -1 and got[2] == 4 and got[5] == 3


@pytest.mark.gpu
def test_sample_distribution(cuda):
    """20000 draws of one row follow its probabilities: every token's count is within six
    standard deviations of a binomial's."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5, 3.0, -2.0]], device=cuda)
    n = 20000
    seeds = torch.arange(n, device=cuda) * 2654435761 + 12345
    pos = torch.zeros(n, dtype=torch.int32, device=cuda)
    got = kern.sample(x.expand(n, 7).contiguous(), seeds, pos, temperature=torch.full((n,), 1.5, device=cuda))
    prob = torch.softmax(x[0].double() / 1.5, 0)
    count = torch.bincount(got.long(), minlength=7).double()
    assert torch.all((count - n * prob).abs() <= 6 * torch.sqrt(n * prob * (1 - prob)))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(700, 1500), (150, 70001)])
def test_sample_many_rows_of_all_kinds(cuda, rows, vocab):
    """More rows than run at once, which are served in another order: each draws what it draws alone."""
    g = torch.Generator(device="cuda").manual_seed(11)
    logits = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
    kind = torch.arange(rows, device="cuda") % 7
    one = torch.ones(rows, device="cuda")
    args = dict(temperature=torch.where(kind == 0, 0 * one, 0.7 * one), top_p=torch.where(kind % 3 == 1, 0.8 * one, one),
                min_p=torch.where(kind == 3, 0.05 * one, 0 * one), top_k=torch.where(kind >= 5, 20 * kind, 0 * kind).int())
    seeds = torch.arange(rows, device="cuda") * 977 + 5
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    got = kern.sample(logits, seeds, pos, **args)
    for r in range(rows):
        alone = kern.sample(logits[r:r + 1], seeds[r:r + 1], pos[r:r + 1], **{k: v[r:r + 1] for k, v in args.items()})
        assert int(alone) == int(got[r]), r


@pytest.mark.gpu
def test_sample_strides(cuda):
    """Rows that start off a vector boundary, on another stream."""
    x, seeds, pos, u = _inputs(6, 5001, torch.float16, 1, cuda)
    wide = torch.zeros(6, 5007, dtype=torch.float16, device=cuda)
    wide[:, 3:5004] = x
    p = 0.5 + 0.4 * u[0]
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kern.sample(wide[:, 3:5004], seeds, pos, top_p=p)
    torch.cuda.current_stream().wait_stream(side)
    _check(x, seeds, pos, got, p=p)
    assert kern.sample(x[:0], seeds[:0], pos[:0]).shape == (0,)


@pytest.mark.gpu
def test_sample_refusals(cuda):
    x, seeds, pos, u = _inputs(3, 100, torch.float32, 1, cuda)
    for bad in (lambda: kern.sample(x.double(), seeds, pos), lambda: kern.sample(x, seeds, pos.long()),
                lambda: kern.sample(x, seeds, pos, top_k=u[0, :3].contiguous()),
                lambda: kern.sample(x, seeds, pos, top_p=u[0, :3].half())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kern.sample(x[0], seeds, pos), lambda: kern.sample(x.t().contiguous().t(), seeds, pos),
                lambda: kern.sample(x, seeds[:2], pos), lambda: kern.sample(x, seeds, pos[:2]),
                lambda: kern.sample(x, seeds, pos, min_p=u[0, :2].contiguous()),
                lambda: kern.sample(x.cpu(), seeds, pos),
                lambda: kern.sample(x, seeds, pos, tokens=pos[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.SlangError):
        kern.sample(torch.zeros(1, 900000, device=cuda), seeds[:1], pos[:1])
