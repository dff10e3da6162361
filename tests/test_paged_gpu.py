"""GPU: the paged-cache operators against plain 64-bit implementations of their formulas."""
import math

import pytest
import torch

from slang_b200 import _lib
from slang_b200 import kernels as kern

pytestmark = pytest.mark.gpu

# One rounding of the result to the cache's type is off by at most half the distance of
# neighbouring numbers: 2^-11 of its size in f16, 2^-8 in bf16.  An attention output also carries
# the rounding of the probabilities, which moves it by at most that share of sum p |v|; scores
# in f32 add a few 2^-22 of their size.  The bounds below are these sums with room for the f32 terms.
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


def _cache(n_pages, nkv, page, hd, dtype, layout, gen, dev):
    shape = (n_pages, nkv, page, hd) if layout == "head" else (n_pages, page, nkv, hd)
    k, v = (torch.randn(shape, generator=gen, device=dev).to(dtype) for _ in range(2))
    if layout == "token":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return kern.PagedKV(k, v)


def _table(lens, page, gen, dev, spare=3, extra=1):
    """Distinct shuffled pages for sequences of these lengths; unused entries hold -1."""
    need = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(need) + spare, generator=gen, device=dev).tolist()
    width = max(need + [0]) + extra
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=dev).view(len(lens), width), sum(need) + spare


# ------------------------------------------------------------------ append

def _append_ref(qkv, k, v, table, seq, pos, cos, sin, nh, q_norm, k_norm, v_norm, eps):
    nkv, page, hd = k.shape[1:]
    half, max_pos = cos.shape[1], cos.shape[0]
    x = qkv.double().view(qkv.shape[0], -1, hd)
    k, v = k.double().clone(), v.double().clone()
    q_out = torch.zeros(x.shape[0], nh, hd, dtype=torch.float64, device=x.device)
    for i, (s, p) in enumerate(zip(seq.tolist(), pos.tolist())):
        if p < 0 or p >= max_pos:
            continue
        y = x[i].clone()
        for h in range(y.shape[0]):
            w = q_norm if h < nh else k_norm if h < nh + nkv else None
            if w is not None or (h >= nh + nkv and v_norm):
                y[h] /= torch.sqrt((y[h] ** 2).mean() + eps)
                if w is not None:
                    y[h] *= w.double()
            if h < nh + nkv:
                a, b = y[h, :half].clone(), y[h, half:2 * half].clone()
                c, sn = cos[p].double(), sin[p].double()
                y[h, :half], y[h, half:2 * half] = a * c - b * sn, b * c + a * sn
        q_out[i] = y[:nh]
        pg = int(table[s, p // page]) if p // page < table.shape[1] else -1
        if 0 <= pg < k.shape[0]:
            k[pg, :, p % page], v[pg, :, p % page] = y[nh:nh + nkv], y[nh + nkv:]
    return q_out, k, v


@pytest.mark.parametrize("nh,nkv,hd,rot,norm,src,dtype,page,layout,lens,starts", [
    (8, 1, 256, 256, True, torch.float32, torch.float16, 16, "head", [1], [1090]),
    (8, 1, 256, 256, True, torch.float16, torch.float16, 16, "head", [1] * 9, [0, 1, 15, 16, 17, 31, 32, 100, 7]),
    (7, 1, 128, 64, True, torch.bfloat16, torch.bfloat16, 1, "token", [5, 1, 33], [0, 3, 9]),
    (6, 3, 64, 64, False, torch.float32, torch.bfloat16, 32, "token", [65, 2], [0, 31]),
    (2, 2, 512, 512, True, torch.float16, torch.bfloat16, 64, "head", [3, 70], [60, 0]),
    (5, 5, 512, 128, False, torch.bfloat16, torch.float16, 8, "token", [9], [2]),
    (3, 1, 64, 16, True, torch.float16, torch.float16, 2, "head", [1, 1, 4], [5, 0, 3]),
    (4, 2, 128, 0, False, torch.float16, torch.float16, 4, "head", [3, 3], [1, 6]),
])
def test_kv_append(cuda, nh, nkv, hd, rot, norm, src, dtype, page, layout, lens, starts):
    gen = torch.Generator(device=cuda).manual_seed(nh * 1000 + hd + page)
    ends = [a + n for a, n in zip(starts, lens)]
    table, n_pages = _table(ends, page, gen, cuda)
    cache = _cache(n_pages, nkv, page, hd, dtype, layout, gen, cuda)
    t, half = sum(lens), rot // 2
    wide = torch.randn(t, (nh + 2 * nkv) * hd + 16, generator=gen, device=cuda).to(src)
    qkv = wide[:, 8:8 + (nh + 2 * nkv) * hd]  # rows spaced wider than they are
    seq = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lens)]).to(cuda)
    pos = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(starts, lens)]).to(cuda)
    ang = torch.rand(max(ends), half, generator=gen, device=cuda) * 6.3
    cos, sin = torch.cos(ang), torch.sin(ang)
    qn, kn = (1 + 0.2 * torch.randn(2, hd, generator=gen, device=cuda)).unbind(0) if norm else (None, None)
    qn, kn = (None if w is None else w.contiguous() for w in (qn, kn))
    ref = _append_ref(qkv, cache.k, cache.v, table, seq, pos, cos, sin, nh, qn, kn, norm, 1e-6)
    q = kern.kv_append_paged(qkv, cache, table, pos, cos, sin, nh, seq=seq, q_norm=qn, k_norm=kn, v_norm=norm, eps=1e-6)
    for got, want, name in ((q, ref[0], "q"), (cache.k, ref[1], "k"), (cache.v, ref[2], "v")):
        # one rounding to the type, and f32 arithmetic on values of a few units
        assert torch.all((got.double() - want).abs() <= EPS[dtype] * want.abs() + 4e-6), name


def test_kv_append_padding_and_missing_pages(cuda):
    """Padding tokens give a zero q and write nothing; places without a page are not written."""
    gen = torch.Generator(device=cuda).manual_seed(5)
    cache = _cache(4, 2, 16, 64, torch.float16, "head", gen, cuda)
    table = torch.tensor([[2, -1], [99, 1]], dtype=torch.int32, device=cuda)
    qkv = torch.randn(7, 8 * 64, generator=gen, device=cuda)
    seq = torch.tensor([0, 0, 0, 1, 1, -1, 2], dtype=torch.int32, device=cuda)
    pos = torch.tensor([-1, 3, 17, 5, 20, 1, 1], dtype=torch.int32, device=cuda)
    cos = torch.zeros(40, 32, device=cuda)
    before_k, before_v = cache.k.clone(), cache.v.clone()
    q = kern.kv_append_paged(qkv, cache, table, pos, cos, cos + 1, 4, seq=seq)
    assert torch.all(q[0] == 0) and torch.all(q[1:].abs().amax((1, 2)) > 0)
    for now, was in ((cache.k, before_k), (cache.v, before_v)):
        changed = (now != was).any(-1).any(1).nonzero().tolist()
        assert changed == [[1, 4], [2, 3]]  # (page, row) of positions 20 of sequence 1 and 3 of sequence 0
    # positions past the tables are padding too
    q = kern.kv_append_paged(qkv[:1], cache, table, pos[2:3], cos[:17], cos[:17], 4, seq=seq[:1])
    assert torch.all(q == 0)


def test_kv_append_packed_outputs(cuda):
    """k_out and v_out hold what the pages hold, and zero rows for padding."""
    gen = torch.Generator(device=cuda).manual_seed(6)
    cache = _cache(6, 3, 8, 128, torch.bfloat16, "token", gen, cuda)
    table = torch.tensor([[4, 1], [0, 5]], dtype=torch.int32, device=cuda)
    qkv = torch.randn(5, 12 * 128, generator=gen, device=cuda).half()
    qkv[3] = math.nan
    seq = torch.tensor([0, 1, 1, 0, 0], dtype=torch.int32, device=cuda)
    pos = torch.tensor([9, 0, 15, -1, 2], dtype=torch.int32, device=cuda)
    cos = torch.rand(16, 64, generator=gen, device=cuda)
    k, v = (torch.full((5, 3, 128), 7.0, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    q = kern.kv_append_paged(qkv, cache, table, pos, cos, cos, 6, seq=seq, k_out=k, v_out=v)
    for i, (s, p) in enumerate(zip(seq.tolist(), pos.tolist())):
        if p < 0:
            assert torch.all(q[i] == 0) and torch.all(k[i] == 0) and torch.all(v[i] == 0)
            continue
        pg = int(table[s, p // 8])
        assert torch.equal(k[i], cache.k[pg, :, p % 8]) and torch.equal(v[i], cache.v[pg, :, p % 8])
    with pytest.raises(ValueError):
        kern.kv_append_paged(qkv, cache, table, pos, cos, cos, 6, seq=seq, k_out=k[:4])
    with pytest.raises(ValueError):
        kern.kv_append_paged(qkv, cache, table, pos, cos, cos, 6, seq=seq, v_out=v.half())


def test_kv_append_nothing(cuda):
    cache = kern.PagedKV.allocate(2, 16, 1, 64, device=cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    cos = torch.ones(4, 32, device=cuda)
    q = kern.kv_append_paged(torch.zeros(0, 3 * 64, device=cuda), cache, table, none, cos, cos, 1)
    assert q.shape == (0, 1, 64)


# ------------------------------------------------------------------ decode

def _decode_ref(q, k, v, table, pos, scale, window):
    """(output, sum of p |v|) in 64 bits; keys on missing pages take no part."""
    b, nh, hd = q.shape
    n_pages, nkv, page = k.shape[:3]
    out = torch.zeros(b, nh, hd, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    for i in range(b):
        last = int(pos[i])
        lo = max(0, last + 1 - window) if window else 0
        keys = [(int(table[i, t // page]), t % page) for t in range(lo, min(last + 1, table.shape[1] * page))]
        keys = [(p, o) for p, o in keys if 0 <= p < n_pages]
        if not keys:
            continue
        pg, off = (torch.tensor(x, device=q.device) for x in zip(*keys))
        for h in range(nh):
            g = h // (nh // nkv)
            p = torch.softmax(scale * (k[pg, g, off].double() @ q[i, h].double()), 0)
            out[i, h], mass[i, h] = p @ v[pg, g, off].double(), p @ v[pg, g, off].double().abs()
    return out, mass


def _check_attention(got, want, mass, dtype):
    tol = EPS[dtype] * (want.abs() + mass) + 2.0 ** -18 * mass + 1e-7
    assert torch.all((got.double() - want).abs() <= tol)


@pytest.mark.parametrize("nh,nkv,hd,dtype,page,layout,window,lens", [
    (8, 1, 256, torch.float16, 16, "head", 0, [1091]),
    (8, 1, 256, torch.float16, 16, "head", 0, [1, 2, 15, 16, 17, 63, 64, 65, 0, 300]),
    (8, 1, 256, torch.bfloat16, 64, "head", 100, [1, 99, 100, 101, 777]),
    (32, 8, 128, torch.bfloat16, 32, "token", 0, [513, 0, 64, 1]),
    (12, 4, 64, torch.float16, 1, "token", 0, [200, 129]),
    (7, 1, 64, torch.float16, 2, "head", 17, [5, 64, 400]),
    (16, 1, 256, torch.bfloat16, 16, "token", 0, [321, 40]),
    (48, 2, 128, torch.float16, 128, "head", 0, [140, 3]),
    (4, 2, 512, torch.float16, 16, "head", 0, [257, 31]),
    (16, 1, 512, torch.bfloat16, 32, "token", 50, [100, 333]),
    (17, 1, 512, torch.float16, 4, "token", 0, [77]),
    (20, 1, 256, torch.float16, 8, "head", 0, [90, 1]),
    (1, 1, 128, torch.float16, 16, "head", 0, [4000]),
])
def test_attn_decode_paged(cuda, nh, nkv, hd, dtype, page, layout, window, lens):
    gen = torch.Generator(device=cuda).manual_seed(nh + hd + page + len(lens))
    table, n_pages = _table(lens, page, gen, cuda)
    cache = _cache(n_pages, nkv, page, hd, dtype, layout, gen, cuda)
    q = torch.randn(len(lens), nh, hd, generator=gen, device=cuda).to(dtype)
    pos = torch.tensor(lens, dtype=torch.int32, device=cuda) - 1
    scale = 3.0 / math.sqrt(hd)
    want, mass = _decode_ref(q, cache.k, cache.v, table, pos, scale, window)
    ws = kern.attn_decode_paged_workspace(cache, nh, len(lens))
    first = kern.attn_decode_paged(q, cache, table, pos, scale=scale, window=window, workspace=ws)
    _check_attention(first, want, mass, dtype)
    # the workspace is left ready, the split does not depend on the order of arrival
    again = kern.attn_decode_paged(q, cache, table, pos, scale=scale, window=window, workspace=ws)
    assert torch.equal(first, again)
    assert torch.equal(first, kern.attn_decode_paged(q, cache, table, pos, scale=scale, window=window))


def test_attn_decode_paged_long_axis(cuda):
    """One sequence over more than 2^31 bytes of cache: every SM works on it, offsets pass 32 bits."""
    page, hd, n = 64, 512, 40000
    gen = torch.Generator(device=cuda).manual_seed(11)
    n_pages = 3000000000 // (page * hd * 2)  # the pages in use lie at both ends of 3 GB of K
    k = torch.empty(n_pages, 1, page, hd, dtype=torch.float16, device=cuda)
    v = torch.empty_like(k)
    need = -(-n // page)
    ids = torch.cat([torch.arange(need // 2), torch.arange(n_pages - (need - need // 2), n_pages)]).to(cuda)
    for t in (k, v):
        t[ids] = torch.randn(need, 1, page, hd, generator=gen, device=cuda).to(torch.float16)
    table = ids[torch.randperm(need, generator=gen, device=cuda)].to(torch.int32)[None]
    cache = kern.PagedKV(k, v)
    q = torch.randn(1, 4, hd, generator=gen, device=cuda).to(torch.float16)
    pos = torch.tensor([n - 1], dtype=torch.int32, device=cuda)
    scale = 3.0 / math.sqrt(hd)
    got = kern.attn_decode_paged(q, cache, table, pos, scale=scale)
    kk, vv = (t[table[0].long(), 0].reshape(-1, hd)[:n].double() for t in (k, v))
    p = torch.softmax(scale * q[0].double() @ kk.T, -1)
    _check_attention(got[0], p @ vv, p @ vv.abs(), torch.float16)


@pytest.mark.parametrize("hd,layout", [(64, "token"), (256, "head"), (512, "head")])
def test_attn_decode_paged_masked_garbage(cuda, hd, layout):
    """NaN and infinities past the sequence's end, before the window, on other pages and behind
    missing pages change nothing."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    page, lens, window = 16, [37, 90, 16], 40
    table, n_pages = _table(lens, page, gen, cuda)
    cache = _cache(n_pages, 2, page, hd, torch.float16, layout, gen, cuda)
    table[1, 3] = n_pages + 7  # a page the cache does not have
    q = torch.randn(3, 6, hd, generator=gen, device=cuda).half()
    pos = torch.tensor(lens, dtype=torch.int32, device=cuda) - 1
    want, mass = _decode_ref(q, cache.k, cache.v, table, pos, 0.2, window)
    seen = torch.zeros(n_pages, page, dtype=torch.bool, device=cuda)
    for i, n in enumerate(lens):
        for t in range(max(0, n - window), n):
            if 0 <= int(table[i, t // page]) < n_pages:
                seen[int(table[i, t // page]), t % page] = True
    for t, bad in ((cache.k, math.nan), (cache.v, math.inf)):
        t.masked_fill_(~seen[:, None, :, None], bad)
    got = kern.attn_decode_paged(q, cache, table, pos, scale=0.2, window=window)
    _check_attention(got, want, mass, torch.float16)


def test_attn_decode_paged_all_keys_missing(cuda):
    gen = torch.Generator(device=cuda).manual_seed(3)
    cache = _cache(4, 1, 16, 128, torch.bfloat16, "head", gen, cuda)
    table = torch.tensor([[-1, -1], [0, 1]], dtype=torch.int32, device=cuda)
    q = torch.randn(2, 3, 128, generator=gen, device=cuda).bfloat16()
    pos = torch.tensor([20, 100], dtype=torch.int32, device=cuda)  # 100: past what the pages hold
    got = kern.attn_decode_paged(q, cache, table, pos, scale=0.3)
    want, mass = _decode_ref(q, cache.k, cache.v, table, pos, 0.3, 0)
    assert torch.all(got[0] == 0)
    _check_attention(got, want, mass, torch.bfloat16)


def test_attn_decode_paged_large_scores(cuda):
    """Scores that climb by hundreds along the keys: the running maximum is raised many times."""
    gen = torch.Generator(device=cuda).manual_seed(9)
    n, hd = 900, 128
    table, n_pages = _table([n], 16, gen, cuda)
    cache = _cache(n_pages, 1, 16, hd, torch.float16, "head", gen, cuda)
    for t in range(n):
        cache.k[int(table[0, t // 16]), 0, t % 16] *= 0.02 * t
    q = torch.randn(1, 8, hd, generator=gen, device=cuda).half()
    pos = torch.tensor([n - 1], dtype=torch.int32, device=cuda)
    got = kern.attn_decode_paged(q, cache, table, pos, scale=2.0)
    want, mass = _decode_ref(q, cache.k, cache.v, table, pos, 2.0, 0)
    # scores of size up to ~2000 carry f32 rounding of 2^-22 of that each
    tol = EPS[torch.float16] * (want.abs() + mass) + 2.0 ** -10 * mass
    assert torch.all((got.double() - want).abs() <= tol)


def test_attn_decode_paged_other_stream_and_strides(cuda):
    gen = torch.Generator(device=cuda).manual_seed(4)
    table, n_pages = _table([70, 130], 32, gen, cuda)
    cache = _cache(n_pages, 2, 32, 64, torch.bfloat16, "token", gen, cuda)
    wide = torch.randn(2, 3, 8, 64, generator=gen, device=cuda).bfloat16()
    q = wide[:, 1]  # sequences spaced three rows apart
    pos = torch.tensor([69, 129], dtype=torch.int32, device=cuda)
    want, mass = _decode_ref(q, cache.k, cache.v, table, pos, 0.3, 0)
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kern.attn_decode_paged(q, cache, table, pos, scale=0.3)
    torch.cuda.current_stream().wait_stream(side)
    _check_attention(got, want, mass, torch.bfloat16)


# ------------------------------------------------------------------ refusals

def test_paged_refusals(cuda):
    dev = cuda
    cache = kern.PagedKV.allocate(4, 16, 2, 64, device=dev)
    table = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    pos = torch.zeros(2, dtype=torch.int32, device=dev)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=dev)
    cos = torch.ones(8, 32, device=dev)
    qkv = torch.zeros(2, 8 * 64, device=dev)
    half = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=dev)
    with pytest.raises(TypeError):
        kern.PagedKV(half.float(), half.float())
    with pytest.raises(ValueError):
        kern.PagedKV(half, half[:3])
    with pytest.raises(ValueError):
        kern.PagedKV(half, half.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(TypeError):
        kern.attn_decode_paged(q.float(), cache, table, pos)
    with pytest.raises(TypeError):
        kern.attn_decode_paged(q, cache, table.long(), pos)
    with pytest.raises(ValueError):
        kern.attn_decode_paged(q, cache, table[:1], pos)
    with pytest.raises(ValueError):
        kern.attn_decode_paged(q[..., :32], cache, table, pos)
    with pytest.raises(ValueError):
        kern.attn_decode_paged(q, cache, table, pos, out=torch.empty(2, 4, 64, device=dev))
    with pytest.raises(_lib.SlangError):  # 3 query heads over 2 kv heads
        kern.attn_decode_paged(q[:, :3], cache, table, pos)
    with pytest.raises(_lib.SlangError):
        kern.attn_decode_paged(q, cache, table, pos, window=-1)
    with pytest.raises(_lib.SlangError) as e:
        kern.attn_decode_paged(q, cache, table, pos, workspace=torch.zeros(16, dtype=torch.uint8, device=dev))
    assert e.value.code == _lib.SB_ERR_WORKSPACE
    with pytest.raises(_lib.SlangError):  # page_size 12 is not a power of two
        odd = torch.zeros(4, 2, 12, 64, dtype=torch.float16, device=dev)
        kern.attn_decode_paged(q, kern.PagedKV(odd, odd), table, pos)
    with pytest.raises(_lib.SlangError):
        odd = torch.zeros(4, 2, 16, 96, dtype=torch.float16, device=dev)
        kern.attn_decode_paged(q.new_zeros(2, 4, 96), kern.PagedKV(odd, odd), table, pos)
    with pytest.raises(_lib.SlangError) as e:  # rows off the 16-byte boundary
        odd = torch.zeros(4, 2, 16, 68, dtype=torch.float16, device=dev)[..., :64]
        kern.attn_decode_paged(q, kern.PagedKV(odd, odd), table, pos)
    assert e.value.code == _lib.SB_ERR_ALIGN
    with pytest.raises(ValueError):
        kern.kv_append_paged(qkv[:, :64], cache, table, pos, cos, cos, 4)
    with pytest.raises(ValueError):
        kern.kv_append_paged(qkv, cache, table, pos[:1], cos, cos, 4)
    with pytest.raises(TypeError):
        kern.kv_append_paged(qkv, cache, table, pos, cos.half(), cos.half(), 4)
    with pytest.raises(TypeError):
        kern.kv_append_paged(qkv.double(), cache, table, pos, cos, cos, 4)
    with pytest.raises(_lib.SlangError):  # rot 2 * 33 is not a multiple of 16
        kern.kv_append_paged(qkv, cache, table, pos, torch.ones(8, 33, device=dev), torch.ones(8, 33, device=dev), 4)
    with pytest.raises(_lib.SlangError):  # three tokens without `seq`, two sequences
        kern.kv_append_paged(torch.zeros(3, 8 * 64, device=dev), cache, table, pos.new_zeros(3), cos, cos, 4)
