"""GPU: one decode workspace through calls of changing batch, head counts and head_dim; the largest page tables."""
import math

import pytest
import torch

from slang_b200 import _lib
from slang_b200 import kernels as kern

pytestmark = pytest.mark.gpu


def _state(cuda, nh, nkv, hd, dtype, batch, ctx, page=16, seed=0):
    """A cache whose sequences hold about ctx keys each (split over several CTAs), and its operands."""
    gen = torch.Generator(device=cuda).manual_seed(seed + nh + hd + batch)
    lens = [max(1, ctx + 37 * b % 101 - 50) for b in range(batch)]
    need = [-(-n // page) for n in lens]
    k, v = (torch.randn(sum(need), nkv, page, hd, generator=gen, device=cuda).to(dtype) for _ in range(2))
    table = torch.full((batch, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    q = torch.randn(batch, nh, hd, generator=gen, device=cuda).to(dtype)
    return kern.PagedKV(k, v), q, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda) - 1


def _attend(state, workspace):
    cache, q, table, pos = state
    out = torch.full_like(q, math.nan)  # rows that nobody joins show
    return kern.attn_decode_paged(q, cache, table, pos, scale=2.0 / math.sqrt(q.shape[2]), out=out, workspace=workspace)


@pytest.mark.parametrize("nh,nkv,hd,dtype,batches,ctx", [
    (8, 1, 256, torch.float16, (5, 1, 5, 40, 1, 256, 1, 40, 256), 300),
    (32, 8, 128, torch.bfloat16, (5, 1, 5, 64, 1, 64), 700),
    (8, 1, 256, torch.float16, (3, 1, 3, 200, 1, 200), 5000),
])
def test_batch_shrinks_and_grows(cuda, nh, nkv, hd, dtype, batches, ctx):
    """Calls of fewer sequences leave the workspace ready for calls of more, up to the batch it was
    made for: the same bits as on a fresh one."""
    states = {b: _state(cuda, nh, nkv, hd, dtype, b, ctx) for b in set(batches)}
    fresh = {b: _attend(s, None) for b, s in states.items()}
    ws = kern.attn_decode_paged_workspace(states[max(batches)][0], nh, max(batches))
    for b in batches:
        got = _attend(states[b], ws)
        assert torch.equal(got, fresh[b]), f"batch {b}"


def test_layers_of_other_shapes_share_a_workspace(cuda):
    """The workspace of the largest shape serves layers of other head_dims, head counts and batches in turn."""
    shapes = [(8, 1, 512, torch.float16, 3, 2000), (4, 4, 64, torch.bfloat16, 90, 1500), (32, 1, 128, torch.float16, 7, 900),
              (8, 1, 512, torch.float16, 1, 9000), (12, 2, 64, torch.float16, 200, 400), (8, 8, 128, torch.bfloat16, 33, 700)]
    states = [_state(cuda, *s) for s in shapes]
    fresh = [_attend(s, None) for s in states]
    ws = max((kern.attn_decode_paged_workspace(s[0], s[1].shape[1], s[1].shape[0]) for s in states), key=torch.numel)
    for _ in range(3):
        for s, want in zip(states, fresh):
            assert torch.equal(_attend(s, ws), want)


def test_page_tables_past_32_bits(cuda):
    """Tables whose rows could hold more blocks of keys than 32 bits count are refused; one short of that
    is served, whatever little of it is used."""
    page = 1 << 20
    none = torch.zeros(0, 1, page, 64, dtype=torch.float16, device=cuda)
    cache = kern.PagedKV(none, none)

    def attend(b, pages):
        q = torch.ones(b, 8, 64, dtype=torch.float16, device=cuda)
        table = torch.full((b, pages), -1, dtype=torch.int32, device=cuda)
        return kern.attn_decode_paged(q, cache, table, torch.arange(b, dtype=torch.int32, device=cuda))

    for b, pages in ((2, 2047), (32, 2047)):  # 32 * 2047 * 2^20 is 2^36 less 2^25
        assert torch.all(attend(b, pages) == 0)
    for b, pages in ((33, 2047), (65536, 1), (1, 2048)):
        with pytest.raises(_lib.SlangError) as e:
            attend(b, pages)
        assert e.value.code == _lib.SB_ERR_ARG
