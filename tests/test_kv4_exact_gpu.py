"""4-bit KV cache: places where a kernel's own arithmetic, and not the inputs, could decide how near an answer comes."""
import math

import pytest
import torch

import kv4_oracle as oracle
from kv4_oracle import int32
from test_kv4_gpu import _check
from triton_distributed_gh_amd.ops import kv4

pytestmark = pytest.mark.gpu


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


# ---- the merge of many splits ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("gone", ["first", "last", "middle", "all but the end"])
@pytest.mark.parametrize("D,splits", [(64, 256), (128, 128), (256, 64), (256, -1)])
def test_whole_passes_of_splits_without_tokens(D, splits, gone):
    """The merge takes its splits in passes.  A pass whose pages are gone from the table says nothing about the others' scale, also
    where all scores are about -100 nats: 2^-144, below what fp32 holds next to 1."""
    gen = _gen(D + len(gone))
    H, Hq, group, page = 1, 2, 32, 64
    L = 16384 if splits < 0 else 128 * splits
    if splits < 0:
        assert kv4.auto_kv_splits(1, H, Hq // H, D, L) == 64
    table, pages = oracle.table_for(1, L, page, gen, device="cuda")
    cache = kv4.Int4KVCache.alloc(pages, page, H, D, group=group, device="cuda")
    k = (0.05 * torch.randn(1, L, H, D, generator=gen) - 100 / D).bfloat16().cuda()
    v = oracle.rows(gen, 1, L, H, D, device="cuda")
    kv4.kv4_append(k, v, cache, int32([0], "cuda"), table)
    there = torch.ones(L, dtype=torch.bool)
    there[{"first": slice(0, L // 2), "last": slice(L // 2, L), "middle": slice(L // 8, L - L // 8),
           "all but the end": slice(0, L - 100)}[gone]] = False
    table[0, (~there[::page]).cuda()] = -1
    there = there[::page].repeat_interleave(page)
    q = torch.ones(1, 1, Hq, D, dtype=torch.bfloat16, device="cuda")
    values = [oracle.held(v[0], group)]
    want, lse = oracle.attention(q, [oracle.held(k[0], group)], values, 1.0, there=[there])
    assert (lse < -80).all() and lse.isfinite().all()
    got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, scale=1.0, kv_split=splits, return_lse=True)
    torch.cuda.synchronize()
    _check(got[..., :D], want, got[..., D], lse, torch.float32, float(values[0].abs().max()), scores=D ** 0.5)


def test_splits_without_any_token_are_an_empty_row():
    gen = _gen(3)
    cache, table, _, _ = oracle.filled(gen, [128 * 70], 1, 128, 64, 64, device="cuda")
    table.fill_(-1)
    q = oracle.rows(gen, 1, 1, 4, 128, device="cuda")
    got = kv4.gqa_fwd_kv4(q, cache, int32([128 * 70], "cuda"), table, kv_split=70, return_lse=True)
    torch.cuda.synchronize()
    assert (got[..., :128] == 0).all() and (got[..., 128] == -math.inf).all()
