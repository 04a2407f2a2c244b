"""4-bit KV cache: places where a kernel's own arithmetic, and not the inputs, could decide how near an answer comes."""
import math

import pytest
import torch

import kv4_oracle as oracle
from kv4_oracle import int32
from test_kv4_gpu import SHAPES, _check
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


# ---- soft caps ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale,soft_cap", [(0.1, 1e4), (-0.3, 1e7), (0.1, 1e30), (0.1, 3e38), (0.1, 1e60),
                                            (0.2, 2.0), (0.1, 1e-39), (0.1, 1e-60)])
@pytest.mark.parametrize("Hq,H,S,D,group", SHAPES)
def test_caps_of_any_size(Hq, H, S, D, group, scale, soft_cap):
    """A cap far above the scores changes nothing; one near them or below bends or flattens them."""
    gen = _gen(42)
    lens, page = [333, 40], 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda")
    q = oracle.rows(gen, 2, S, Hq, D, device="cuda")
    keys, values = [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs]
    want, lse = oracle.attention(q, keys, values, scale, soft_cap)
    for splits in (1, 2):
        got = kv4.gqa_fwd_kv4(q, cache, int32(lens, "cuda"), table, scale=scale, soft_cap=soft_cap, kv_split=splits, return_lse=True)
        torch.cuda.synchronize()
        _check(got[..., :D], want, got[..., D], lse, torch.float32, max(float(x.abs().max()) for x in values),
               scores=max(1.0, abs(scale) * D ** 0.5))


# ---- queries of any size, and scores up to where they are whole numbers ------------------------------------------------
@pytest.mark.parametrize("q_size,k_size", [(2.0 ** 120, 2.0 ** -120), (2.0 ** 102, 2.0 ** -102), (2.0 ** -110, 2.0 ** 110)])
@pytest.mark.parametrize("Hq,H,S,D,group", [*SHAPES, (40, 1, 2, 128, 64), (40, 1, 3, 256, 64)])
def test_large_queries_over_small_keys(Hq, H, S, D, group, q_size, k_size, monkeypatch):
    """The same scores, from far larger queries and far smaller keys or the other way round."""
    monkeypatch.setattr(kv4, "takes_chunks", lambda *a: a[2] > 64 and a[5] == 0)
    gen = _gen(47)
    L, page = 150, 16
    cache, table, ks, vs = oracle.filled(gen, [L], H, D, group, page, torch.bfloat16, "cuda")
    k = ks[0] * k_size
    kv4.kv4_append(k[None], vs[0][None], cache, int32([0], "cuda"), table)
    q = oracle.rows(gen, 1, S, Hq, D, device="cuda") * q_size
    values = [oracle.held(vs[0], group)]
    want, lse = oracle.attention(q, [oracle.held(k, group)], values, D ** -0.5)
    got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, return_lse=True)
    torch.cuda.synchronize()
    _check(got[..., :D], want, got[..., D], lse, torch.float32, float(values[0].abs().max()))


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("Hq,H,S,D,group", [*SHAPES, (40, 1, 2, 128, 64), (40, 1, 3, 256, 64)])
def test_scores_up_to_2_to_the_27(Hq, H, S, D, group, sign, monkeypatch):
    """All the weight is the best token's, and the LSE is its score."""
    monkeypatch.setattr(kv4, "takes_chunks", lambda *a: a[2] > 64 and a[5] == 0)
    gen = _gen(48)
    L, page = 150, 16
    cache, table, ks, vs = oracle.filled(gen, [L], H, D, group, page, torch.bfloat16, "cuda")
    k = sign * ks[0].abs()
    kv4.kv4_append(k[None], vs[0][None], cache, int32([0], "cuda"), table)
    q = (oracle.rows(gen, 1, S, Hq, D, device="cuda").abs() * 2.0 ** 22).to(torch.bfloat16)
    keys, values = oracle.held(k, group), oracle.held(vs[0], group)
    scores = (q[0].double().cpu().unsqueeze(1) * keys.repeat_interleave(Hq // H, 1)).sum(-1).transpose(1, 2) * D ** -0.5
    assert 2.0 ** 24 < scores.abs().max() < 2.0 ** 27
    scores.masked_fill_(torch.arange(L) > L - S + torch.arange(S)[:, None, None], -math.inf)
    top, at = scores.max(-1)
    second = scores.scatter(-1, at.unsqueeze(-1), -math.inf).max(-1).values
    # the larger of two scores is the larger in the kernel too where they differ by what keys rounded to 2^-11 leave
    clear = top - second > 2.0 ** -10 * top.abs()
    assert clear.any()
    got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, return_lse=True)[0].double().cpu()
    want = values.repeat_interleave(Hq // H, 1)[at, torch.arange(Hq)]
    assert ((got[..., :D] - want).abs() <= 2.0 ** -9 * values.abs().max())[clear].all()
    assert ((got[..., D] - top).abs() <= 2.0 ** -10 * top.abs()).all()


# ---- many columns ---------------------------------------------------------------------------------------------------
@pytest.fixture
def chunks(monkeypatch):
    monkeypatch.setattr(kv4, "takes_chunks", lambda *a: a[2] >= 32 and a[5] == 0)


def _first_rows(D, group, size, q_size, k_size, rows):
    """A prompt of 96 tokens, the first ``rows`` of them with V of ``size`` and K of ``k_size``; (out [96, Hq, D], lse) and what
    is exact."""
    gen = _gen(D + group)
    L, H, Hq, page = 96, 1, 2, 16
    table, pages = oracle.table_for(1, L, page, gen, device="cuda")
    cache = kv4.Int4KVCache.alloc(pages, page, H, D, group=group, device="cuda")
    k, v = oracle.rows(gen, L, H, D), oracle.rows(gen, L, H, D)
    k[:rows] *= k_size
    v[:rows] *= size
    kv4.kv4_append(k[None].cuda(), v[None].cuda(), cache, int32([0], "cuda"), table)
    q = oracle.rows(gen, 1, L, Hq, D, device="cuda") * q_size
    got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, return_lse=True)
    torch.cuda.synchronize()
    keys, values = oracle.held(k, group), oracle.held(v, group)
    want, lse = oracle.attention(q[:, :rows], [keys[:rows]], [values[:rows]], D ** -0.5)
    terms = float((keys[:rows, 0].abs() @ q[0, :rows].double().abs().cpu().transpose(1, 2)).max()) * D ** -0.5
    return got[0, :rows].double().cpu(), want[0], lse[0], values[:rows], terms


@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 0.0])
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (128, 128), (256, 64)])
def test_rows_that_see_small_values_alone(D, group, size, chunks):
    """The first rows of a prompt see tokens whose V is far smaller than that of the tokens beside them, which they do not see:
    what comes out is as near, measured by their own size, as for any other row.

    Row 0 sees one token, and no weight is rounded in its result: a value is an fp16 number at most 2^-11 of itself off or, at the
    smallest size that is taken so, 17 halves of fp16's last step (15 from the scale, one from low, one from the result) of a group
    no smaller than 2^-9: 17 * 2^-25 / 2^-9 < 2^-11.9 of the group's 15 scale + |low| <= 3 max |v|.  Where codes are multiplied instead, P
    times scale is an fp16 number: 2^-11 of 15 scale.  Together under 2^-11 |v| + 2^-11 * 3 max |v| <= 2^-9 max |v| of its group."""
    got, want, lse, values, _ = _first_rows(D, group, size, 1.0, 1.0, 3)
    top = values.abs().unflatten(-1, (-1, group)).amax(-1).repeat_interleave(group, -1)     # [rows, H, D]
    off = (got[0, :, :D] - want[0]).abs()
    assert (off <= 2.0 ** -9 * top[0]).all(), float((off / top[0].clamp(min=1e-30)).max())
    # rows 1 and 2: the weights' own errors too, on what their tokens hold (2^-11 of a weight, and 2^-11 for the scores)
    for r in (1, 2):
        off = (got[r, :, :D] - want[r]).abs()
        assert (off <= (2.0 ** -9 + 2.0 ** -10 + 2.0 ** -11) * top[:r + 1].amax(0)).all()


@pytest.mark.parametrize("k_size,q_size", [(2.0 ** -20, 2.0 ** 20), (2.0 ** -14, 2.0 ** 14), (2.0 ** -12, 2.0 ** 8), (2.0 ** -20, 1.0)])
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (128, 128), (256, 64)])
def test_rows_that_see_small_keys_alone(D, group, k_size, q_size, chunks):
    """The same for K, with queries that are large enough for scores of a few nats from such keys."""
    got, want, lse, values, terms = _first_rows(D, group, 1.0, q_size, k_size, 12)
    scores, v_max = max(1.0, k_size * q_size), float(values.abs().max())
    off = (got[..., :D] - want).abs()
    # K as fp16 numbers: a score is off by 2^-11 of its terms (|q| |k| summed) at most, and by 2^-12 where K is too small for that; an
    # output by twice the largest |v| times as much.  Then the bounds of the weights and the scores.
    rounded = 2.0 ** -11 * terms + 2.0 ** -12
    assert (off <= oracle.bounds(want, torch.float32, v_max, scores=scores) + 2 * rounded * v_max).all()
    assert ((got[..., D] - lse).abs() <= scores * 5e-4 + rounded).all()


def _flags(q, cache, lens, table, splits, scale):
    """What csrc/ops/kv4_chunk.hip leaves to the other kernel: [column blocks, batch, splits, KV heads]."""
    batch, S, Hq, D = q.shape
    at_once = kv4.CHUNK_COLUMNS[D]
    blocks = -(-(Hq // cache.kv_heads * S) // at_once)
    flags = torch.full((blocks, batch, splits, cache.kv_heads), 7, dtype=torch.int32, device="cuda")
    part = torch.empty(batch * S * Hq * splits * (D + 1), dtype=torch.float32, device="cuda")
    out = torch.empty(batch, S, Hq, D + 1, dtype=torch.float32, device="cuda")
    args = [*cache._native, q.data_ptr(), *q.stride()[:3], table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(),
            part.data_ptr(), out.data_ptr(), batch, S, Hq, splits, 1, 2, scale]
    kv4._launch("tdist_kv4_chunk", cache.device, *args, 0, flags.data_ptr(), at_once)
    torch.cuda.synchronize()
    return flags.cpu()


@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (128, 128), (256, 64)])
def test_what_goes_to_the_other_kernel(D, group):
    """Exactly the splits and heads that hold something fp16 values do not reach are flagged; small values that they do reach, and
    small keys under ordinary queries, are not."""
    S, H, Hq, page, splits, L = 50, 2, 4, 16, 3, 600            # splits: tokens 0 .. 255, 256 .. 511, 512 .. 599
    cases = [
        ("nothing", None, []),
        ("small V", lambda k, v, q: v[192:256].mul_(2.0 ** -11), []),
        ("small K", lambda k, v, q: k[64:128].mul_(2.0 ** -17), []),
        ("small K of one token", lambda k, v, q: k[70].mul_(2.0 ** -17), []),
        ("V of zero", lambda k, v, q: v[0].zero_(), []),
        ("large K", lambda k, v, q: k[37, 1, 3].fill_(2.0 ** 16), [(0, 1)]),
        ("large V", lambda k, v, q: v[590:, 0].mul_(2.0 ** 17), [(2, 0)]),
        ("tiny V of one token", lambda k, v, q: v[300, 1].mul_(2.0 ** -24), [(1, 1)]),
        ("tiny V", lambda k, v, q: v[192:320].mul_(2.0 ** -24), [(0, 0), (0, 1), (1, 0), (1, 1)]),
        ("a NaN", lambda k, v, q: k[555, 0, 0].fill_(math.nan), [(2, 0)]),
        ("large queries, small K", lambda k, v, q: (q.mul_(2.0 ** 14), k[255, 0].mul_(2.0 ** -14)), [(0, 0)]),
        ("a page that is none", "page", [(1, 0), (1, 1)]),
    ]
    for name, change, wanted in cases:
        gen = _gen(45)
        cache, table, ks, vs = oracle.filled(gen, [L], H, D, group, page, torch.bfloat16, "cuda")
        k, v, q = ks[0].clone(), vs[0].clone(), oracle.rows(gen, 1, S, Hq, D, device="cuda")
        if change == "page":
            table[0, 20] = -1
        elif change is not None:
            change(k, v, q)
            kv4.kv4_append(k[None], v[None], cache, int32([0], "cuda"), table)
        flags = _flags(q, cache, int32([L], "cuda"), table, splits, D ** -0.5)
        expect = torch.zeros_like(flags)
        for split, head in wanted:
            expect[:, 0, split, head] = 1
        assert torch.equal(flags, expect), (name, flags.tolist())


CHUNKS = [
    # lens, S, Hq, Hkv, D, group, page, splits
    ([64], 64, 1, 1, 128, 64, 16, 1),
    ([300, 70, 0, 129], 70, 4, 2, 128, 64, 16, 1),
    ([777], 40, 14, 2, 128, 32, 48, 3),
    ([2000], 65, 2, 1, 128, 128, 64, 2),
    ([513, 1], 96, 4, 4, 64, 32, 16, 2),
    ([400], 150, 8, 4, 64, 64, 1040, 1),
    ([333, 900], 33, 8, 2, 256, 32, 16, 2),
    ([2000], 65, 1, 1, 256, 128, 16, 5),
]


def _fp16_rows(x, group, boost):
    """What the chunk kernel makes of rows: fp16(scale * code + low) from fp16 scale and low, all of them times ``boost``."""
    code, scale, low = kv4.quantise_reference(x.cpu(), group)
    s, w = ((t.double() * boost).half().double().repeat_interleave(group, -1) for t in (scale, low))
    return (code.double() * s + w).half().double() / boost


def _attention(q, keys, values, scale, causal):
    """fp64 (out, lse, sum of p |v - out|, largest sum of |q| |k| scale)."""
    B, S, Hq, D = q.shape
    out, spread = torch.zeros(B, S, Hq, D, dtype=torch.float64), torch.zeros(B, S, Hq, D, dtype=torch.float64)
    lse, terms = torch.full((B, S, Hq), -math.inf, dtype=torch.float64), 0.0
    q = q.double().cpu()
    for b in range(B):
        L, H = keys[b].shape[:2]
        for s in range(S):
            n = max(0, min(L, L - S + s + 1)) if causal else L
            if n == 0:
                continue
            for h in range(Hq):
                k, v = keys[b][:n, h // (Hq // H)], values[b][:n, h // (Hq // H)]
                x = k @ q[b, s, h] * scale
                p = torch.softmax(x, 0)
                out[b, s, h] = p @ v
                spread[b, s, h] = p @ (v - out[b, s, h]).abs()
                lse[b, s, h] = torch.logsumexp(x, 0)
                terms = max(terms, float((k.abs() @ q[b, s, h].abs()).max()) * abs(scale))
    return out, lse, spread, terms


@pytest.mark.parametrize("lens,S,Hq,H,D,group,page,splits", CHUNKS)
def test_many_columns_against_values_as_they_are_held(lens, S, Hq, H, D, group, page, splits, chunks):
    """Against fp64 over K and V as the kernel holds them, so that their rounding is not part of the tolerance.

    What is left: P is one fp16 number, and the sum that divides is of the same numbers: e_i <= 2^-11 moves the output by sum p_i e_i
    (v_i - out).  A score is summed in fp32 over D / 32 <= 8 products of 32 terms: 2^-24 each of their absolute sum, 2^-21 together and
    for two weights' difference twice, twice more for Q in log2 units and the exponential's argument: 2^-18 of the terms.  The sums over
    tokens are in fp32: 64 tokens at a time, 2^-24 each, under 2^-18 of the largest V.  The smallest weights, 2^-25 off next to a largest
    of 2^6 at least, are 2000 * 2^-31 < 2^-20 together."""
    gen = _gen(sum(lens) + S)
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda", room=max(lens) + 40)
    q = oracle.rows(gen, len(lens), S, Hq, D, device="cuda")
    keys, values = [_fp16_rows(x, group, 1.0) for x in ks], [_fp16_rows(x, group, 128.0) for x in vs]
    v_max = max(float(x.abs().max()) for x in values if x.numel())
    n = int32(lens, "cuda")
    for causal in (True, False):
        want, lse, spread, terms = _attention(q, keys, values, D ** -0.5, causal)
        full = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal, return_lse=True).double().cpu()
        out = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal).double().cpu()
        tol = (2.0 ** -11 + 2.0 ** -18 * terms) * spread + (2.0 ** -18 + 2.0 ** -20) * v_max
        off = (full[..., :D] - want).abs()
        assert (off <= tol).all(), float((off / tol.clamp(min=1e-12)).max())
        assert ((out - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()
        fine = lse != -math.inf
        assert torch.equal(full[..., D] == -math.inf, ~fine)
        assert ((full[..., D] - lse)[fine].abs() <= 2.0 ** -11 + 2.0 ** -18 * terms + 2.0 ** -22 * lse[fine].abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (256, 128)])
def test_many_columns_of_a_fp16_cache_are_as_exact_as_few(D, group):
    """A row that sees one token is its V; a prompt's rows are those of the same call in pieces of few columns.  At a size that is many
    columns' for bf16: a fp16 result has steps of 2^-11, and what is held in one fp16 number on the way would show.

    Row 0: P times scale is two fp16 numbers (2^-22 of 15 scale), P times low and the sums are fp32: under 2^-19 of 3 max |v|."""
    gen = _gen(D)
    S, H, Hq, page = 1536 if D == 256 else 2560, 2, 16, 64
    assert kv4.takes_chunks(1, H, S * Hq // H, D, S)
    table, pages = oracle.table_for(1, S, page, gen, device="cuda")
    cache = kv4.Int4KVCache.alloc(pages, page, H, D, group=group, dtype=torch.float16, device="cuda")
    k, v = (oracle.rows(gen, 1, S, H, D, dtype=torch.float16, device="cuda") for _ in range(2))
    kv4.kv4_append(k, v, cache, int32([0], "cuda"), table)
    q = oracle.rows(gen, 1, S, Hq, D, dtype=torch.float16, device="cuda")
    got = kv4.gqa_fwd_kv4(q, cache, int32([S], "cuda"), table, return_lse=True)
    torch.cuda.synchronize()
    held = oracle.held(v[0, 0], group).repeat_interleave(Hq // H, 0)
    top = held.abs().unflatten(-1, (-1, group)).amax(-1).repeat_interleave(group, -1)
    assert ((got[0, 0, :, :D].double().cpu() - held).abs() <= 2.0 ** -17 * top).all()
    # the same rows, few columns at a time: the same arithmetic but for the splits, whose weights are fp32 (2^-20 at most)
    for s in (1, 63, 700, S - 1):
        few = kv4.gqa_fwd_kv4(q[:, s:s + 1], cache, int32([s + 1], "cuda"), table, return_lse=True, kv_split=1)
        torch.cuda.synchronize()
        off = (got[0, s].double() - few[0, 0].double()).abs().cpu()
        assert (off[:, :D] <= 2.0 ** -13 * float(v.abs().max())).all(), float(off[:, :D].max())
        assert (off[:, D] <= 5e-4).all()


# ---- more sequences than a grid's dimension holds -----------------------------------------------------------------------
def test_more_sequences_than_a_grid_dimension_holds():
    gen = _gen(61)
    B, H, Hq, D, group, page = 65536 + 70, 1, 1, 64, 64, 16
    cpu = kv4.Int4KVCache.alloc(B + 1, page, H, D, group=group)
    gpu = kv4.Int4KVCache.alloc(B + 1, page, H, D, group=group, device="cuda")
    table = torch.randperm(B + 1, generator=gen)[:B].view(B, 1).int()
    x = oracle.rows(gen, B, 1, 3 * D)
    k, v = x[..., :D].view(B, 1, 1, D), x[..., D:2 * D].view(B, 1, 1, D)
    offset, news = torch.randint(0, 15, (B,), generator=gen).int(), torch.randint(0, 2, (B,), generator=gen).int()
    kv4.kv4_append(k, v, cpu, offset, table, new_lens=news)
    kv4.kv4_append(k.cuda(), v.cuda(), gpu, offset.cuda(), table.cuda(), new_lens=news.cuda())
    torch.cuda.synchronize()

    def same():
        return all(torch.equal(getattr(cpu, n), getattr(gpu, n).cpu()) for n in ("k_codes", "v_codes", "k_params", "v_params"))

    assert same()
    rope, pos, w = torch.ones(16, D // 2), offset.long().view(B, 1), torch.ones(D).bfloat16()
    outs = []
    for c, dev in ((cpu, "cpu"), (gpu, "cuda")):
        total = torch.zeros(B, dtype=torch.int32, device=dev)
        q = kv4.kv4_qkv_prep(x.to(dev), w.to(dev), None, 1e-6, 1e-6, pos.to(dev), rope.to(dev), rope.to(dev), c, offset.to(dev), total,
                             table.to(dev), Hq)
        outs.append((q.cpu(), total.cpu()))
    assert same() and torch.equal(outs[0][1], outs[1][1])
    # (Q's norm is in 32 bits on the GPU and in 64 here: a step of its rounding, and one of the result's, for values under 8)
    assert (outs[0][0] == outs[1][0]).float().mean() > 0.999 and ((outs[0][0] - outs[1][0]).abs() <= 2.0 ** -6 * 8).all()
