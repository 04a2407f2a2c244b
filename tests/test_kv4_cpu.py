"""4-bit KV cache on the CPU path: the format, the packed layout, bad pages, refusals, and the run of the operators together."""
import math

import pytest
import torch

import kv4_oracle as oracle
from kv4_oracle import int32
from triton_distributed_gh_amd.ops import kv4

FORMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,group", FORMS)
def test_rows_come_back_as_the_definition_says(D, group, dtype):
    gen = _gen(D + group)
    lens, page, H = [37, 0, 1, 64], 16, 3
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, dtype)
    cu = int32([0, 37, 37, 38, 102])
    k, v = kv4.kv4_read(cache, table, cu, 102)
    for got, raw in ((k, ks), (v, vs)):
        want = oracle.held(torch.cat(raw), group)
        # the value is one fp32 multiply-add (its product is exact), rounded to 16 bits: at most half a step, and 2^-24 of it
        assert ((got.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * want.abs() + 2.0 ** -26).all()


def test_reconstruction_error_is_half_a_step():
    """|x - value| <= scale / 2 and what the scale's own rounding does over fifteen steps (eps / 2 each), for finite rows."""
    gen = _gen(5)
    for dtype in (torch.bfloat16, torch.float16):
        x = oracle.rows(gen, 200, 1, 128, dtype=dtype)
        code, scale, low = kv4.quantise_reference(x, 64)
        back = kv4.dequantise_reference(code, scale, low)
        slack = 0.5 + 15 * torch.finfo(dtype).eps / 2
        assert ((back - x.float()).abs() <= slack * scale.float().repeat_interleave(64, -1) * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_constant_tiny_huge_and_nonfinite_groups(dtype):
    D, H = 64, 1
    x = torch.zeros(6, H, D, dtype=dtype)
    x[0] = 3.25                                             # no range: scale 0, the value itself
    x[1, :, ::2] = torch.finfo(dtype).max
    x[1, :, 1::2] = -torch.finfo(dtype).max                 # bf16: the range itself overflows fp32
    x[2, 0, 5] = math.inf
    x[3, 0, 5] = math.nan
    x[4, 0, 40] = -math.inf                                 # second group of 32 only
    x[5, 0, 0] = torch.finfo(dtype).smallest_normal
    cache = kv4.Int4KVCache.alloc(1, 16, H, D, group=32, dtype=dtype)
    table = int32([[0]])
    kv4.kv4_append(x[None], x[None], cache, int32([0]), table)
    for got in kv4.kv4_read(cache, table, int32([0, 6]), 6):
        assert (got[0] == 3.25).all()
        if dtype == torch.float16:
            assert (got[1].double() - x[1].double()).abs().max() <= 65504 * 2.0 ** -11
        else:
            assert got[1].isnan().all()
        assert got[2, 0, :32].isnan().all() and (got[2, 0, 32:] == 0).all()
        assert got[3, 0, :32].isnan().all() and (got[3, 0, 32:] == 0).all()
        assert got[4, 0, 32:].isnan().all() and (got[4, 0, :32] == 0).all()
        assert got[5].isfinite().all() and got[5].abs().max() <= 2 * torch.finfo(dtype).smallest_normal


def test_offsets_padding_starts_and_rows_behind_the_last_sequence():
    gen = _gen(1)
    B, S, H, D, group, page = 3, 9, 2, 128, 64, 16
    table, pages = oracle.table_for(B, 64, page, gen)
    cache = kv4.Int4KVCache.alloc(pages, page, H, D, group=group)
    first = oracle.rows(gen, B, 20, H, D)
    kv4.kv4_append(first, -first, cache, int32([0, 0, 0]), table)
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params)]
    k, v = oracle.rows(gen, B, S, H, D), oracle.rows(gen, B, S, H, D)
    offsets, news = [3, 14, 61], [9, 0, 7]                  # in the middle; nothing; over the end of the last page
    kv4.kv4_append(k, v, cache, int32(offsets), table, new_lens=int32(news))
    # the sequence without new tokens kept every bit
    own = table[1].long()
    for was, now in zip(before, (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params)):
        assert torch.equal(was[own], now[own])
    out = (torch.full((20, H, D), 7.0, dtype=torch.bfloat16), torch.full((20, H, D), 7.0, dtype=torch.bfloat16))
    kk, vv = kv4.kv4_read(cache, table, int32([0, 9, 9, 16]), 20, starts=int32(offsets), out=out)
    assert kk is out[0] and (kk[16:] == 7).all() and (vv[16:] == 7).all()
    want = oracle.held(k, group)
    assert (kk[:9].double() - want[0]).abs().max() <= 2.0 ** -8 * want.abs().max()
    assert (kk[9:12].double() - want[2, :3]).abs().max() <= 2.0 ** -8 * want.abs().max()
    assert (kk[12:16] == 0).all() and (vv[12:16] == 0).all()        # tokens 64 .. 67: no page
    # tokens 0 .. 2 of the first sequence and 12 .. are still the old ones
    k0, v0 = kv4.kv4_read(cache, table, int32([0, 20, 20, 20]), 20)
    old = oracle.held(first, group)[0]
    keep = [0, 1, 2, *range(12, 20)]
    assert (k0[keep].double() - old[keep]).abs().max() <= 2.0 ** -8 * old.abs().max()
    assert (v0[keep].double() - oracle.held(-first, group)[0][keep]).abs().max() <= 2.0 ** -8 * old.abs().max()


def test_entries_that_are_no_page_are_dropped_read_as_zeros_and_not_attended():
    gen = _gen(2)
    H, D, group, page = 2, 64, 32, 16
    cache = kv4.Int4KVCache.alloc(4, page, H, D, group=group)
    table = int32([[2, -1, 0, 99]])
    k, v = oracle.rows(gen, 1, 64, H, D), oracle.rows(gen, 1, 64, H, D)
    kv4.kv4_append(k, v, cache, int32([0]), table)
    assert (cache.k_codes[[1, 3]] == 0).all() and (cache.v_params[[1, 3]] == 0).all()
    kk, vv = kv4.kv4_read(cache, table, int32([0, 64]), 64)
    there = torch.zeros(64, dtype=torch.bool)
    there[0:16] = there[32:48] = True
    assert (kk[~there] == 0).all() and (vv[~there] == 0).all() and (kk[there] != 0).any()
    q = oracle.rows(gen, 1, 2, 4, D)
    got = kv4.gqa_fwd_kv4(q, cache, int32([64]), table, return_lse=True).double()
    want, lse = oracle.attention(q, [oracle.held(k[0], group)], [oracle.held(v[0], group)], D ** -0.5, there=[there])
    assert (got[..., :D] - want).abs().max() < 1e-4 and (got[..., D] - lse).abs().max() < 1e-4
    none = kv4.gqa_fwd_kv4(q, cache, int32([64]), int32([[-1, -1, 7, 99]]), return_lse=True)
    assert (none[..., :D] == 0).all() and (none[..., D] == -math.inf).all()


@pytest.mark.parametrize("S,causal,soft_cap", [(1, True, 0.0), (3, True, 0.0), (3, False, 0.0), (2, True, 20.0)])
def test_attention_against_the_definition(S, causal, soft_cap):
    gen = _gen(3)
    lens, H, D, group, page = [33, 0, 1, 2, 80], 2, 128, 64, 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page)
    q = oracle.rows(gen, len(lens), S, 6, D)
    got = kv4.gqa_fwd_kv4(q, cache, int32(lens), table, scale=0.07, soft_cap=soft_cap, causal=causal, return_lse=True).double()
    want, lse = oracle.attention(q, [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs], 0.07, soft_cap, causal)
    assert (got[..., :D] - want).abs().max() < 1e-4
    assert torch.equal(got[..., D] == -math.inf, lse == -math.inf)
    fine = lse != -math.inf
    assert (got[..., D] - lse)[fine].abs().max() < 1e-4


def test_projection_writes_what_append_would():
    gen = _gen(4)
    B, S, Hq, H, D, group, page = 2, 5, 4, 2, 128, 32, 16
    table, pages = oracle.table_for(B, 48, page, gen)
    a, b = (kv4.Int4KVCache.alloc(pages, page, H, D, group=group) for _ in range(2))
    qkv = oracle.rows(gen, B, S, Hq + 2 * H, D).flatten(2)
    qw, kw = (1 + 0.1 * torch.randn(D, generator=gen)).bfloat16(), (1 + 0.1 * torch.randn(D, generator=gen)).bfloat16()
    ang = torch.outer(torch.arange(64.0), 1e4 ** (-torch.arange(0, D, 2) / D))
    cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
    offset, total = int32([0, 30]), int32([0, 0])
    pos = offset[:, None].long() + torch.arange(S)
    q = kv4.kv4_qkv_prep(qkv, qw, kw, 1e-6, 1e-6, pos, cos, sin, a, offset, total, table, Hq)
    assert total.tolist() == [5, 35]
    x = qkv.unflatten(-1, (-1, D)).double()
    normed = (x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()).float()

    def turned(rows, w):
        rows = (rows.double() * w.double()).bfloat16().double()
        c, s = cos[pos].unsqueeze(2).double(), sin[pos].unsqueeze(2).double()
        f, g = rows.chunk(2, -1)
        return torch.cat([f * c - g * s, g * c + f * s], -1)

    want_q, want_k = turned(normed[:, :, :Hq], qw), turned(normed[:, :, Hq:Hq + H], kw)
    # a norm that rounds the other way moves both members of a rotated pair by half a step, the rotation rounds once more
    def near(got, want):
        pair = (want.chunk(2, -1)[0].square() + want.chunk(2, -1)[1].square()).sqrt().repeat(1, 1, 1, 2)
        return ((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + 2 * pair)).all()

    assert near(q, want_q)
    kv4.kv4_append(want_k.bfloat16(), x[:, :, Hq + H:].bfloat16(), b, offset, table)
    assert torch.equal(a.v_codes, b.v_codes) and torch.equal(a.v_params, b.v_params)
    same = (a.k_codes == b.k_codes).float().mean()
    assert same > 0.999


def test_a_prompt_and_decode_steps_together():
    """append -> attend -> append one -> attend, against rows kept outside of the cache."""
    gen = _gen(6)
    B, H, Hq, D, group, page = 2, 2, 4, 64, 32, 16
    table, pages = oracle.table_for(B, 48, page, gen)
    cache = kv4.Int4KVCache.alloc(pages, page, H, D, group=group)
    ks, vs = [torch.zeros(0, H, D, dtype=torch.bfloat16)] * B, [torch.zeros(0, H, D, dtype=torch.bfloat16)] * B
    offset = int32([0, 0])
    for S in (13, 1, 1, 4, 1):
        k, v, q = oracle.rows(gen, B, S, H, D), oracle.rows(gen, B, S, H, D), oracle.rows(gen, B, S, Hq, D)
        kv4.kv4_append(k, v, cache, offset, table)
        offset = offset + S
        ks, vs = [torch.cat([a, b]) for a, b in zip(ks, k)], [torch.cat([a, b]) for a, b in zip(vs, v)]
        got = kv4.flash_attn_with_kv4cache(q, cache, offset, table).double()
        want, _ = oracle.attention(q, [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs], D ** -0.5)
        assert ((got - want).abs() <= oracle.bounds(want, torch.bfloat16, max(float(x.abs().max()) for x in vs))).all()


def test_masked_nan_does_not_reach_earlier_queries():
    gen = _gen(7)
    H, D, group, page, S = 1, 64, 64, 16, 3
    table, pages = oracle.table_for(1, 32, page, gen)
    cache = kv4.Int4KVCache.alloc(pages, page, H, D, group=group)
    k, v = oracle.rows(gen, 1, 20, H, D), oracle.rows(gen, 1, 20, H, D)
    k[0, 19], v[0, 19] = math.nan, math.nan                 # the last token is seen by the last query alone
    kv4.kv4_append(k, v, cache, int32([0]), table)
    out = kv4.gqa_fwd_kv4(oracle.rows(gen, 1, S, 2, D), cache, int32([20]), table)
    assert out[0, 0].isfinite().all() and out[0, 2].isnan().all()


def _valid():
    gen = _gen(8)
    cache = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32)
    return dict(k=oracle.rows(gen, 2, 3, 2, 64), v=oracle.rows(gen, 2, 3, 2, 64), cache=cache, kv_offset=int32([0, 0]),
                block_table=int32([[0, 1], [2, 3]]))


@pytest.mark.parametrize("change,error", [
    (dict(k=torch.zeros(2, 3, 2, 64)), TypeError),
    (dict(k=torch.zeros(2, 3, 2, 64, dtype=torch.float16)), TypeError),
    (dict(k=torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(kv_offset=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(kv_offset=int32([0])), ValueError),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), ValueError),
    (dict(block_table=int32([[0, 1]])), ValueError),
    (dict(block_table=int32([[0, 1, 2, 3], [0, 1, 2, 3]])[:, ::2]), ValueError),
    (dict(new_lens=int32([1, 1, 1])), ValueError),
    (dict(k=torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, requires_grad=True)), RuntimeError),
])
def test_append_refuses(change, error):
    args = {**_valid(), **change}
    with pytest.raises(error):
        kv4.kv4_append(**args)


def test_caches_that_cannot_be():
    for bad in (dict(page_size=24), dict(page_size=0), dict(head_dim=96), dict(group=16), dict(group=128), dict(dtype=torch.float32),
                dict(num_pages=0)):
        args = {**dict(num_pages=2, page_size=16, kv_heads=1, head_dim=64, group=32, dtype=torch.bfloat16), **bad}
        with pytest.raises((ValueError, TypeError)):
            kv4.Int4KVCache.alloc(**args)
    c = kv4.Int4KVCache.alloc(2, 16, 1, 64, group=32)
    with pytest.raises(ValueError):
        kv4.Int4KVCache(c.k_codes, c.v_codes[:, :, :2], c.k_params, c.v_params)
    with pytest.raises(ValueError):
        kv4.Int4KVCache(c.k_codes, c.v_codes, c.k_params[:1], c.v_params)
    with pytest.raises(TypeError):
        kv4.Int4KVCache(c.k_codes, c.v_codes, c.k_params, c.v_params.half())


@pytest.mark.parametrize("call", [
    lambda c, t: kv4.gqa_fwd_kv4(torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16), c, int32([1, 1]), t),
    lambda c, t: kv4.gqa_fwd_kv4(torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16), c, int32([1, 1]), t),
    lambda c, t: kv4.gqa_fwd_kv4(torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16), c, int32([1, 1]), t),
    lambda c, t: kv4.gqa_fwd_kv4(torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16), c, int32([1, 1]).long(), t),
    lambda c, t: kv4.gqa_fwd_kv4(torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16), c, int32([1, 1]), t, soft_cap=-1.0),
    lambda c, t: kv4.gqa_fwd_kv4(torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16), c, int32([1, 1]), t, kv_split=0),
    lambda c, t: kv4.kv4_read(c, t, int32([0, 1]), 2),
    lambda c, t: kv4.kv4_read(c, t, int32([0, 1, 2]), -1),
    lambda c, t: kv4.kv4_read(c, t, int32([0, 1, 2]), 2, out=(torch.zeros(2, 2, 64, dtype=torch.bfloat16),) * 2, starts=int32([0])),
    lambda c, t: kv4.kv4_read(c, t, int32([0, 1, 2]), 2, out=(torch.zeros(3, 2, 64, dtype=torch.bfloat16),) * 2),
])
def test_reads_and_attention_refuse(call):
    cache, table = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32), int32([[0, 1], [2, 3]])
    with pytest.raises(ValueError):
        call(cache, table)


def test_types_that_are_refused():
    cache, table = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32), int32([[0, 1], [2, 3]])
    with pytest.raises(TypeError):
        kv4.gqa_fwd_kv4(torch.zeros(2, 1, 2, 64, dtype=torch.float16), cache, int32([1, 1]), table)
    half = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32, dtype=torch.float16)
    z = torch.zeros(1, 32)
    with pytest.raises(TypeError):
        kv4.kv4_qkv_prep(torch.zeros(2, 1, 6 * 64, dtype=torch.float16), None, None, 0.0, 0.0, torch.zeros(2, 1).long(), z, z, half,
                         int32([0, 0]), int32([0, 0]), table, 2)


def test_empty_calls():
    cache, table = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32), int32([[0, 1], [2, 3]])
    none = torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16)
    kv4.kv4_append(none, none, cache, int32([0, 0]), table)
    assert kv4.gqa_fwd_kv4(none, cache, int32([0, 0]), table).shape == (2, 0, 2, 64)
    assert kv4.kv4_read(cache, table, int32([0, 0, 0]), 0)[0].shape == (0, 2, 64)
    zero = torch.zeros(0, 3, 2, 64, dtype=torch.bfloat16)
    kv4.kv4_append(zero, zero, cache, int32([]), torch.zeros(0, 2, dtype=torch.int32))
    assert (cache.k_codes == 0).all()


def test_argument_types_of_the_native_calls_match_the_sources():
    import re

    from triton_distributed_gh_amd import build

    source = "".join((build.CSRC / "ops" / f).read_text() for f in ("kv4.hip", "kv4_attn.hip", "kv4_chunk.hip"))
    for name, signature in kv4._SIGNATURES.items():
        args = re.search(rf"TDIST_API int {name}\((.*?)\) \{{", source, re.S).group(1).split(",")
        kinds = ["p" if "*" in a else "q" if "long long" in a else "f" if "float" in a else "i" for a in args]
        assert "".join(kinds) == signature, name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_layer_over_a_4bit_cache(dtype):
    from kv4_layer_checks import attention_layer

    attention_layer("cpu", dtype)


def test_engine_with_a_4bit_cache(monkeypatch):
    monkeypatch.setenv("RANDOM_PARAMS", "1")
    monkeypatch.setenv("TDIST_NO_HF_CONFIG", "1")
    from triton_distributed_gh_amd.models import Engine, KV4_Cache, ModelConfig

    config = ModelConfig(model_name="tdist/tiny-dense", max_length=64, dtype=torch.bfloat16, rank=0, world_size=1)
    with pytest.raises(ValueError):
        Engine(config, kv_cache_bits=8)
    eng = Engine(config, kv_cache_bits=4)
    ids = torch.randint(0, 1000, (2, 9), generator=_gen(3))
    first = eng.serve(ids, gen_len=4)
    assert isinstance(eng.kv_cache, KV4_Cache) and eng.kv_cache.get_kv_len().tolist() == [13, 13]
    assert first.shape == (2, 4) and torch.equal(first, eng.serve(ids, gen_len=4))


def test_facade_serves_the_operators():
    import triton_dist.kernels.amd.kv4 as facade
    from triton_dist.models.kv_cache import KV4_Cache  # noqa: F401

    assert facade is kv4


def test_a_table_without_pages_is_empty_sequences():
    _no_pages("cpu")


def _no_pages(device):
    gen = _gen(51)
    cache = kv4.Int4KVCache.alloc(2, 16, 2, 64, group=32, device=device)
    table = torch.zeros(3, 0, dtype=torch.int32, device=device)
    rows = oracle.rows(gen, 3, 2, 2, 64, device=device)
    kv4.kv4_append(rows, rows, cache, int32([0, 1, 5], device), table)
    assert not cache.k_params.any() and not cache.v_codes.any()
    out = kv4.gqa_fwd_kv4(rows, cache, int32([2, 9, 0], device), table, return_lse=True)
    assert not out[..., :64].any() and (out[..., 64] == -math.inf).all()
    k, v = kv4.kv4_read(cache, table, int32([0, 1, 2, 4], device), 4)
    assert not k.any() and not v.any()


def test_projection_refuses_to_write_over_the_offsets_it_reads():
    cache = kv4.Int4KVCache.alloc(4, 16, 1, 64, group=32)
    table, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    qkv, rope = torch.zeros(2, 1, 3 * 64, dtype=torch.bfloat16), torch.ones(8, 32)
    pos = torch.zeros(2, 1, dtype=torch.int64)
    for total in (n[:2], n[1:]):
        with pytest.raises(ValueError, match="share memory"):
            kv4.kv4_qkv_prep(qkv, None, None, 0.0, 0.0, pos, rope, rope, cache, n[:2], total, table, 1)
    kv4.kv4_qkv_prep(qkv, None, None, 0.0, 0.0, pos, rope, rope, cache, n[:2], int32([0, 0]), table, 1)


def test_tables_of_more_than_2_to_the_30_tokens_are_refused():
    cache = kv4.Int4KVCache.alloc(1, 1 << 20, 1, 64, group=64)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    table = torch.full((1, 1025), -1, dtype=torch.int32)
    with pytest.raises(ValueError, match="2\\^30"):
        kv4.gqa_fwd_kv4(q, cache, int32([1]), table)
    kv4.gqa_fwd_kv4(q, cache, int32([1]), table[:, :1024])


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_split_and_chunk_rules_stay_within_their_launches(head_dim):
    for batch in (0, 1, 7, 64, 70000):
        for columns in (0, 1, 5, 100, 1000, 1 << 20):
            for capacity in (0, 16, 500, 4096, 1 << 30):
                for chunk in (False, True):
                    splits = kv4.auto_kv_splits(batch, 8, columns, head_dim, capacity, chunk=chunk)
                    assert 1 <= splits <= 64 and (splits == 1 or capacity // splits >= 128)
                assert not kv4.takes_chunks(batch, 8, columns, head_dim, capacity, 1.0)
    assert not kv4.takes_chunks(64, 8, 16, head_dim, 1 << 20)
    assert kv4.takes_chunks(1, 8, 4096, head_dim, 16384)


def test_copies_of_a_cache_have_their_own_memory():
    import copy
    import pickle

    gen = _gen(52)
    cache, table, _, _ = oracle.filled(gen, [20], 2, 64, 32, 16)
    before = cache.k_codes.clone()
    for twin in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        tensors = (twin.k_codes, twin.v_codes, twin.k_params, twin.v_params)
        assert twin._native[:4] == tuple(t.data_ptr() for t in tensors) and twin._native[4:] == cache._native[4:]
        rows = oracle.rows(gen, 1, 20, 2, 64)
        kv4.kv4_append(rows, rows, twin, int32([0]), table)
        assert torch.equal(cache.k_codes, before) and not torch.equal(twin.k_codes, before)


def test_tables_whose_rows_are_2_to_the_31_entries_apart_are_refused():
    """The kernels take a row's distance in 32 bits: a longer one would be cut, and the rows looked for elsewhere."""
    cache = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32, device="meta")
    rows, cu = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="meta"), int32([0, 1, 2], "meta")
    n = int32([1, 1], "meta")
    far = torch.empty_strided((2, 2), (2 ** 31, 1), dtype=torch.int32, device="meta")
    for call in (lambda: kv4.kv4_append(rows, rows, cache, n, far), lambda: kv4.kv4_read(cache, far, cu, 2),
                 lambda: kv4.gqa_fwd_kv4(rows, cache, n, far),
                 lambda: kv4.kv4_qkv_prep(rows.view(2, 1, 128).repeat(1, 1, 3), None, None, 0.0, 0.0, n.long().view(2, 1),
                                          torch.zeros(8, 32, device="meta"), torch.zeros(8, 32, device="meta"), cache, n, n.clone(), far, 2)):
        with pytest.raises(ValueError, match="2\\^31 entries"):
            call()
    near = torch.empty_strided((2, 2), (2 ** 31 - 1, 1), dtype=torch.int32, device="meta")
    assert kv4._check_table(cache, 2, near) == 2


@pytest.mark.parametrize("soft_cap", [1e-60, 1e-39, 2.0, 1e4, 1e7, 1e30, 3e38, 1e60])
def test_caps_of_any_size(soft_cap):
    gen = _gen(53)
    lens, H, D, group, page = [70, 3], 2, 64, 32, 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page)
    q = oracle.rows(gen, 2, 2, 4, D)
    got = kv4.gqa_fwd_kv4(q, cache, int32(lens), table, scale=0.1, soft_cap=soft_cap, return_lse=True).double()
    want, lse = oracle.attention(q, [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs], 0.1, soft_cap)
    assert (got[..., :D] - want).abs().max() < 1e-4 and (got[..., D] - lse).abs().max() < 1e-4


def test_lds_writes_and_reads_of_other_lanes_keep_their_order(tmp_path):
    """Each lane writes its neighbour's word and reads its own: never the same address in one lane, so that the compiler may issue the
    read first (and it does), unless it is told that the lanes meet there."""
    import subprocess

    from triton_distributed_gh_amd import build

    source = tmp_path / "probe.hip"
    source.write_text("""#include "tdist/kv4.hpp"
template <bool MEET>
__global__ void probe(float* out, const float* in) {
  __shared__ float s[65];
  s[threadIdx.x + 1] = in[threadIdx.x];
  if (MEET) tdist::kv4::lanes_meet();
  out[threadIdx.x] = s[threadIdx.x];
}
template __global__ void probe<true>(float*, const float*);
""")
    asm = subprocess.run([build._hipcc(), *build.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", "-", str(source)], check=True,
                         capture_output=True, text=True).stdout
    order = [line.split()[0] for line in asm.splitlines() if line.strip().startswith(("ds_write", "ds_read"))]
    assert order == ["ds_write_b32", "ds_read_b32"]
    # the places where the kernels hand data from lane to lane of one wave: a tile of V that is written, rows of V that are read
    # back, a block's parameters and weights
    for name, least in (("kv4.hip", 4), ("kv4_attn.hip", 3)):
        assert (build.CSRC / "ops" / name).read_text().count("lanes_meet();") >= least


@pytest.mark.parametrize("which", ["k_codes", "v_codes", "k_params", "v_params"])
@pytest.mark.parametrize("change", [
    lambda t: t.set_(t.clone()),
    lambda t: t.resize_(4 * t.shape[0], *t.shape[1:]),
    lambda t: setattr(t, "data", t.clone()),
    lambda t: t.untyped_storage().resize_(0),
])
def test_a_cache_whose_tensors_got_other_memory_is_refused(which, change):
    """The kernels go by the addresses that the cache was made with: what is there may have been freed."""
    gen = _gen(54)
    cache, table, _, _ = oracle.filled(gen, [20], 2, 64, 32, 16)
    rows, n = oracle.rows(gen, 1, 1, 2, 64), int32([20])
    kv4.gqa_fwd_kv4(rows, cache, n, table)
    keep = change(getattr(cache, which))
    rope, pos = torch.ones(32, 32), torch.zeros(1, 1, dtype=torch.int64)
    for call in (lambda: kv4.gqa_fwd_kv4(rows, cache, n, table), lambda: kv4.kv4_append(rows, rows, cache, n, table),
                 lambda: kv4.kv4_read(cache, table, int32([0, 20]), 20),
                 lambda: kv4.kv4_qkv_prep(torch.cat([rows] * 3, 2).flatten(2), None, None, 0.0, 0.0, pos, rope, rope, cache, n, int32([0]),
                                          table, 2)):
        with pytest.raises(RuntimeError, match="other memory"):
            call()
    del keep


def _calls_with(change):
    """The entry points with each of their floating-point inputs passed through ``change`` in turn."""
    gen = _gen(55)
    cache, table, _, _ = oracle.filled(gen, [20], 2, 64, 32, 16)
    x, n, pos = oracle.rows(gen, 1, 1, 2, 64), int32([20]), torch.zeros(1, 1, dtype=torch.int64)
    qkv, w, rope = torch.cat([x] * 3, 2).flatten(2), torch.ones(64).bfloat16(), torch.ones(32, 32)
    prep = lambda *a: kv4.kv4_qkv_prep(a[0], a[1], a[2], 0.0, 0.0, pos, a[3], a[4], cache, n, int32([0]), table, 2)  # noqa: E731
    out = torch.zeros(20, 2, 64, dtype=torch.bfloat16)
    for call, args in ((lambda q: kv4.gqa_fwd_kv4(q, cache, n, table), [x]),
                       (lambda q: kv4.flash_attn_with_kv4cache(q, cache, n, table), [x]),
                       (lambda k, v: kv4.kv4_append(k, v, cache, n, table), [x, x.clone()]),
                       (prep, [qkv, w, w.clone(), rope, rope.clone()]),
                       (lambda k, v: kv4.kv4_read(cache, table, int32([0, 20]), 20, out=(k, v)), [out, out.clone()])):
        call(*args)
        for i in range(len(args)):
            yield lambda: call(*args[:i], change(args[i]), *args[i + 1:])


def test_inputs_that_carry_a_tangent_or_require_a_gradient_are_refused():
    from torch.autograd import forward_ad

    for call in _calls_with(lambda t: t.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    with forward_ad.dual_level():
        for call in _calls_with(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
    with torch.no_grad():
        for call in _calls_with(lambda t: t.clone().requires_grad_()):
            call()
    cache = kv4.Int4KVCache.alloc(1, 16, 1, 64)
    with pytest.raises(ValueError, match="gradient"):
        kv4.Int4KVCache(cache.k_codes, cache.v_codes, cache.k_params.clone().requires_grad_(), cache.v_params)


def test_results_that_share_memory_are_refused():
    cache, table, cu = kv4.Int4KVCache.alloc(4, 16, 2, 64, group=32), int32([[0, 1], [2, 3]]), int32([0, 3, 5])
    x = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    k, v = kv4.kv4_read(cache, table, cu, 5, out=(x[:, :2], x[:, 2:]))     # parts of the same rows
    assert k.data_ptr() == x.data_ptr() and v.data_ptr() == x[:, 2:].data_ptr()
    own = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    for out in ((x[:, :2], x[:, :2]), (x[:1, :2].expand(5, 2, 64), own), (own, x[:, :1].expand(5, 2, 64))):
        with pytest.raises(ValueError, match="memory"):
            kv4.kv4_read(cache, table, cu, 5, out=out)
