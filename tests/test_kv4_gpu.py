"""4-bit KV cache kernels: the bits of the CPU path, and attention against its definition in 64 bits."""
import math

import pytest
import torch

import kv4_oracle as oracle
from kv4_oracle import int32
from triton_distributed_gh_amd.ops import flash_decode, kv4

pytestmark = pytest.mark.gpu

FORMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]
DTYPES = [torch.bfloat16, torch.float16]


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _to(cache, device):
    return kv4.Int4KVCache(*(t.to(device) for t in (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params)))


def _same(a, b):
    """The same bits, but for the low of a group that holds a NaN or an infinity (its scale is NaN on both sides)."""
    assert torch.equal(a.k_codes.cpu(), b.k_codes.cpu()) and torch.equal(a.v_codes.cpu(), b.v_codes.cpu())
    for x, y in ((a.k_params.cpu(), b.k_params.cpu()), (a.v_params.cpu(), b.v_params.cpu())):
        bad = x[..., 0].isnan()
        assert torch.equal(bad, y[..., 0].isnan())
        assert torch.equal(x[~bad], y[~bad])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,group", FORMS)
def test_append_and_read_give_the_bits_of_the_cpu_path(D, group, dtype):
    gen = _gen(D + group)
    B, S, H, page = 3, 45, 3, 48
    table, pages = oracle.table_for(B, 100, page, gen)
    cpu = kv4.Int4KVCache.alloc(pages, page, H, D, group=group, dtype=dtype)
    gpu = _to(cpu, "cuda")
    k, v = oracle.rows(gen, B, S, H, D, dtype=dtype), oracle.rows(gen, B, S, H, D, dtype=dtype)
    k[0, 3, 1, 5], v[1, 2, 0, 7], v[2, 1, 2, D - 1] = math.nan, math.inf, -math.inf
    k[2, 4], v[2, 4] = 1.5, 0.0                             # no range
    k[1, 0, 0, ::2], k[1, 0, 0, 1::2] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    v[1, 1] *= 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -124       # scales at the bottom of the type
    offsets, news = int32([0, 31, 97]), int32([45, 13, 45])                # in order; in the middle; over the end
    kv4.kv4_append(k, v, cpu, offsets, table, new_lens=news)
    kv4.kv4_append(k.cuda(), v.cuda(), gpu, offsets.cuda(), table.cuda(), new_lens=news.cuda())
    torch.cuda.synchronize()
    _same(cpu, gpu)
    cu, starts = int32([2, 60, 60, 110]), int32([0, 5, 60])
    outs = []
    for c, dev in ((cpu, "cpu"), (gpu, "cuda")):
        out = tuple(torch.full((115, H, D), 7.0, dtype=dtype, device=dev) for _ in range(2))
        outs.append(kv4.kv4_read(c, table.to(dev), cu.to(dev), 115, starts=starts.to(dev), out=out))
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        b = b.cpu()
        assert (b[:2] == 7).all() and (b[110:] == 7).all()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


@pytest.mark.parametrize("S", [1, 2, 3, 4, 5, 17, 64, 65])
def test_append_token_counts_and_strided_rows(S):
    gen = _gen(S)
    B, H, D, group, page = 2, 5, 128, 64, 16
    table, pages = oracle.table_for(B, 96, page, gen)
    cpu = kv4.Int4KVCache.alloc(pages, page, H, D, group=group)
    gpu = _to(cpu, "cuda")
    qkv = oracle.rows(gen, B, S, 3 * H, D)                  # K and V as parts of one projection's rows
    odd = oracle.rows(gen, B, S, H, D + 4)                  # rows that are not 16-byte aligned: copied by the call
    offsets = int32([7, 30])
    for k, v in ((qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]), (odd[..., 4:], odd[..., :D]),
                 (qkv[:, :, :H].transpose(0, 1).contiguous().transpose(0, 1), qkv[:, :, H:2 * H])):
        dk, dv = (x.to("cuda") for x in (qkv, odd))
        strided = {qkv.data_ptr(): dk, odd.data_ptr(): dv}

        def there(x):
            base = strided.get(x.untyped_storage().data_ptr())
            return x.cuda() if base is None else torch.as_strided(base, x.shape, x.stride(), x.storage_offset())

        kv4.kv4_append(k, v, cpu, offsets, table)
        kv4.kv4_append(there(k), there(v), gpu, offsets.cuda(), table.cuda())
        torch.cuda.synchronize()
        _same(cpu, gpu)


@pytest.mark.parametrize("D,group,page", [(64, 32, 16), (128, 64, 48), (256, 128, 16)])
def test_reads_that_start_anywhere(D, group, page):
    """Sequences of 0 .. 70 rows that start at any token, in front of the first one and behind the last page too; more
    sequences than a wave looks up at a time."""
    gen = _gen(31)
    B, H = 70, 2
    cpu, table, _, _ = oracle.filled(gen, [96] * B, H, D, group, page)
    lens = torch.randint(0, 71, (B,), generator=gen)
    lens[3:9] = 0
    starts = torch.randint(-5, 90, (B,), generator=gen).int()
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0).int()])
    total = int(cu[-1])
    want = kv4.kv4_read(cpu, table, cu, total, starts=starts)
    got = kv4.kv4_read(_to(cpu, "cuda"), table.cuda(), cu.cuda(), total, starts=starts.cuda())
    some = kv4.kv4_read(_to(cpu, "cuda"), table.cuda(), cu.cuda(), total - 37, starts=starts.cuda())
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, some):
        assert torch.equal(a, b.cpu()) and torch.equal(a[:total - 37], c.cpu())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_one_row_of_each_of_many_sequences(D):
    """A decode step's rows: one of each sequence, some without any - more than sixty of those in a row."""
    gen = _gen(32)
    B, H, group, page = 300, 2, 64, 16
    lens = torch.ones(B, dtype=torch.int64)
    lens[10:90] = 0
    lens[::17] = 0
    lens[200:210] = 3
    cpu, table, _, _ = oracle.filled(gen, [16] * B, H, D, group, page)
    starts = torch.randint(0, 14, (B,), generator=gen).int()
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0).int()])
    total = int(cu[-1])
    want = kv4.kv4_read(cpu, table, cu, total, starts=starts)
    got = kv4.kv4_read(_to(cpu, "cuda"), table.cuda(), cu.cuda(), total, starts=starts.cuda())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.cpu()) for a, b in zip(want, got))


def test_append_leaves_everything_else_alone():
    """Bytes around the written tokens, and pages of other sequences, keep their bits."""
    gen = _gen(11)
    H, D, group, page = 2, 128, 128, 16
    cache, table, _, _ = oracle.filled(gen, [60, 60], H, D, group, page, device="cuda")
    table = table.clone()
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params)]
    bad = table.clone()
    bad[0, 1], bad[0, 2] = -5, cache.num_pages              # tokens 16 .. 47 of the first sequence go nowhere
    k = oracle.rows(gen, 2, 40, H, D, device="cuda")
    kv4.kv4_append(k, k, cache, int32([14, 100], "cuda"), bad)      # the second sequence is behind its table
    torch.cuda.synchronize()
    touched = torch.zeros(cache.num_pages, page, dtype=torch.bool)
    touched[int(table[0, 0]), 14:] = True
    touched[int(table[0, 3]), :6] = True
    touched = touched.cuda()
    now = (cache.k_codes, kv4._v_units(cache), cache.k_params, cache.v_params)
    was = (before[0], kv4._v_units(kv4.Int4KVCache(*before)), before[2], before[3])
    for i, (a, b) in enumerate(zip(was, now)):
        if i == 1:                                          # [pages, H, quads, 16, halves, 4, 2] -> tokens in front
            a, b = (x.permute(0, 2, 5, 1, 3, 4, 6).flatten(1, 2).flatten(2) for x in (a, b))
        elif i == 0:
            a, b = (x.transpose(1, 2).flatten(2) for x in (a, b))
        else:
            a, b = (x.permute(0, 3, 1, 2, 4).flatten(2) for x in (a, b))
        assert torch.equal(a[~touched], b[~touched])
        assert not torch.equal(a[touched], b[touched])


@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (128, 128), (256, 32)])
@pytest.mark.parametrize("B,S,norm", [(3, 1, True), (2, 7, True), (1, 150, False)])
def test_projection_writes_the_bits_of_the_cpu_path(D, group, B, S, norm):
    gen = _gen(D + S)
    Hq, H, page = 6, 2, 32
    table, pages = oracle.table_for(B, 192, page, gen)
    cpu = kv4.Int4KVCache.alloc(pages, page, H, D, group=group)
    gpu = _to(cpu, "cuda")
    wide = oracle.rows(gen, B, S, (Hq + 2 * H) * D + 8)
    qw, kw = ((1 + 0.1 * torch.randn(2, D, generator=gen)).bfloat16().unbind(0)) if norm else (None, None)
    ang = torch.outer(torch.arange(160.0), 1e4 ** (-torch.arange(0, D, 2) / D))
    cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
    offset = int32([0, 30, 41][:B])
    pos = offset[:, None].long() + torch.arange(S)
    pos[0, 0] = 10 ** 9                                     # behind the tables: their last row
    args = (1e-6, 1e-5, pos, cos, sin)
    total = torch.zeros(B, dtype=torch.int32)
    qc = kv4.kv4_qkv_prep(wide[..., :-8], qw, kw, *args, cpu, offset, total, table, Hq)
    dev = [x.cuda() if isinstance(x, torch.Tensor) else x for x in args]
    total_g = torch.zeros(B, dtype=torch.int32, device="cuda")
    qg = kv4.kv4_qkv_prep(wide.cuda()[..., :-8], *(w if w is None else w.cuda() for w in (qw, kw)), *dev, gpu, offset.cuda(), total_g,
                          table.cuda(), Hq)
    torch.cuda.synchronize()
    assert torch.equal(total, total_g.cpu()) and total.tolist() == (offset + S).tolist()
    _same(cpu, gpu)
    # Q is computed in 32 bits here and in 64 there: the norm's rounding may fall the other way, a whole step (2^-7) of either
    # member of a rotated pair, and the last rounding another one; a rounding is that near to its border a few times in 10^5
    a, b = qc.float(), qg.float().cpu()
    pair = (a.chunk(2, -1)[0].abs() + a.chunk(2, -1)[1].abs()).repeat(1, 1, 1, 2) * 2 ** 0.5
    assert ((a - b).abs() <= 2.0 ** -7 * (a.abs() + pair)).all()
    assert (a == b).float().mean() > 0.999


def _fp16_keys(q, keys, scale):
    """What rounding K to fp16 (2^-11 of each value at most) can do to a score of q [B, S, Hq, D] over lists of [L, Hkv, D]."""
    worst = 0.0
    for x, k in zip(q.double().abs().cpu(), keys):
        k = k.abs().nan_to_num(0.0).transpose(0, 1)                            # [Hkv, L, D]
        x = x.transpose(0, 1).reshape(k.shape[0], -1, k.shape[2])               # [Hkv, heads and tokens, D]
        if k.numel():
            worst = max(worst, float((x @ k.transpose(1, 2)).max()))
    return 2.0 ** -11 * abs(scale) * worst


def _check(got, want, lse_got, lse, dtype, v_max, cache_dtype=torch.bfloat16, scores=1.0, rounded=None):
    """``rounded``: K and V are fp16 numbers on the way, which moves a score by that at most: an LSE by as much, an output,
    sum of p_i e_i (v_i - out), by 2 v_max as much, and by V's own 2^-11."""
    assert torch.equal(got.isnan().cpu(), want.isnan())
    off = (got.double().cpu() - want).abs()
    extra = 0.0 if rounded is None else 2 * rounded + 2.0 ** -11
    assert (off <= oracle.bounds(want, dtype, v_max, cache_dtype, scores) + extra * v_max).all(), off.max()
    if lse_got is not None:
        assert torch.equal(lse_got.cpu() == -math.inf, lse == -math.inf)
        fine = lse != -math.inf
        # a score's 8e-5 six times over, and the half step of an fp32 LSE that is not near 1
        assert ((lse_got.double().cpu() - lse)[fine].abs() <= scores * 5e-4 + (rounded or 0.0) + 2.0 ** -24 * lse[fine].abs()).all()


ATTEND = [
    # lens, S, Hq, Hkv, D, group, page, splits
    ([37, 0, 1, 2, 33], 1, 8, 2, 128, 64, 16, -1),
    ([300, 129], 1, 40, 8, 64, 32, 16, 3),                  # five heads to a KV head
    ([1000], 1, 32, 2, 128, 128, 64, 4),                    # sixteen
    ([700, 31, 512], 1, 18, 1, 128, 32, 48, 2),             # eighteen: a second column block, ragged
    ([513, 64, 5], 5, 8, 2, 256, 64, 32, 3),                # several tokens; a sequence shorter than them is no sequence, 5 is
    ([260], 1, 4, 4, 256, 128, 16, -1),                     # no sharing
    ([95, 200], 7, 12, 4, 256, 32, 16, 1),
    ([1025], 9, 4, 2, 64, 64, 1040, 5),                     # one page of odd size for the sequence
    ([15, 16, 17], 17, 4, 2, 128, 64, 16, 1),               # more queries than tokens: the first rows see nothing
    ([4096], 1, 8, 1, 128, 64, 64, 32),
    ([100] * 20, 1, 4, 1, 64, 32, 16, -1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,S,Hq,H,D,group,page,splits", ATTEND)
def test_attention_against_the_definition(lens, S, Hq, H, D, group, page, splits, dtype):
    gen = _gen(sum(lens) + S)
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, dtype, "cuda", room=max(lens) + 40)
    q = oracle.rows(gen, len(lens), S, Hq, D, dtype=dtype, device="cuda")
    keys, values = [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs]
    v_max = max(float(x.abs().max()) if x.numel() else 0.0 for x in values)
    n = int32(lens, "cuda")
    for causal in (True, False) if S > 1 else (True,):
        want, lse = oracle.attention(q, keys, values, D ** -0.5, causal=causal)
        out = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal)
        full = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal, return_lse=True)
        torch.cuda.synchronize()
        assert out.dtype == dtype and full.dtype == torch.float32
        _check(out, want, None, None, dtype, v_max, dtype)
        _check(full[..., :D], want, full[..., D], lse, torch.float32, v_max, dtype)
        again = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal)
        assert torch.equal(out, again)
    if S == 1:
        assert torch.equal(kv4.gqa_fwd_kv4(q[:, 0], cache, n, table, kv_split=splits), out[:, 0])


@pytest.mark.parametrize("soft_cap", [0.0, 15.0])
def test_large_scores_and_peaked_rows(soft_cap):
    """Scores far apart (the running maximum moves in every block) and one token that takes nearly all the weight."""
    gen = _gen(21)
    H, Hq, D, group, page, L = 2, 8, 128, 64, 16, 900
    cache, table, ks, vs = oracle.filled(gen, [L], H, D, group, page, torch.bfloat16, "cuda")
    q = oracle.rows(gen, 1, 1, Hq, D, device="cuda") * 2
    order = torch.argsort((ks[0][:, 0].float() @ q[0, 0, 0].float()))       # ascending scores for the first head
    k, v = ks[0][order][None].contiguous(), vs[0][order][None].contiguous()
    kv4.kv4_append(k, v, cache, int32([0], "cuda"), table)
    keys, values = [oracle.held(k[0], group)], [oracle.held(v[0], group)]
    for splits in (1, 4):
        want, lse = oracle.attention(q, keys, values, 0.5, soft_cap)
        got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, scale=0.5, soft_cap=soft_cap, kv_split=splits)
        torch.cuda.synchronize()
        # scores: a scale of 0.5 instead of 128^-0.5 is 5.7 times as much, q twice as wide 2 more
        _check(got, want, None, None, torch.bfloat16, float(values[0].abs().max()), scores=12.0)


# query heads and KV heads, new tokens, head_dim, group: the forms with tokens across the lanes (at most 4, at most 8 columns),
# one block of sixteen columns, two blocks, heads of 256
SHAPES = [(3, 1, 1, 128, 64), (8, 1, 1, 128, 32), (4, 2, 3, 64, 32), (12, 1, 1, 128, 128), (20, 1, 2, 64, 64), (4, 1, 9, 128, 64),
          (4, 1, 1, 256, 64), (4, 1, 3, 256, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,H,S,D,group", SHAPES)
def test_values_far_from_one(Hq, H, S, D, group, dtype):
    """Groups of V 2^22 apart, tokens of one group 2^14 apart, large ones first and last: each channel to its own size."""
    gen = _gen(41)
    L, page = 700, 16
    cache, table, ks, _ = oracle.filled(gen, [L], H, D, group, page, dtype, "cuda")
    size = torch.ones(L, 1, D)
    size[:, :, :group] = 2.0 ** 10
    if D > group:
        size[:, :, -group:] = 2.0 ** -12
    size[100:400, :, :group] = 2.0 ** -4
    size[256:300] *= 2.0 ** -2
    v = (oracle.rows(gen, L, H, D).float() * size).to(dtype).cuda()
    kv4.kv4_append(ks[0][None].contiguous(), v[None], cache, int32([0], "cuda"), table)
    q = oracle.rows(gen, 1, S, Hq, D, dtype=dtype, device="cuda")
    keys, values = [oracle.held(ks[0], group)], [oracle.held(v, group)]
    # one size per group of channels; 2^-25 of fp16's last bits, the P of a weight at its reference 2^6 at least
    v_max = values[0].abs().amax((0, 1)).unflatten(0, (-1, group)).amax(1).repeat_interleave(group)
    for splits in (1, 3):
        want, lse = oracle.attention(q, keys, values, D ** -0.5)
        got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, kv_split=splits, return_lse=True)
        torch.cuda.synchronize()
        _check(got[..., :D], want, got[..., D], lse, torch.float32, v_max, dtype)


@pytest.fixture
def chunks(monkeypatch):
    """Many columns go to the kernel for them however short the sequences are."""
    monkeypatch.setattr(kv4, "takes_chunks", lambda *a: a[2] >= 32 and a[5] == 0)


CHUNKS = [
    # lens, S, Hq, Hkv, D, group, page, splits
    ([64], 64, 1, 1, 128, 64, 16, 1),                       # a prompt of its own
    ([300, 70, 0, 129], 70, 4, 2, 128, 64, 16, 1),          # ragged; one shorter than its queries, one that is not there
    ([777], 40, 14, 2, 128, 32, 48, 3),                     # a second block of columns that is nearly empty
    ([1500], 300, 2, 2, 128, 128, 64, 2),
    ([513, 1], 96, 4, 4, 64, 32, 16, 2),
    ([400], 260, 8, 4, 64, 64, 1040, 1),
    ([333, 900], 33, 8, 2, 256, 32, 16, 2),
    ([450], 200, 2, 1, 256, 64, 32, 1),
    ([2000], 65, 1, 1, 256, 128, 16, 5),
    ([90], 80, 4, 1, 128, 64, 16, 40),                      # more splits than there is to split
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,S,Hq,H,D,group,page,splits", CHUNKS)
def test_many_columns_against_the_definition(lens, S, Hq, H, D, group, page, splits, dtype, chunks):
    gen = _gen(sum(lens) + S)
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, dtype, "cuda", room=max(lens) + 40)
    q = oracle.rows(gen, len(lens), S, Hq, D, dtype=dtype, device="cuda")
    keys, values = [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs]
    v_max = max(float(x.abs().max()) if x.numel() else 0.0 for x in values)
    n = int32(lens, "cuda")
    for causal in (True, False):
        want, lse = oracle.attention(q, keys, values, D ** -0.5, causal=causal)
        out = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal)
        full = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal, return_lse=True)
        torch.cuda.synchronize()
        e = _fp16_keys(q, keys, D ** -0.5)
        _check(out, want, None, None, dtype, v_max, rounded=e)
        _check(full[..., :D], want, full[..., D], lse, torch.float32, v_max, rounded=e)
        assert torch.equal(out, kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=splits, causal=causal))


@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("splits", [1, 3])
def test_chunks_with_blocks_that_fp16_does_not_reach(D, group, splits, chunks):
    """A few tokens with a large K, with tiny K, with tiny and large V, a NaN and a page that is none: these blocks go the other
    way, the rest does not, and the columns of both are right."""
    gen = _gen(45)
    S, H, Hq, page = 100, 2, 4, 16
    for what in range(7):
        cache, table, ks, vs = oracle.filled(gen, [600], H, D, group, page, torch.bfloat16, "cuda")
        k, v, there = ks[0].clone(), vs[0].clone(), torch.ones(600, dtype=torch.bool)
        if what == 0:
            k[37, 1, 3] = 2.0 ** 16
        elif what == 1:
            k[64:128] *= 2.0 ** -17
        elif what == 2:
            v[192:256] *= 2.0 ** -18
        elif what == 6:                     # (small, but not for the other kernel)
            k[64:128] *= 2.0 ** -10
            v[192:256] *= 2.0 ** -11
        elif what == 3:
            v[590:] *= 2.0 ** 17
        elif what == 4:
            k[555, 0, 0] = math.nan
        kv4.kv4_append(k[None], v[None], cache, int32([0], "cuda"), table)
        if what == 5:
            table[0, 20] = -1
            there[320:336] = False
        q = oracle.rows(gen, 1, S, Hq, D, device="cuda")
        if what == 0:
            q *= 2.0 ** -10                 # (scores of a few nats)
        keys, values = [oracle.held(k, group)], [oracle.held(v, group)]
        want, lse = oracle.attention(q, keys, values, D ** -0.5, there=[there])
        got = kv4.gqa_fwd_kv4(q, cache, int32([600], "cuda"), table, kv_split=splits, return_lse=True)
        torch.cuda.synchronize()
        if what == 4:                       # a query that sees the NaN, of either of its KV head's, is NaN
            assert got[0, 55:, :2].isnan().all() and got[0, :55].isfinite().all() and got[0, :, 2:].isfinite().all()
            want[0, 55:, :2], lse[0, 55:, :2] = 0.0, 0.0
            got[0, 55:, :2] = 0.0
        _check(got[..., :D], want, got[..., D], lse, torch.float32, float(values[0].nan_to_num(0.0).abs().max()),
               rounded=_fp16_keys(q, keys, D ** -0.5))


@pytest.mark.parametrize("scale", [-0.11, 0.0, 0.3])
def test_chunks_at_other_scales_strides_and_streams(scale, chunks):
    gen = _gen(46)
    lens, S, H, Hq, D, group, page = [333, 70], 40, 2, 8, 128, 64, 32
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda")
    q = oracle.rows(gen, 2, S + 3, Hq + 2, D, device="cuda")[:, 2:S + 2, 1:Hq + 1]
    keys, values = [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs]
    want, lse = oracle.attention(q, keys, values, scale)
    n = int32(lens, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = kv4.gqa_fwd_kv4(q, cache, n, table, scale=scale, return_lse=True, kv_split=2)
    here = kv4.gqa_fwd_kv4(q, cache, n, table, scale=scale, return_lse=True, kv_split=2)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(here, there)
    _check(here[..., :D], want, here[..., D], lse, torch.float32, max(float(x.abs().max()) for x in values),
           scores=max(1.0, abs(scale) * D ** 0.5), rounded=_fp16_keys(q, keys, scale))


def test_chunks_replay_from_a_graph(chunks):
    """A flagged block and a plain one, replayed with other queries and another cache behind the same addresses."""
    gen = _gen(47)
    lens, S, H, Hq, D, group, page = [500, 300], 80, 1, 4, 128, 32, 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda")
    n, q = int32(lens, "cuda"), oracle.rows(gen, 2, S, Hq, D, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        q.copy_(oracle.rows(gen, 2, S, Hq, D, device="cuda"))
        k = oracle.rows(gen, 2, 64, H, D, device="cuda")
        if i % 2:
            k[0] *= 2.0 ** 17
        kv4.kv4_append(k, k, cache, int32([100 * (i % 3), 64 * (i % 4)], "cuda"), table)
        graph.replay()
        torch.cuda.synchronize()
        eager = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_large_chunks_and_small_ones_agree(monkeypatch):
    """The same call by either kernel, at a size where it is the other one's: each is within its bounds of the definition."""
    gen = _gen(48)
    S, H, Hq, D, group, page, L = 70, 8, 32, 128, 64, 64, 16000
    cache, table, ks, vs = oracle.filled(gen, [L], H, D, group, page, torch.bfloat16, "cuda")
    q, n = oracle.rows(gen, 1, S, Hq, D, device="cuda"), int32([L], "cuda")
    assert kv4.takes_chunks(1, H, S * Hq // H, D, table.shape[1] * page)
    one = kv4.gqa_fwd_kv4(q, cache, n, table, return_lse=True)
    monkeypatch.setattr(kv4, "takes_chunks", lambda *a: False)
    other = kv4.gqa_fwd_kv4(q, cache, n, table, return_lse=True)
    torch.cuda.synchronize()
    v_max = float(vs[0].abs().max())
    _check(one[..., :D], other[..., :D].double().cpu(), one[..., D], other[..., D].double().cpu(), torch.float32, v_max, scores=2.0,
           rounded=_fp16_keys(q, [oracle.held(ks[0], group)], D ** -0.5))


@pytest.mark.parametrize("scale,soft_cap", [(-0.11, 0.0), (0.3, 7.0), (-0.3, 7.0), (0.0, 0.0), (0.0, 5.0), (0.1, 1e-30)])
@pytest.mark.parametrize("Hq,H,S,D,group", SHAPES)
def test_scales_and_caps(Hq, H, S, D, group, scale, soft_cap):
    gen = _gen(42)
    lens, page = [333, 40], 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda")
    q = oracle.rows(gen, 2, S, Hq, D, device="cuda")
    keys, values = [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs]
    v_max = max(float(x.abs().max()) for x in values)
    want, lse = oracle.attention(q, keys, values, scale, soft_cap)
    for splits in (1, 2):
        got = kv4.gqa_fwd_kv4(q, cache, int32(lens, "cuda"), table, scale=scale, soft_cap=soft_cap, kv_split=splits, return_lse=True)
        torch.cuda.synchronize()
        _check(got[..., :D], want, got[..., D], lse, torch.float32, v_max, scores=max(1.0, abs(scale) * D ** 0.5))


@pytest.mark.parametrize("Hq,S,D", [(4, 1, 64), (16, 1, 64), (20, 1, 64), (4, 1, 256)])
def test_one_heavy_token_and_a_long_tail_of_light_ones(Hq, S, D):
    """20001 tokens, one with the weight of 2^14 others: the light ones are most of the sum, far below the reference."""
    gen = _gen(43)
    L, group, page = 20001, 32, 64
    table, pages = oracle.table_for(1, L, page, gen, device="cuda")
    cache = kv4.Int4KVCache.alloc(pages, page, 1, D, group=group, device="cuda")
    q = torch.ones(1, S, Hq, D, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(1, L, 1, D, dtype=torch.bfloat16, device="cuda")
    k[0, 17] = 14 * math.log(2) / D
    v = oracle.rows(gen, 1, L, 1, D, device="cuda")
    kv4.kv4_append(k, v, cache, int32([0], "cuda"), table)
    keys, values = [oracle.held(k[0], group)], [oracle.held(v[0], group)]
    want, lse = oracle.attention(q, keys, values, 1.0)
    for splits in (1, 7):
        got = kv4.gqa_fwd_kv4(q, cache, int32([L], "cuda"), table, scale=1.0, kv_split=splits, return_lse=True)
        torch.cuda.synchronize()
        # light weights are 2^-14 of the heaviest, 2^-8 at least: whole fp16 numbers (scales down to 2^-6 of the widest)
        _check(got[..., :D], want, got[..., D], lse, torch.float32, float(values[0].abs().max()))


@pytest.mark.parametrize("batch,splits", [(70, 2), (3, 300), (1, 65535), (66, -1)])
def test_batches_and_splits_of_unusual_counts(batch, splits):
    gen = _gen(44)
    lens = [(37 * b) % 301 for b in range(batch)]
    lens[0] = 513
    H, Hq, D, group, page = 2, 6, 64, 64, 32
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda")
    q = oracle.rows(gen, batch, 1, Hq, D, device="cuda")
    keys, values = [oracle.held(x, group) for x in ks], [oracle.held(x, group) for x in vs]
    want, lse = oracle.attention(q, keys, values, D ** -0.5)
    got = kv4.gqa_fwd_kv4(q, cache, int32(lens, "cuda"), table, kv_split=splits, return_lse=True)
    torch.cuda.synchronize()
    _check(got[..., :D], want, got[..., D], lse, torch.float32, max(float(x.abs().max()) for x in values if x.numel()))


def test_garbage_outside_of_the_sequences_is_not_read_into_the_result():
    gen = _gen(22)
    lens, H, D, group, page = [21, 50], 2, 128, 32, 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda", room=96)
    q = oracle.rows(gen, 2, 2, 4, D, device="cuda")
    n = int32(lens, "cuda")
    clean = kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2)
    there = torch.zeros(cache.num_pages, page, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        for t in range(L):
            there[table[b, t // page].long(), t % page] = True
    for p in (cache.k_params, cache.v_params):              # every token that is in no sequence: NaN and infinity
        x = p.permute(0, 3, 1, 2, 4)
        x[~there] = torch.tensor([math.nan, math.inf], dtype=p.dtype, device="cuda")
    cache.k_codes.transpose(1, 2)[~there] = 255
    far = table.clone()
    far[0, 2:], far[1, 4:] = -1, 10 ** 6                    # and no pages behind the lengths
    dirty = kv4.gqa_fwd_kv4(q, cache, n, far, kv_split=2)
    torch.cuda.synchronize()
    assert torch.equal(clean, dirty)


def test_masked_nan_reaches_the_query_that_sees_it_alone():
    gen = _gen(23)
    H, D, group, page = 1, 128, 64, 16
    for splits in (1, 2):
        cache, table, _, _ = oracle.filled(gen, [300], H, D, group, page, torch.bfloat16, "cuda")
        k = torch.full((1, 1, H, D), math.nan, dtype=torch.bfloat16, device="cuda")
        kv4.kv4_append(k, k, cache, int32([299], "cuda"), table)
        out = kv4.gqa_fwd_kv4(oracle.rows(gen, 1, 3, 2, D, device="cuda"), cache, int32([300], "cuda"), table, kv_split=splits)
        torch.cuda.synchronize()
        assert out[0, :2].isfinite().all() and out[0, 2].isnan().all()


def test_a_table_without_pages_is_empty_sequences():
    from test_kv4_cpu import _no_pages

    _no_pages("cuda")


def test_bad_pages_inside_a_sequence():
    gen = _gen(24)
    H, Hq, D, group, page = 2, 4, 64, 32, 16
    cache, table, ks, vs = oracle.filled(gen, [90], H, D, group, page, torch.float16, "cuda")
    bad = table.clone()
    bad[0, 1], bad[0, 4] = -1, cache.num_pages
    there = torch.ones(90, dtype=torch.bool)
    there[16:32] = there[64:80] = False
    q = oracle.rows(gen, 1, 3, Hq, D, dtype=torch.float16, device="cuda")
    values = [oracle.held(vs[0], group)]
    want, lse = oracle.attention(q, [oracle.held(ks[0], group)], values, D ** -0.5, there=[there])
    got = kv4.gqa_fwd_kv4(q, cache, int32([90], "cuda"), bad, return_lse=True, kv_split=1)
    torch.cuda.synchronize()
    _check(got[..., :D], want, got[..., D], lse, torch.float32, float(values[0].abs().max()), torch.float16)
    over = kv4.gqa_fwd_kv4(q, cache, int32([10 ** 6], "cuda"), table)       # a length beyond the table is the table's
    assert torch.equal(over, kv4.gqa_fwd_kv4(q, cache, int32([96], "cuda"), table))


def test_parts_of_a_sequence_on_two_ranks_merge():
    gen = _gen(25)
    lens, H, Hq, D, group, page = [[200, 64], [77, 0]], 2, 8, 128, 64, 16
    q = oracle.rows(gen, 2, Hq, D, device="cuda")
    parts, ks, vs = [], [], []
    for n in lens:
        cache, table, k, v = oracle.filled(gen, n, H, D, group, page, torch.bfloat16, "cuda")
        parts.append(kv4.gqa_fwd_kv4(q, cache, int32(n, "cuda"), table, return_lse=True))
        ks.append(k), vs.append(v)
    out = flash_decode.gqa_fwd_batch_decode_inter_rank_combine(torch.stack(parts), int32(lens, "cuda"))
    whole = [torch.cat([oracle.held(x[b], group) for x in y]) for y in (ks, vs) for b in range(2)]
    want, _ = oracle.attention(q[:, None], whole[:2], whole[2:], D ** -0.5)
    torch.cuda.synchronize()
    _check(out, want[:, 0], None, None, torch.bfloat16, max(float(x.abs().max()) for x in whole[2:]))


def test_strided_queries_and_another_stream():
    gen = _gen(26)
    lens, H, Hq, D, group, page = [70, 300], 2, 8, 128, 64, 16
    cache, table, ks, vs = oracle.filled(gen, lens, H, D, group, page, torch.bfloat16, "cuda")
    n = int32(lens, "cuda")
    wide = oracle.rows(gen, 2, 3, Hq + 4, D, device="cuda")
    q = wide[:, :, 2:2 + Hq]
    want = kv4.gqa_fwd_kv4(q.contiguous(), cache, n, table, kv_split=2)
    assert torch.equal(kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2), want)
    unaligned = torch.empty(2 * 3 * Hq * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 3, Hq, D)
    unaligned.copy_(q)
    assert torch.equal(kv4.gqa_fwd_kv4(unaligned, cache, n, table, kv_split=2), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2) for _ in range(3)]
    here = [kv4.gqa_fwd_kv4(q, cache, n, table, kv_split=2) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + here)


def test_decode_steps_replay_from_two_graphs():
    """append + attention as a captured step; two graphs that share the cache replay in turn and equal the eager steps."""
    gen = _gen(27)
    B, H, Hq, D, group, page = 2, 2, 8, 128, 64, 16
    start = [100, 37]
    cache, table, _, _ = oracle.filled(gen, start, H, D, group, page, torch.bfloat16, "cuda", room=128)
    twin = kv4.Int4KVCache(*(t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params)))
    steps = 6
    k, v = (oracle.rows(gen, steps, B, 1, H, D, device="cuda") for _ in range(2))
    q = oracle.rows(gen, steps, B, 1, Hq, D, device="cuda")
    bufs = [k[0].clone(), v[0].clone(), q[0].clone()]
    offset, total = int32(start, "cuda"), int32(start, "cuda")

    def step(c, kk, vv, qq, splits):
        kv4.kv4_append(kk, vv, c, offset, table)
        torch.add(offset, 1, out=total)
        return kv4.gqa_fwd_kv4(qq, c, total, table, kv_split=splits)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(cache, *bufs, 2)
        for splits in (1, 3):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(cache, *bufs, splits)
            graphs.append((g, out, splits))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(steps):
        g, out, splits = graphs[i % 2]
        for b, x in zip(bufs, (k[i], v[i], q[i])):
            b.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        eager = step(twin, k[i], v[i], q[i], splits)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        offset += 1
    _same(cache, twin)


def test_pages_far_beyond_32_bit_offsets():
    """Pages at the end of a cache of more than 4 GiB of codes."""
    H, D, group, page = 8, 256, 128, 64
    pages = (9 << 29) // (H * page * D // 2)                # 4.5 GiB of K codes
    cache = kv4.Int4KVCache(torch.empty(pages, H, page, D // 2, dtype=torch.uint8, device="cuda"),
                            torch.empty(pages, H, page // 4, 2 * D, dtype=torch.uint8, device="cuda"),
                            *(torch.empty(pages, H, D // group, page, 2, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    gen = _gen(28)
    table = int32([[pages - 1, 3]], "cuda")
    k, v = oracle.rows(gen, 1, 100, H, D, device="cuda"), oracle.rows(gen, 1, 100, H, D, device="cuda")
    kv4.kv4_append(k, v, cache, int32([0], "cuda"), table)
    got = kv4.kv4_read(cache, table, int32([0, 100], "cuda"), 100)
    q = oracle.rows(gen, 1, 1, H, D, device="cuda")
    out = kv4.gqa_fwd_kv4(q, cache, int32([100], "cuda"), table)
    torch.cuda.synchronize()
    kh, vh = oracle.held(k[0], group), oracle.held(v[0], group)
    for g, w in zip(got, (kh, vh)):
        assert ((g.double().cpu() - w).abs() <= (2.0 ** -8 + 2.0 ** -23) * w.abs() + 2.0 ** -26).all()
    want, _ = oracle.attention(q, [kh], [vh], D ** -0.5)
    _check(out, want, None, None, torch.bfloat16, float(vh.abs().max()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_layer_over_a_4bit_cache(dtype):
    from kv4_layer_checks import attention_layer

    attention_layer("cuda", dtype)


@pytest.mark.parametrize("backend", ["torch", "triton_dist_AR"])
def test_engine_decodes_from_a_graph_over_a_4bit_cache(backend, monkeypatch):
    monkeypatch.setenv("RANDOM_PARAMS", "1")
    monkeypatch.setenv("TDIST_NO_HF_CONFIG", "1")
    from triton_distributed_gh_amd.models import Engine, KV4_Cache, ModelConfig
    from triton_distributed_gh_amd.utils.testing import VirtualCluster

    config = ModelConfig(model_name="tdist/tiny-dense-d128", max_length=128, dtype=torch.bfloat16, rank=0, world_size=1)
    vc = VirtualCluster(1, heap_bytes=1 << 26)
    try:
        eng = Engine(config, env=vc.envs[0], kv_cache_bits=4)
        eng.backend = backend
        ids = torch.randint(0, 1000, (3, 37), generator=_gen(33))
        replayed = eng.serve(ids, gen_len=12)
        assert isinstance(eng.kv_cache, KV4_Cache)
        eng.no_graph = True
        assert torch.equal(replayed, eng.serve(ids, gen_len=12))
    finally:
        vc.close()


def test_sequence_parallel_decode_over_4bit_shards():
    from triton_distributed_gh_amd.layers import SpGQAFlashDecodeAttention
    from triton_distributed_gh_amd.utils.testing import VirtualCluster

    gen = _gen(34)
    w, Hq, H, D, group, page = 2, 8, 2, 128, 64, 16
    lens = [[70, 16], [33, 0]]
    q = oracle.rows(gen, 2, Hq, D, device="cuda")
    shards = [oracle.filled(gen, n, H, D, group, page, torch.bfloat16, "cuda") for n in lens]
    whole = [torch.cat([oracle.held(s[i][b], group) for s in shards]) for i in (2, 3) for b in range(2)]
    want, _ = oracle.attention(q[:, None], whole[:2], whole[2:], D ** -0.5)
    vc = VirtualCluster(w, heap_bytes=1 << 26)
    try:
        layers = vc.collective(lambda r, env: SpGQAFlashDecodeAttention(r, 0, w, 1, Hq, H, D, D, page_size=page, scale=D ** -0.5,
                                                                        max_allowed_batch=2, env=env))
        n = int32(lens, "cuda")
        torch.cuda.synchronize()
        for _ in range(3):
            for out in vc.run(lambda r, env: layers[r](q, shards[r][0], None, n, shards[r][1])):
                torch.cuda.synchronize()
                _check(out, want[:, 0], None, None, torch.bfloat16, max(float(x.abs().max()) for x in whole[2:]))
    finally:
        vc.close()
