"""What the 4-bit KV cache has to hold and answer, from its definition in 64 bits and one row at a time - nothing here knows
the packed layout.  Also the builders that the CPU and the GPU tests share."""
import math

import torch

from triton_distributed_gh_amd.ops import kv4


def held(x: torch.Tensor, group: int) -> torch.Tensor:
    """fp64 values that rows x [..., D] (16-bit) stand for once they are cached.

    fl32 of an fp64 difference / quotient of such numbers is the IEEE fp32 one (53 >= 2 * 24 + 2 bits: the double rounding
    is innocuous), so the border between two codes is the definition's own."""
    v = x.double().cpu().unflatten(-1, (-1, group))
    low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    span = (high - low).float()
    scale = torch.where(span.isfinite(), (span.double() / 15).float(), torch.nan).to(x.dtype).double()
    code = ((v - low).float().double() / scale).float().round().clamp(0, 15)
    code = torch.where(scale > 0, code, 0.0)
    return (code.double() * scale + low).flatten(-2)


def attention(q, keys, values, scale, soft_cap=0.0, causal=True, there=None):
    """fp64 (out [B, S, Hq, D], lse [B, S, Hq]) of q [B, S, Hq, D] over lists of [L, Hkv, D] fp64 rows; there[b] [L]: tokens
    that have a page."""
    q = q.double().cpu()
    B, S, Hq, D = q.shape
    out, lse = torch.zeros(B, S, Hq, D, dtype=torch.float64), torch.full((B, S, Hq), -math.inf, dtype=torch.float64)
    for b in range(B):
        k, v = keys[b].double().cpu(), values[b].double().cpu()
        L = k.shape[0]
        for s in range(S):
            see = torch.arange(L) < (L - S + s + 1 if causal else L)
            if there is not None:
                see &= there[b][:L].cpu()
            if not see.any():
                continue
            ks, vs = k[see], v[see]
            for h in range(Hq):
                kh = h // (Hq // k.shape[1])
                x = ks[:, kh] @ q[b, s, h] * scale
                if soft_cap > 0:
                    x = soft_cap * torch.tanh(x / soft_cap)
                out[b, s, h] = torch.softmax(x, 0) @ vs[:, kh]
                lse[b, s, h] = torch.logsumexp(x, 0)
    return out, lse


def table_for(batch, tokens, page, gen, spare=3, device="cpu"):
    """A shuffled block table with room for `tokens` per sequence, and the number of pages it indexes."""
    each = -(-tokens // page)
    pages = batch * each + spare
    table = torch.randperm(pages, generator=gen)[: batch * each].view(batch, each).int()
    return table.to(device), pages


def rows(gen, *shape, dtype=torch.bfloat16, device="cpu"):
    """Rows whose channels have means and widths of their own."""
    D = shape[-1]
    wide = torch.exp(0.4 * torch.randn(D, generator=gen))
    return ((torch.randn(*shape, generator=gen) * wide + 0.4 * torch.randn(D, generator=gen))).to(dtype).to(device)


def int32(values, device="cpu"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def filled(gen, lens, kv_heads, D, group, page, dtype=torch.bfloat16, device="cpu", room=None):
    """(cache, table, raw K list, raw V list): sequences of the given lengths in a cache of shuffled pages."""
    B, longest = len(lens), max(max(lens), 1)
    table, pages = table_for(B, room or longest, page, gen, device=device)
    cache = kv4.Int4KVCache.alloc(pages, page, kv_heads, D, group=group, dtype=dtype, device=device)
    k, v = rows(gen, B, longest, kv_heads, D, dtype=dtype, device=device), rows(gen, B, longest, kv_heads, D, dtype=dtype, device=device)
    kv4.kv4_append(k, v, cache, int32([0] * B, device), table, new_lens=int32(lens, device))
    return cache, table, [k[b, :n] for b, n in enumerate(lens)], [v[b, :n] for b, n in enumerate(lens)]


def bounds(ref: torch.Tensor, dtype, v_max, cache_dtype=torch.bfloat16, scores: float = 1.0) -> torch.Tensor:
    """How far an output may be from its 64-bit value: half a step of its type (eps / 2, relative), and what the scores and the
    weights leave.  ``v_max``: the largest |V|, a number or one per channel; ``scores``: scale times size of q, over 1 / sqrt(D).

    Weights.  P * scale is one fp16 number where the cache is bf16: half a step, 2^-11 of the weight, times a code's 15 * scale,
    a group's range of at most 2 v_max: 2^-10 v_max (a remainder in a second number for fp16 caches: 2^-21).

    Scores.  codes are summed with 1024 added to half of them, in fp32: the accumulator passes through about 1024 times the
    signed sum of a group's even channels of q, for `rows` 1024 * sqrt(64) * 1.1 = 9e3 in groups of 128, and is rounded
    some 8 times in each of 4 products: 2^-24 / sqrt(3) * 9e3 * sqrt(32) = 1.8e-3 codes, times a scale of 0.5 and 1 / sqrt(128)
    that is 8e-5 of a nat, independent from token to token (one standard deviation).  Errors e of two weights p and 1 - p move
    the output by p (1 - p) (e1 - e2) (v1 - v2) <= 1 / 4 * sqrt(2) * 8e-5 * 2 v_max = 5.7e-5 v_max, more tokens average it:
    2^-11 v_max are more than eight deviations."""
    half = torch.finfo(dtype).eps / 2
    weights = 2.0 ** -10 if cache_dtype == torch.bfloat16 else 2.0 ** -21
    return half * ref.abs() + (scores * 2.0 ** -11 + weights) * v_max
