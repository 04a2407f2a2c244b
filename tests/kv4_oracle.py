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


def bounds(ref: torch.Tensor, dtype, v_max: float) -> torch.Tensor:
    """How far an output may be from its 64-bit value: half a step of its type (eps / 2, relative), and what 32-bit scores and
    a 16-significant-bit P leave.  A score is a chain of D / 32 MFMA accumulations and a few fp32 operations on magnitudes of
    at most 31 sum|q| (about 31 * 0.8 * 256 = 6350 codes for unit q of 256 channels): at most 8 * 2^-24 * 6350 = 3.1e-3 codes,
    times a scale of at most 1 and 1 / sqrt(256) = 2e-4 of a nat at the very worst.  An error e of every weight moves the
    output by at most 2 e max|v| = 4e-4 max|v| < 2^-11 max|v|; P's 2^-17 and the exponentials' 2^-22 are small beside it."""
    half = torch.finfo(dtype).eps / 2
    return half * ref.abs() + 2.0 ** -11 * v_max
