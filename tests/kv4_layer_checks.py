"""Checks of the layers over a 4-bit cache that run on either backend."""
from types import SimpleNamespace

import torch

import kv4_oracle as oracle
from triton_distributed_gh_amd.layers.tp_attn import TP_Attn, _set_cos_sin_cache
from triton_distributed_gh_amd.models import KV4_Cache, KV_Cache
from triton_distributed_gh_amd.ops import kv4


def _to_cpu(c):
    return kv4.Int4KVCache(*(t.cpu() for t in (c.k_codes, c.v_codes, c.k_params, c.v_params)))


def attention_layer(device, dtype):
    """A prompt and decode steps through the attention layer: what the cache holds against the 16-bit cache's rows, what comes out
    against the definition over what the cache holds."""
    gen = torch.Generator().manual_seed(41)
    B, H, Hq, Hkv, D, group, room = 2, 256, 8, 2, 128, 32, 100
    lin = lambda o, i: SimpleNamespace(weight=(torch.randn(o, i, generator=gen) * i ** -0.5).to(dtype).to(device), bias=None)  # noqa: E731
    norm = lambda: SimpleNamespace(weight=(1 + 0.1 * torch.randn(D, generator=gen)).to(dtype).to(device), variance_epsilon=1e-6)  # noqa: E731
    attn = TP_Attn(rank=0, world_size=1)
    attn._device = lambda: torch.device(device)
    attn._init_parameters(SimpleNamespace(head_dim=D, q_proj=lin(Hq * D, H), k_proj=lin(Hkv * D, H), v_proj=lin(Hkv * D, H),
                                          o_proj=lin(H, Hq * D), q_norm=norm(), k_norm=norm()))
    cos_sin = _set_cos_sin_cache(1.0 / (1e4 ** (torch.arange(0, D, 2, device=device).float() / D)), 128)
    args = dict(num_layers=2, batch_size=B, max_length=room, kv_heads=Hkv, head_dim=D, dtype=dtype, world_size=1, device=device)
    four, wide = KV4_Cache(**args, page_size=16, group=group), KV_Cache(**args)
    twin = KV4_Cache(**args, page_size=16, group=group)
    for S in (37, 1, 1, 3, 1):
        qkv = oracle.rows(gen, B, S, (Hq + 2 * Hkv) * D, dtype=dtype, device=device)
        pos = four.get_kv_len()[:, None].long() + torch.arange(S, device=device)
        out = attn._attend(qkv, pos, cos_sin, four, 1)
        attn._attend(qkv, pos, cos_sin, wide, 1)
        queries = []
        seen, kv4.flash_attn_with_kv4cache = kv4.flash_attn_with_kv4cache, lambda q, *a: queries.append(q) or q
        try:
            attn._attend(qkv, pos, cos_sin, twin, 1)        # the same step, for its queries
        finally:
            kv4.flash_attn_with_kv4cache = seen
        for c in (four, wide, twin):
            c.inc_offset(S)
        total = int(four.get_kv_len()[0])
        if device != "cpu":
            torch.cuda.synchronize()
        cache, table = _to_cpu(four.kv4_layer(1)), four.block_table.cpu()
        at = torch.arange(total)
        rows = [kv4._load_reference(cache, torch.full_like(at, b), at, table)[1:] for b in range(B)]
        want, _ = oracle.attention(queries[0], [k for k, _ in rows], [v for _, v in rows], D ** -0.5)
        got = out.view(B, S, Hq, D).double().cpu()
        assert ((got - want).abs() <= oracle.bounds(want, dtype, float(rows[0][1].abs().max()), dtype)).all()
        # the 16-bit cache's rows, rounded by the definition: a norm that rounds the other way in 64 bits may move a code by one,
        # or a group's scale and low by a rounding (two of 16 bits, 16 steps of the scale's: less than a step together)
        for b in range(B):
            for held, raw in zip(rows[b], (wide.k_cache[1, b, :total], wide.v_cache[1, b, :total])):
                step = raw.double().cpu().unflatten(-1, (-1, group))
                step = ((step.amax(-1) - step.amin(-1)) / 15).repeat_interleave(group, -1)
                off = (held.double() - oracle.held(raw, group)).abs()
                assert (off <= 2 * step).all() and (off > 0.1 * step).double().mean() < 1e-2
    assert int(four.total_len[0]) == total
    assert (four.kv4_layer(0).k_codes == 0).all()
    k, v, cu = four.read(1)
    assert cu.tolist() == [0, total, 2 * total] and k.shape == v.shape == (2 * total, Hkv, D)
    four.clear()
    assert four.read(1)[0].shape[0] == 0
