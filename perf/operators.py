"""What is measured of the 4-bit KV cache: writing it, reading it back and attending over it.

The cache holds every row (one token, one KV head, ``head_dim`` channels) in groups of ``group`` channels.  A group has
a ``low`` (its smallest value) and a ``scale`` (a fifteenth of its range), both in the cache's 16-bit type, and one code
0 .. 15 for each channel: ``scale = round16((max - low) / 15)``, ``code = round((x - low) / scale)`` in 32 bits with ties
to even (0 where ``scale`` is 0), and the value it stands for is ``scale * code + low``.  Pages of ``page`` tokens belong to
sequences through a table.

Four operators, by a case's ``op``:

* ``write``: K / V rows of new tokens go into the cache; what comes out is the rows as the cache now holds them;
* ``project``: the same from a QKV projection, whose q and k heads get their RMSNorm and rotation on the way;
* ``read``: whole sequences of the cache as 16-bit rows, one sequence behind the other;
* ``attend``: grouped-query attention of the last ``new`` tokens of each sequence over its cached tokens, causal.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one new token of one sequence: what a single user's decode step writes in each layer; latency is all
        _case("write", "write_step", batch=1, new=1, length=21, kv_heads=8, dim=128, group=64, page=64),
        # prompts of different lengths, padded to the longest, behind prefixes that are cached already
        _case("write", "write_prompts", batch=8, new=4001, length=4500, kv_heads=8, dim=128, group=128, page=64, ragged=True),
        # one request's short odd prefix in half precision, heads of 64 channels: a prefix that is moved or checked
        _case("read", "read_prefix", batch=1, new=0, length=1037, kv_heads=5, dim=64, group=32, page=16, type="fp16"),
        # the caches of a batch, read back for a kernel that wants 16-bit rows
        _case("read", "read_batch", batch=16, new=0, length=8192, kv_heads=8, dim=128, group=64, page=128, ragged=True),
        # a decode step of sixteen sequences, from the projection on
        _case("project", "project_step", batch=16, new=1, length=2049, heads=32, kv_heads=8, dim=128, group=32, page=64, ragged=True),
        # two prompts from the projection on
        _case("project", "project_prompt", batch=2, new=1500, length=1500, heads=64, kv_heads=8, dim=128, group=32, page=64),
        # the first steps of a chat: next to nothing in the cache, so the launch itself is what counts
        _case("attend", "attend_short", batch=1, new=1, length=37, heads=32, kv_heads=8, dim=128, group=64, page=64),
        # one long document
        _case("attend", "attend_long", batch=1, new=1, length=131072, heads=32, kv_heads=8, dim=128, group=64, page=64),
        # a serving batch: the cache is what the step's time goes into
        _case("attend", "attend_batch", batch=64, new=1, length=4096, heads=32, kv_heads=8, dim=128, group=128, page=64),
        # lengths all over the place, one of them zero, five query heads to a KV head, half precision, small pages
        _case("attend", "attend_ragged", batch=13, new=1, length=2500, heads=40, kv_heads=8, dim=64, group=32, page=16, type="fp16", ragged=True),
        # drafted tokens checked together, wide heads
        _case("attend", "attend_drafts", batch=16, new=5, length=6151, heads=16, kv_heads=4, dim=256, group=64, page=32, ragged=True),
        # a chunk of a long prompt over what the chunks before it left in the cache
        _case("attend", "attend_chunk", batch=1, new=1024, length=16384, heads=32, kv_heads=8, dim=128, group=64, page=64),
    ]


def _case(op, name=None, *, batch, new, length, kv_heads, dim, group, page, heads=0, type="bf16", ragged=False):
    case = {"op": op, "batch": batch, "new": new, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "group": group, "page": page, "type": type, "ragged": ragged}
    return {"name": name, **case} if name else case


def draw(rng):
    def spread(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    op = rng.choice(("write", "read", "project", "attend", "attend", "attend"))
    dim = rng.choice((64, 128, 128, 256))
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 5, 8))
    page = rng.choice((16, 32, 48, 64, 128))
    type = rng.choice(("bf16", "fp16"))
    ragged = rng.random() < 0.6
    room = (8 << 20) // dim             # rows of all heads together: a fourth of the largest listed write
    batch = spread(1, 64)
    if op == "write":
        new = 1 if rng.random() < 0.3 else spread(1, max(1, min(4000, room // (batch * kv_heads))))
        length = new + spread(1, 500) - 1
    elif op == "project":
        type, group = "bf16", 32
        new = 1 if rng.random() < 0.4 else spread(1, max(1, min(1500, room // (batch * (heads + 2 * kv_heads)))))
        length = new + spread(1, 500) - 1
    elif op == "read":
        new, length = 0, spread(1, max(1, min(8192, 3 * room // (batch * kv_heads))))
    else:
        new = rng.choice((1, 1, 1, 2, 3, 4, 7, spread(8, 700)))
        length = spread(1, max(1, min(131072, 12 * room // (batch * kv_heads))))
        if new > 1:                     # the score of every pair is computed: at most an eighth of the listed chunk's
            new = max(1, min(new, math.isqrt((1 << 26) // (batch * heads)), room // (batch * heads)))
            length = max(new, min(length, (1 << 26) // (batch * heads * new)))
    return _case(op, batch=batch, new=new, length=length, heads=heads if op in ("project", "attend") else 0, kv_heads=kv_heads,
                 dim=dim, group=group, page=page, type=type, ragged=ragged)


def _lengths(case):
    """(tokens of each sequence, new ones among them): the longest first; ragged ones spread evenly down to none."""
    batch, longest, new = case["batch"], case["length"], case["new"]
    if not case["ragged"]:
        return [longest] * batch, [new] * batch
    shares = [1.0] + [(i * 0.6180339887498949) % 1.0 for i in range(1, batch)]
    if case["op"] == "attend":
        lengths = [round(longest * s) for s in shares]
        if batch > 2:
            lengths[batch // 2] = 0
        return lengths, [new] * batch
    if case["op"] == "read":
        return [round(longest * s) for s in shares], [0] * batch
    if case["op"] == "project":         # the prefixes are ragged; every sequence brings the same number of tokens
        return [new + round((longest - new) * s) for s in shares], [new] * batch
    news = [max(1, round(new * s)) for s in shares]
    return [n + round((longest - new) * s) for n, s in zip(news, reversed(shares))], news


def _inputs(case, seed):
    """Everything that the seed decides, the same for both forms and for ``exact``."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dim, kv_heads, batch, new = TYPES[case["type"]], case["dim"], case["kv_heads"], case["batch"], case["new"]
    lengths, news = _lengths(case)

    def rows(n, heads, spread):
        """[n, heads, dim]: normal values, on channels of different means and widths as keys have them."""
        wide = torch.exp(spread * torch.randn(heads, dim, generator=gen, device="cuda"))
        mean = spread * torch.randn(heads, dim, generator=gen, device="cuda")
        return (torch.randn(n, heads, dim, generator=gen, device="cuda") * wide + mean).to(kind)

    pages_each = -(-max(case["length"], 1) // case["page"])
    pages = batch * pages_each + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[: batch * pages_each].view(batch, -1).int()
    length = torch.tensor(lengths, dtype=torch.int32)
    fresh = torch.tensor(news, dtype=torch.int32)
    s = {"table": table, "lengths": length.cuda(), "offsets": (length - fresh).cuda(), "news": fresh.cuda(), "pages": pages}
    if case["op"] in ("write", "project"):
        counts, first = fresh, length - fresh       # the rows that come out: the new ones
    else:
        counts, first = length, torch.zeros_like(length)    # all of them
    s["total"] = int(counts.sum())
    s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int32), counts.cumsum(0).int()]).cuda()
    s["of"] = torch.repeat_interleave(torch.arange(batch), counts).cuda()
    s["nth"] = (torch.arange(s["total"]) - torch.repeat_interleave(counts.cumsum(0) - counts, counts)).cuda()
    position = s["nth"] + torch.repeat_interleave(first, counts).cuda()
    s["slots"] = table[s["of"], position // case["page"]].long() * case["page"] + position % case["page"]
    if case["op"] == "write":           # K and V as two of three parts of one projection's rows
        both = torch.cat([rows(batch * new, kv_heads, 0.5), rows(batch * new, kv_heads, 0.1)], 1).view(batch, new, 2 * kv_heads, dim)
        s["k"], s["v"] = both[:, :, :kv_heads], both[:, :, kv_heads:]
    elif case["op"] == "project":
        parts = [rows(batch * new, case["heads"] + kv_heads, 0.1), rows(batch * new, kv_heads, 0.1)]
        s["qkv"] = torch.cat(parts, 1).view(batch, new, -1)
        s["q_w"], s["k_w"] = ((1 + 0.1 * torch.randn(2, dim, generator=gen, device="cuda")).to(kind)).unbind(0)
        angles = torch.outer(torch.arange(case["length"], device="cuda", dtype=torch.float64),
                             THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
        s["positions"] = s["offsets"][:, None].long() + torch.arange(new, device="cuda")
        s["totals"] = torch.zeros(batch, dtype=torch.int32, device="cuda")
    else:                               # rows that earlier calls have cached
        s["k"], s["v"] = rows(s["total"], kv_heads, 0.5), rows(s["total"], kv_heads, 0.1)
    if case["op"] == "attend":          # scores spread over a few units, as trained heads have them
        q = torch.randn(batch, new, case["heads"], dim, generator=gen, device="cuda")
        s["q"] = (q * torch.exp(0.4 * torch.randn(case["heads"], 1, generator=gen, device="cuda"))).to(kind)
    return s


def prepare(case, seed):
    """The rows of this step and the cache as a serving program holds it: its own pages in either form, filled by what
    came before the call."""
    s = _inputs(case, seed)
    shape = (s["pages"], case["page"], case["kv_heads"], case["dim"], case["group"], TYPES[case["type"]])
    if own:
        from triton_distributed_gh_amd.ops import kv4

        pages, page, heads, dim, group, kind = shape
        s["cache"] = kv4.Int4KVCache.alloc(pages, page, heads, dim, group=group, dtype=kind, device="cuda")
    else:
        s["cache"] = _empty(*shape)
    if case["op"] in ("read", "attend"):
        k, v = s.pop("k"), s.pop("v")
        if own and s["total"]:
            longest = int(s["lengths"].max())
            padded = [torch.zeros(case["batch"], longest, *x.shape[1:], dtype=x.dtype, device=x.device) for x in (k, v)]
            for x, rows in zip(padded, (k, v)):
                x[s["of"], s["nth"]] = rows
            kv4.kv4_append(*padded, s["cache"], torch.zeros_like(s["offsets"]), s["table"], new_lens=s["lengths"])
        elif s["total"]:
            _store(s["cache"], s["slots"], k, v)
    s["case"] = case
    return s


def run(s):
    return {"write": _write, "project": _project, "read": _read, "attend": _attend}[s["case"]["op"]](s)


def _write(s):
    if own:
        from triton_distributed_gh_amd.ops import kv4

        kv4.kv4_append(s["k"], s["v"], s["cache"], s["offsets"], s["table"], new_lens=s["news"])
        return kv4.kv4_read(s["cache"], s["table"], s["cu"], s["total"], starts=s["offsets"])
    _store(s["cache"], s["slots"], s["k"][s["of"], s["nth"]], s["v"][s["of"], s["nth"]])
    return _load(s["cache"], s["slots"])


def _read(s):
    if own:
        from triton_distributed_gh_amd.ops import kv4

        return kv4.kv4_read(s["cache"], s["table"], s["cu"], s["total"])
    return _load(s["cache"], s["slots"])


def _project(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if own:
        from triton_distributed_gh_amd.ops import kv4

        q = kv4.kv4_qkv_prep(s["qkv"], s["q_w"], s["k_w"], EPS, EPS, s["positions"], s["cos"], s["sin"], s["cache"],
                             s["offsets"], s["totals"], s["table"], heads)
        return (q, s["totals"], *kv4.kv4_read(s["cache"], s["table"], s["cu"], s["total"], starts=s["offsets"]))
    q, k, v = s["qkv"].unflatten(-1, (-1, dim)).split([heads, kv_heads, kv_heads], 2)
    q, k = _normed(q, s["q_w"]), _normed(k, s["k_w"])
    cos, sin = (t[s["positions"]].unsqueeze(2).double() for t in (s["cos"], s["sin"]))
    q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    s["totals"].copy_(s["offsets"] + case["new"])
    _store(s["cache"], s["slots"], k.flatten(0, 1), v.flatten(0, 1))
    return (q, s["totals"], *_load(s["cache"], s["slots"]))


def _attend(s):
    case = s["case"]
    if own:
        from triton_distributed_gh_amd.ops import kv4

        return kv4.flash_attn_with_kv4cache(s["q"], s["cache"], s["lengths"], s["table"])
    batch, new, heads, dim = s["q"].shape
    kv_heads = case["kv_heads"]
    table = s["table"].long()
    slots = (table.unsqueeze(-1) * case["page"] + torch.arange(case["page"], device=table.device)).flatten(1)
    k, v = (_values(p, slots).transpose(1, 2).contiguous() for p in s["cache"])
    q = s["q"].float().view(batch, new, kv_heads, -1, dim).transpose(1, 2).reshape(batch, kv_heads, -1, dim)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(dim)
    scores = scores.view(batch, kv_heads, new, -1, slots.shape[1])
    last = s["lengths"][:, None] - new + torch.arange(new, device=table.device)     # the last token that a query sees
    hidden = torch.arange(slots.shape[1], device=table.device) > last.unsqueeze(-1)
    scores = scores.masked_fill_(hidden[:, None, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    weights = weights / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(weights.flatten(2, 3), v).view(batch, kv_heads, new, -1, dim)
    return out.transpose(1, 2).reshape(batch, new, heads, dim).to(s["q"].dtype)


# ---- the plain cache: two codes to a byte, pages of [token, head] rows ---------------------------------------------
def _empty(pages, page, heads, dim, group, kind):
    def half():
        return (torch.zeros(pages * page, heads, dim // 2, dtype=torch.uint8, device="cuda"),
                torch.zeros(pages * page, heads, dim // group, dtype=kind, device="cuda"),
                torch.zeros(pages * page, heads, dim // group, dtype=kind, device="cuda"))

    return half(), half()


def _store(cache, slots, k, v):
    _store_one(cache[0], slots, k)
    _store_one(cache[1], slots, v)


def _store_one(part, slots, x):
    codes, scale, low = part
    x = x.float().unflatten(-1, (scale.shape[-1], -1))
    least = x.amin(-1, keepdim=True)
    step = ((x.amax(-1, keepdim=True) - least) / 15).to(scale.dtype).float()
    code = torch.where(step == 0, 0.0, torch.round((x - least) / step)).clamp(0, 15).to(torch.uint8).flatten(-2)
    codes[slots] = code[..., 0::2] | (code[..., 1::2] << 4)
    scale[slots] = step.squeeze(-1).to(scale.dtype)
    low[slots] = least.squeeze(-1).to(low.dtype)


def _load(cache, slots):
    return tuple(_values(p, slots).to(p[1].dtype) for p in cache)


def _values(part, slots):
    """The 32-bit values that the rows at ``slots`` stand for."""
    codes, scale, low = part
    code = codes[slots]
    code = torch.stack([code & 15, code >> 4], -1).flatten(-2).float().unflatten(-1, (scale.shape[-1], -1))
    return (code * scale[slots].float().unsqueeze(-1) + low[slots].float().unsqueeze(-1)).flatten(-2)


def _normed(x, weight):
    """Values beside the border between two codes decide a code: the mean square is taken in 64 bits."""
    inverse = (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
    return (x.float() * inverse * weight.float()).to(x.dtype)


def _rotated(x, cos, sin):
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float().to(x.dtype)


# ---- counts and 64-bit results -------------------------------------------------------------------------------------
def work(case):
    """One pass's bytes and operations: inputs once, outputs once, the cached rows as 4 bits and their group's two numbers."""
    lengths, news = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    cached = 2 * kv_heads * (dim / 2 + 4 * dim / case["group"])        # one token's K and V in the cache
    wide = 2 * kv_heads * dim * 2                                      # and in 16 bits
    tokens, fresh = sum(lengths), sum(news)
    if case["op"] == "write":           # rows in, codes out and in again, rows out
        return {"bytes": fresh * (2 * wide + 2 * cached), "flops": fresh * wide * 3}
    if case["op"] == "read":
        return {"bytes": tokens * (wide + cached), "flops": tokens * wide}
    if case["op"] == "project":         # the rotation's tables are read once
        return {"bytes": fresh * (2 * wide + 2 * cached + 2 * heads * dim * 2) + case["length"] * dim * 4,
                "flops": fresh * (wide * 5 + heads * dim * 7)}
    pairs = sum(max(0, n - i) for n in lengths for i in range(case["new"]))
    return {"bytes": tokens * cached + 2 * case["batch"] * case["new"] * heads * dim * 2, "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    """From the definition, in 64 bits; the rows' own roundings (to 16 bits, to a code) are part of it."""
    s = _inputs(case, seed)
    kind, dim = TYPES[case["type"]], case["dim"]

    def held(x):
        parts = x.double().reshape(*x.shape[:-1], -1, case["group"])
        low, high = parts.min(-1, keepdim=True).values, parts.max(-1, keepdim=True).values
        step = ((high - low).float() / 15).to(kind).double()
        code = torch.where(step > 0, ((parts - low).float().double() / step).float().round(), 0.0).clamp(0, 15)
        return (code.double() * step + low).reshape(x.shape)

    if case["op"] in ("write", "read"):
        k, v = (s["k"][s["of"], s["nth"]], s["v"][s["of"], s["nth"]]) if case["op"] == "write" else (s["k"], s["v"])
        return held(k), held(v)
    if case["op"] == "project":
        heads, kv_heads, new = case["heads"], case["kv_heads"], case["new"]
        rows = s["qkv"].reshape(case["batch"] * new, -1, dim)
        at = s["positions"].flatten()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at].unsqueeze(1)

        def turned(x, weight):
            x = x.double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + EPS) * weight.double()
            x = x.to(kind).double()
            z = torch.complex(x[..., : dim // 2].contiguous(), x[..., dim // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        q, k = turned(rows[:, :heads], s["q_w"]), turned(rows[:, heads:heads + kv_heads], s["k_w"]).to(kind)
        return q.view(case["batch"], new, heads, dim), None, held(k), held(rows[:, heads + kv_heads:])
    if case["new"] * case["length"] * case["batch"] * case["heads"] > 1 << 30:
        return None
    out = torch.zeros(case["batch"], case["new"], case["heads"], dim, dtype=torch.float64, device="cuda")
    k, v = held(s["k"]), held(s["v"])
    lengths, _ = _lengths(case)
    share = case["heads"] // case["kv_heads"]
    start = 0
    for b, length in enumerate(lengths):
        for h in range(case["kv_heads"] if length else 0):
            q = s["q"][b, :, h * share:(h + 1) * share].double()
            scores = (q.reshape(-1, dim) @ k[start:start + length, h].T.contiguous()).view(case["new"], share, length) * dim ** -0.5
            sees = length - case["new"] + torch.arange(case["new"], device="cuda")
            scores[(torch.arange(length, device="cuda") > sees[:, None])[:, None].expand_as(scores)] = -math.inf
            weights = torch.softmax(scores, -1).nan_to_num(0.0)
            out[b, :, h * share:(h + 1) * share] = (weights.view(-1, length) @ v[start:start + length, h]).view(case["new"], share, dim)
        start += length
    return out
