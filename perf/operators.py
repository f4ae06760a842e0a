"""The paged key/value cache of a decode layer and the attention over it: what is measured, and the plain forms.

Three operators, called in a row between the qkv and the o projection: `append` writes the new tokens' keys and values
into the cache (quantised to e4m3 with a power of two per row, or copied), `read` brings cached tokens back, `attend`
is the attention of each sequence's new tokens over its cached ones. All lengths of a case follow from its own values.
"""

import math
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LOW, HIGH = -100, 119  # range of a row's exponent


def _gemm():
    if "sm120-lowlat-gemm_b200" not in sys.path:
        sys.path.insert(0, "sm120-lowlat-gemm_b200")
    import lowlat_gemm

    return lowlat_gemm


# ---------------------------------------------------------------------------------------------------------------------
# cases


def _case(name, op, **kw):
    c = dict(op=op, batch=1, new_min=1, new_max=1, kv_min=1, kv_max=1, heads=8, kv_heads=1, dim=128, page=16, dtype="bf16",
             cache="e4m3", window=0, lse=False, spread=0)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one sequence decodes one token of a 64-head layer with 8 key/value heads: pure latency
        _case("append_one_token", "append", kv_min=700, kv_max=700, heads=64, kv_heads=8, page=64),
        # a serving batch on one of eight tensor-parallel ranks, 16-bit cache, a ragged number of new tokens
        _case("append_batch_16bit", "append", batch=48, new_min=0, new_max=9, kv_min=40, kv_max=3000, heads=8, kv_heads=1,
              dtype="f16", cache="same", spread=1),
        # a prompt's chunk of 8192 tokens
        _case("append_prompt_chunk", "append", new_min=8192, new_max=8192, kv_min=8192, kv_max=8192, heads=64, kv_heads=8, page=64),
        # a few short sequences brought back, head dimension 64
        _case("read_short", "read", batch=3, kv_min=75, kv_max=333, heads=32, kv_heads=4, dim=64, dtype="f16", spread=2),
        # prefix hand-over of a full batch
        _case("read_prefixes", "read", batch=8, kv_min=5000, kv_max=8192, heads=64, kv_heads=8, page=64, spread=3),
        # one user decoding on one of eight tensor-parallel ranks: pure latency
        _case("decode_one", "attend", kv_min=777, kv_max=777, heads=8, kv_heads=1, page=16),
        # an ordinary decode batch over an e4m3 cache, ragged lengths
        _case("decode_batch", "attend", batch=32, kv_min=900, kv_max=8200, heads=64, kv_heads=8, page=64, spread=4),
        # four long documents on one of four tensor-parallel ranks, 16-bit cache
        _case("decode_long", "attend", batch=4, kv_min=50000, kv_max=65531, heads=16, kv_heads=2, page=128, cache="same", spread=5),
        # drafted tokens verified: five new tokens per sequence, four query heads to a key/value head, dimension 64
        _case("verify_drafts", "attend", batch=16, new_min=5, new_max=5, kv_min=300, kv_max=2500, heads=32, kv_heads=8, dim=64,
              dtype="f16", cache="same", page=16, lse=True, spread=6),
        # a chunk of a prompt behind its first 8 thousand tokens, e4m3 cache
        _case("chunk_512", "attend", new_min=512, new_max=512, kv_min=8704, kv_max=8704, heads=64, kv_heads=8, page=64),
        # prompts' chunks and decoding sequences in one batch, sliding window, odd lengths
        _case("mixed_window", "attend", batch=12, new_min=0, new_max=700, kv_min=800, kv_max=4100, heads=32, kv_heads=4,
              cache="same", page=32, window=1024, spread=7),
        # the last chunk of a long prompt
        _case("chunk_2048_long", "attend", new_min=2048, new_max=2048, kv_min=16384, kv_max=16384, heads=64, kv_heads=8,
              cache="same", page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 16])
    while kv_heads * group > 64:
        group = rng.choice([1, 2, 4, 5, 7, 8])
    dtype, cache = rng.choice(["bf16", "f16"]), rng.choice(["e4m3", "same"])
    kw = dict(heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, cache=cache, page=rng.choice([16, 32, 48, 64, 128, 256]),
              spread=rng.randrange(1 << 20))
    if op == "append":
        batch = _log(rng, 1, 256)
        new = _log(rng, 1, max(1, 8192 // batch))
        kv = new + _log(rng, 1, 4000)
        if rng.random() < 0.2 and cache == "e4m3":
            kw["dtype"] = "f32"
        return _case("", op, batch=batch, new_min=rng.choice([new, new // 2]), new_max=new, kv_min=new, kv_max=kv, **kw)
    if op == "read":
        batch = _log(rng, 1, 32)
        kv = _log(rng, 1, 65536 // batch)
        return _case("", op, batch=batch, kv_min=rng.choice([kv, max(1, kv // 3)]), kv_max=kv, **kw)
    form = rng.choice(["decode", "drafts", "chunk", "mixed"])
    if form == "decode":
        batch = _log(rng, 1, 128)
        low = new = 1
        kv = _log(rng, 1, 262144 // (batch * max(1, kv_heads // 2)))
    elif form == "drafts":
        batch = _log(rng, 1, 64)
        low = new = rng.randint(2, 8)
        kv = new + _log(rng, 1, 65536 // batch)
    elif form == "chunk":
        batch = 1
        low = new = _log(rng, 16, 2048)
        kv = new + _log(rng, 1, 14336)
    else:
        batch = rng.randint(2, 12)
        low, new = 0, _log(rng, 8, 700)
        kv = new + _log(rng, 1, 3400)
    window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    return _case("", op, batch=batch, new_min=low, new_max=new, kv_min=max(new, kv // rng.choice([1, 4])), kv_max=kv, window=window,
                 lse=rng.random() < 0.3, **kw)


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence; in a mixed batch one in three is a chunk."""
    rng = random.Random(case["spread"])
    new, kv = [], []
    for i in range(case["batch"]):
        n = case["new_max"] if i == 0 else rng.randint(case["new_min"], case["new_max"])
        if case["new_max"] > 16 and case["new_min"] == 0 and i % 3:
            n = min(n, 1)
        length = case["kv_max"] if i == 0 else rng.randint(case["kv_min"], case["kv_max"])
        new.append(n)
        kv.append(length)
    return new, kv


def _pairs(n, length, window):
    """Visible (query, key) pairs of one sequence, and the first key that any query sees."""
    first = length - n  # position of the first new token
    if not window:
        return n * first + n * (n + 1) // 2, 0
    pairs = sum(min(first + t + 1, window) for t in range(n))
    return pairs, max(0, first + 1 - window) if n else length


def work(case):
    new, kv = _lengths(case)
    dim, kvh, heads = case["dim"], case["kv_heads"], case["heads"]
    wide = TYPES[case["dtype"]].itemsize
    row = dim + 1 if case["cache"] == "e4m3" else dim * wide  # bytes of a cached row
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": 2 * tokens * kvh * (dim * wide + row), "flops": 2 * tokens * kvh * dim}
    if case["op"] == "read":
        return {"bytes": 2 * kvh * (sum(kv) * row + case["batch"] * max(kv) * dim * wide), "flops": 2 * sum(kv) * kvh * dim}
    pairs = read = 0
    for n, length in zip(new, kv):
        p, first = _pairs(n, length, case["window"])
        pairs += p
        read += length - first if n else 0
    return {"bytes": 2 * tokens * heads * dim * wide + 2 * read * kvh * row + (4 * tokens * heads if case["lse"] else 0),
            "flops": 4 * dim * heads * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    new, kv = _lengths(case)
    batch, page, kvh, dim = case["batch"], case["page"], case["kv_heads"], case["dim"]
    dtype = TYPES[case["dtype"]]
    per_seq = [-(-n // page) for n in kv]
    pages, width = sum(per_seq) + 3, max(per_seq)
    order = torch.randperm(pages, generator=g, device=dev, dtype=torch.int32).tolist()  # pages lie anywhere in the cache
    table, at = [], 0
    for n in per_seq:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    s = {"case": case, "max_len": max(kv), "k_scale": None, "v_scale": None, "q_starts": None}
    s["page_table"] = torch.tensor(table, dtype=torch.int32, device=dev)
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device=dev)
    if len(set(new)) > 1:
        s["q_starts"] = torch.tensor([sum(new[:i]) for i in range(batch + 1)], dtype=torch.int32, device=dev)
    shape = (pages, kvh, page, dim)
    if case["cache"] == "e4m3":
        for name in ("k", "v"):
            x = torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16)
            s[name + "_cache"] = (x * 100).clamp(-448, 448).to(E4M3)
            e = torch.randint(119, 122, shape[:3], generator=g, device=dev)  # rows of about 0.4 to 1.6
            s[name + "_scale"] = e.to(torch.uint8).view(E8M0)
    else:
        for name in ("k", "v"):
            s[name + "_cache"] = torch.randn(shape, generator=g, device=dev, dtype=dtype)
    heads, tokens = case["heads"], sum(new)
    if case["op"] != "read":
        # what the qkv projection leaves: [tokens, (heads + 2 * kv_heads) * dim], some channels much larger than the rest
        qkv = torch.randn(tokens, (heads + 2 * kvh) * dim, generator=g, device=dev, dtype=torch.float32)
        loud = torch.rand(qkv.shape[1], generator=g, device=dev) < 0.02
        qkv = (qkv * torch.where(loud, 4.0, 1.0)).to(dtype)
        s["q"] = qkv[:, :heads * dim].view(tokens, heads, dim)
        s["k"] = qkv[:, heads * dim:(heads + kvh) * dim].view(tokens, kvh, dim)
        s["v"] = qkv[:, (heads + kvh) * dim:].view(tokens, kvh, dim)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass


def run(s):
    case = s["case"]
    cache = (s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"])
    scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if case["op"] == "append":
        if own:
            _gemm().kv_append(s["k"], s["v"], *cache, q_starts=s["q_starts"], **scales)
        else:
            _plain_append(s)
        return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None}
    if case["op"] == "read":
        if own:
            return _gemm().kv_read(*cache, s["max_len"], out_dtype=TYPES[case["dtype"]], **scales)
        return _plain_read(s)
    if own:
        return _gemm().paged_attention(s["q"], *cache, q_starts=s["q_starts"], window=case["window"], return_lse=case["lse"], **scales)
    return _plain_attend(s)


def _starts(s, tokens):
    if s["q_starts"] is not None:
        return s["q_starts"].long()
    batch = s["kv_lens"].shape[0]
    return torch.arange(batch + 1, device=s["kv_lens"].device) * (tokens // batch)


def _plain_append(s):
    tokens = s["k"].shape[0]
    starts, lens = _starts(s, tokens), s["kv_lens"].long()
    t = torch.arange(tokens, device=lens.device)
    seq = torch.searchsorted(starts, t, right=True) - 1
    pos = lens[seq] - starts[seq + 1] + t
    page = s["k_cache"].shape[2]
    where = s["page_table"].long()[seq, pos // page]
    slot = pos % page
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        if scale is None:
            cache[where, :, slot] = x
            continue
        x = x.float()
        amax = x.abs().amax(-1)
        m, e = torch.frexp(amax)  # amax = m * 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
        e = (e - 9 + (m > 0.875)).clamp(LOW, HIGH)
        e = torch.where(amax > 0, e, LOW)
        y = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(E4M3)
        cache.view(torch.uint8)[where, :, slot] = y.view(torch.uint8)
        scale.view(torch.uint8)[where, :, slot] = (e + 127).to(torch.uint8)


def _gathered(s, name, length):
    """float32 [batch, kv_heads, length, dim]: the cached rows of every sequence in order."""
    table = s["page_table"].long()
    x = s[name + "_cache"].view(torch.uint8)[table].view(E4M3) if s[name + "_scale"] is not None else s[name + "_cache"][table]
    x = x.float()
    if s[name + "_scale"] is not None:
        x = x * torch.exp2(s[name + "_scale"].view(torch.uint8)[table].float() - 127)[..., None]
    b, p, h, page, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * page, d)[:, :, :length]


def _plain_read(s):
    length, dtype = s["max_len"], TYPES[s["case"]["dtype"]]
    there = torch.arange(length, device=s["kv_lens"].device) < s["kv_lens"][:, None]
    return tuple(torch.where(there[:, :, None, None], _gathered(s, name, length).transpose(1, 2), 0.0).to(dtype).contiguous()
                 for name in ("k", "v"))


def _plain_attend(s):
    case, q = s["case"], s["q"]
    tokens, heads, dim = q.shape
    kvh, length = case["kv_heads"], s["max_len"]
    dev = q.device
    starts, lens = _starts(s, tokens), s["kv_lens"].long()
    count = starts[1:] - starts[:-1]
    most = case["new_max"]
    j = torch.arange(most, device=dev)
    token = (starts[:-1, None] + j).clamp(max=tokens - 1)
    batch = lens.shape[0]
    qp = q.float()[token].view(batch, most, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(batch, kvh, -1, dim)
    k, v = _gathered(s, "k", length), _gathered(s, "v", length)
    x = torch.matmul(qp, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))  # [batch, kv_heads, group * most, length]
    pos = (lens - count)[:, None] + j  # position of query j
    key = torch.arange(length, device=dev)
    seen = (key <= pos[:, :, None]) & (key < lens[:, None, None])
    if case["window"]:
        seen &= key > pos[:, :, None] - case["window"]
    seen = seen[:, None, None].expand(batch, kvh, heads // kvh, most, length).reshape(batch, kvh, -1, length)
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).squeeze(-1)
    o = o.view(batch, kvh, heads // kvh, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    lse = lse.view(batch, kvh, heads // kvh, most).permute(0, 3, 1, 2).reshape(batch, most, heads)
    t = torch.arange(tokens, device=dev)
    seq = torch.searchsorted(starts, t, right=True) - 1
    o, lse = o[seq, t - starts[seq]].to(q.dtype), lse[seq, t - starts[seq]]
    return (o, lse) if case["lse"] else o


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence


def _nearest_e4m3(y):
    """The e4m3 value nearest to y, ties to even: steps of 1/8 of the power of two below, 2^-9 at the least."""
    size = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
    size = torch.where(y.abs() >= torch.exp2(size + 1), size + 1, size)
    step = torch.exp2(size.clamp_min(-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _row64(s, name, i, j0, j1):
    """Keys or values j0..j1 of sequence i, float64 [kv_heads, j1 - j0, dim]."""
    page = s["case"]["page"]
    j = torch.arange(j0, j1, device=s["kv_lens"].device)
    where = s["page_table"][i].long()[torch.div(j, page, rounding_mode="floor")]
    if s[name + "_scale"] is None:
        return s[name + "_cache"][where, :, j % page].double().transpose(0, 1)
    x = s[name + "_cache"].view(torch.uint8)[where, :, j % page].view(E4M3).double()
    return (x * torch.exp2(s[name + "_scale"].view(torch.uint8)[where, :, j % page].double() - 127)[..., None]).transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    new, kv = _lengths(case)
    if case["op"] == "append":
        return _exact_append(s, new, kv)
    if case["op"] == "read":
        out = []
        for name in ("k", "v"):
            x = torch.zeros(case["batch"], max(kv), case["kv_heads"], case["dim"], dtype=torch.float64, device="cuda")
            for i, n in enumerate(kv):
                x[i, :n] = _row64(s, name, i, 0, n).transpose(0, 1)
            out.append(x)
        return tuple(out)
    group, at = case["heads"] // case["kv_heads"], 0
    o = torch.zeros(sum(new), case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for i, (n, length) in enumerate(zip(new, kv)):
        if n == 0:
            continue
        k, v = _row64(s, "k", i, 0, length), _row64(s, "v", i, 0, length)
        ahead = torch.arange(length, device="cuda")[None] - torch.arange(length - n, length, device="cuda")[:, None]
        hidden = ahead > 0
        if case["window"]:
            hidden |= ahead <= -case["window"]
        for h in range(case["heads"]):
            x = s["q"][at:at + n, h].double() @ k[h // group].T / math.sqrt(case["dim"])
            x[hidden] = -math.inf
            lse[at:at + n, h] = torch.logsumexp(x, -1)
            o[at:at + n, h] = torch.softmax(x, -1) @ v[h // group]
        at += n
    return (o, lse) if case["lse"] else o


def _exact_append(s, new, kv):
    page, at = s["case"]["page"], 0
    out = {}
    for name in ("k", "v"):
        scaled = s[name + "_scale"] is not None
        cache = s[name + "_cache"].float().double()
        scale = torch.exp2(s[name + "_scale"].view(torch.uint8).double() - 127) if scaled else None
        at = 0
        for i, (n, length) in enumerate(zip(new, kv)):
            j = torch.arange(length - n, length, device="cuda")
            where = s["page_table"][i].long()[torch.div(j, page, rounding_mode="floor")]
            x = s[name][at:at + n].double()
            if scaled:
                amax = x.abs().amax(-1)
                e = torch.ceil(torch.log2(amax / 448))
                e = torch.where(amax <= 448 * torch.exp2(e - 1), e - 1, e)  # log2 may miss a power of two by its last bit
                e = torch.where(amax > 448 * torch.exp2(e), e + 1, e).clamp(LOW, HIGH)
                scale[where, :, j % page] = torch.exp2(e)
                x = _nearest_e4m3(x / torch.exp2(e)[..., None])
            cache[where, :, j % page] = x
            at += n
        out[name + "_cache"] = cache
        if scaled:
            out[name + "_scale"] = scale
    return out
