"""Paged cache and attention where they can go wrong: the cache's end, rows that a query may not see, powers of two far apart,
weights far below the largest."""
import ctypes as C
import math

import pytest
import torch

import lowlat_gemm as L
from lowlat_gemm import _native as N, tp as TP

from test_gpu_attention import BF, E4M3, E8M0, HF, make_cache, pages_for, rows_of
from test_gpu_decode_attention import SHAPE, recorded

pytestmark = pytest.mark.gpu


def expected(q, kc, vc, ks, vs, table, lens, starts, *, scale=None, causal=True, window=0, shared=0):
    """(o, lse, tolerance of o) in float64 by the definition: the new tokens' positions count back from the length as it is given,
    keys end where the page table ends, and every bound comes from the keys that the query sees."""
    tokens, heads, dim = q.shape
    group, cap = heads // kc.shape[1], table.shape[1] * kc.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    o = torch.zeros(tokens, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    for i, length in enumerate(lens):
        t0, t1 = starts[i], starts[i + 1]
        keys, n = min(length, cap), t1 - t0
        if n == 0 or keys == 0:
            continue
        k, v = (rows_of(c, s, table, i, keys).repeat_interleave(group, 1) for c, s in ((kc, ks), (vc, vs)))
        e = rows_of(torch.ones_like(vc), vs, table, i, keys)[..., :1].repeat_interleave(group, 1)  # powers of two of V's rows, 1 for 16 bits
        qq = q[t0:t1].double()
        s = torch.einsum("thd,jhd->thj", qq, k) * scale
        pos = length - n + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(keys, device="cuda")[None]
        seen = (j <= pos) if causal else torch.ones(n, keys, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & (j > pos - window)
        s = torch.where(seen[:, None], s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        w = p / torch.where(total == 0, 1.0, total)
        o[t0:t1] = torch.einsum("thj,jhd->thd", w, v)
        lse[t0:t1] = (top + torch.log(total)).squeeze(-1)
        # half a step of the result, half a step of each probability, 2^-24 for each product and sum over keys; a score is a dot
        # product of dim fp32 products and sums, 2^-24 each of sum |q||k|, and moves a weight by twice its error; exp2 adds 2^-21
        mass = torch.einsum("thj,jhd->thd", w, v.abs())
        sizes = torch.einsum("thd,jhd->thj", qq.abs(), k.abs()) * abs(scale)
        delta = torch.where(seen[:, None], sizes, 0.0).amax(-1, keepdim=True) * (dim + 4) * 2.0 ** -24 + 2.0 ** -21
        # f16 probabilities, times their row's power of two, are whole multiples of 2^-24, off by half of one, the largest being 2^7 at
        # the least; rows of a tile may share a power of two `shared` binary orders above their own
        least = torch.einsum("tj,jhd->thd", seen.double(), (v / e).abs()) * (w * e.permute(2, 1, 0)).amax(-1, keepdim=True) * 2.0 ** (shared - 32)
        tol[t0:t1] = half * o[t0:t1].abs() + mass * (half + 2 * delta + keys * 2.0 ** -24) + torch.finfo(q.dtype).tiny + (0 if kc.dtype == BF else least)
    return o, lse, tol


def setup(news, lens, heads, kvh, dim, page, qt, ct, *, seed=0, width=None, ragged=True):
    """(q, cache arguments, scales, starts): lens may go beyond width * page, where no row of the cache lies."""
    cap = (width or 1 << 30) * page
    table, pages = pages_for([min(n, cap) for n in lens], page, seed, width=width)
    kc, vc, ks, vs = make_cache(pages, kvh, page, dim, ct, seed + 1)
    q = torch.randn(sum(news), heads, dim, generator=torch.Generator().manual_seed(seed + 2)).to(qt).cuda()
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    kw = dict(k_scale=ks, v_scale=vs)
    if ragged:
        kw["q_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    return q, (kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda")), kw, starts


def compare(q, cache, kw, starts, lens, *, causal=True, window=0, scale=None, shared=0):
    out, lse = L.paged_attention(q, *cache, causal=causal, window=window, scale=scale, return_lse=True, **kw)
    want, wl, tol = expected(q, cache[0], cache[1], kw["k_scale"], kw["v_scale"], cache[2], lens, starts, causal=causal, window=window,
                             scale=scale, shared=shared)
    most = torch.finfo(q.dtype).max  # a result behind the type's largest value is infinite
    err = torch.where((out == torch.copysign(torch.full_like(out, math.inf), out)) & (want * out.sign() + tol >= most), 0.0, (out.double() - want).abs())
    assert bool((err <= tol).all()), f"error {err.max().item():.3e}, {(err / tol).max().item():.2f} of its bound"
    assert torch.equal(torch.isfinite(lse), torch.isfinite(wl))
    fin = torch.isfinite(wl)
    # a score is off by 2^-18 of its size (|lse| and dim bound it here), the logarithm of the sum by 2^-19
    assert bool(((lse.double() - wl)[fin].abs() <= 2.0 ** -18 * (1 + wl[fin].abs() + q.shape[2])).all())
    assert N.device_status() == 0
    return out


# ---------------------------------------------------------------------------------------------------------------------
# lengths beyond the page table


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("news,lens", [([3], [66]), ([1, 1], [65, 64]), ([5, 5, 5], [70, 64, 68]), ([40, 2], [80, 65]), ([300], [120]),
                                       ([2], [500]), ([90], [700])])
def test_positions_beyond_the_page_table(news, lens, ct):
    """Four pages of 16: tokens behind the 64th are not there, and the queries before and behind the end keep their positions."""
    for qt, dim, heads, kvh in ((BF, 128, 8, 1), (HF, 64, 10, 2)):
        for kw in ({}, dict(window=9), dict(window=70), dict(causal=False), dict(causal=False, window=9)):
            for ragged in (True, False) if len(set(news)) == 1 else (True,):
                q, cache, args, starts = setup(news, lens, heads, kvh, dim, 16, qt, E4M3 if ct == "e4m3" else qt, seed=lens[0], width=4,
                                               ragged=ragged)
                compare(q, cache, args, starts, lens, **kw)


@pytest.mark.parametrize("ct", [BF, E4M3])
@pytest.mark.parametrize("new", [3, 40])
def test_append_and_attention_agree_on_positions(new, ct):
    """With a window of one a query's result is its own token's value, or zero where the cache had no place for it."""
    table, pages = pages_for([64], 16, 3)
    kc, vc, ks, vs = make_cache(pages, 1, 16, 128, ct, 4)
    kv = torch.randint(8, 16, (new, 2, 128), generator=torch.Generator().manual_seed(5)).to(BF).cuda()  # four bits: e4m3 holds them
    q = torch.randn(new, 8, 128, generator=torch.Generator().manual_seed(6)).to(BF).cuda()
    for length in (64, 65, 64 + new - 1, 64 + new, 64 + 2 * new):
        ln = torch.tensor([length], dtype=torch.int32, device="cuda")
        L.kv_append(kv[:, :1], kv[:, 1:], kc, vc, table, ln, k_scale=ks, v_scale=vs)
        out = L.paged_attention(q, kc, vc, table, ln, k_scale=ks, v_scale=vs, window=1)
        there = (torch.arange(length - new, length, device="cuda") < 64)[:, None, None]
        want = torch.where(there, kv[:, 1:].double(), 0.0).expand(new, 8, 128)
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want).all()), length  # the result's rounding; the one weight is 1


@pytest.mark.parametrize("dtype", [E4M3, BF])
def test_steps_that_cross_the_end_of_the_cache(dtype):
    """Tokens behind the cache's end are not stored; queries of the step that crosses it and of later ones still see what is there."""
    batch, new, dev = 2, 3, torch.device("cuda", 0)
    cache = TP.DecodeCache(1, batch, 8, 2, dev, page_size=4, dtype=dtype)
    step = TP.DecodeStep("bf16", 1, 1, 0, dev, SHAPE, residual=True, cache=cache)
    calls = recorded(step)
    g = torch.Generator().manual_seed(5)
    for t in range(4):
        calls.clear()
        step.run((torch.randn(batch * new, 1024, generator=g) * 0.5).to(BF).to(dev))
        q = calls[0][1][:, :1024].reshape(batch * new, 8, 128)
        (kc, vc, table, _), scales = cache.layers[0]
        want, _, tol = expected(q, kc, vc, scales.get("k_scale"), scales.get("v_scale"), table, [(t + 1) * new] * batch, [0, new, 2 * new])
        assert bool(((calls[1][0].view_as(q).double() - want).abs() <= tol).all()), t
    assert N.device_status() == 0


def test_a_refused_step_leaves_the_cache_alone():
    dev = torch.device("cuda", 0)
    cache = TP.DecodeCache(1, 2, 64, 2, dev)
    step = TP.DecodeStep("bf16", 1, 1, 0, dev, SHAPE, cache=cache)
    for x in (torch.zeros(2, 1000, dtype=BF, device=dev), torch.zeros(2, 1024, dtype=torch.float32, device=dev),
              torch.zeros(3, 1024, dtype=BF, device=dev)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            step.run(x)
        assert cache.kv_lens.tolist() == [0, 0]
    step.run(torch.zeros(2, 1024, dtype=BF, device=dev))
    assert cache.kv_lens.tolist() == [1, 1]


# ---------------------------------------------------------------------------------------------------------------------
# powers of two of e4m3 rows


def cached_row(cache, table, i, j):
    return int(table[i, j // cache.shape[2]]), j % cache.shape[2]


@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("new,length,late,window", [(70, 70, 65, 0), (70, 400, 395, 0), (90, 300, 215, 8), (300, 300, 131, 0), (1, 70, 40, 8)])
def test_rows_that_a_query_may_not_see_do_not_matter(new, length, late, window, which):
    """One token's rows are 2^30 larger than their neighbours'. Queries before it, or whose window lies behind it, never see it."""
    for qt, dim, page in ((BF, 128, 16), (HF, 64, 5)):
        q, cache, kw, starts = setup([new], [length], 8, 2, dim, page, qt, E4M3, seed=late)
        kc, vc, table, _ = cache
        pg, slot = cached_row(kc, table, 0, late)
        for n, s in (("k", kw["k_scale"]), ("v", kw["v_scale"])):
            if n in which:
                s.view(torch.uint8)[pg, :, slot] = 151
        compare(q, cache, kw, starts, [length], window=window, shared=7)


@pytest.mark.parametrize("qt", [BF, HF])
@pytest.mark.parametrize("spread", [0, 7, 8, 15, 16, 24, 40])
@pytest.mark.parametrize("new", [1, 70, 200])
def test_row_scales_of_any_spread(new, spread, qt):
    """Powers of two of neighbouring rows up to 2^spread apart: each query's error goes by what it sees, per element."""
    for dim, page, slots_last in ((128, 16, False), (64, 24, True)):
        q, cache, kw, starts = setup([new], [700], 8, 2, dim, page, qt, E4M3, seed=spread)
        g = torch.Generator().manual_seed(spread)
        for name in ("k_scale", "v_scale"):
            s = kw[name].view(torch.uint8)
            s.copy_(torch.randint(121 - spread, 122, s.shape, generator=g).to(torch.uint8))
            if slots_last:  # scale bytes that do not lie together
                kw[name] = s.transpose(1, 2).contiguous().transpose(1, 2).view(E8M0)
        compare(q, cache, kw, starts, [700], shared=7)


def test_rows_of_zeros_beside_others():
    """A row of zeros has the smallest power of two: its neighbours keep theirs, and its key keeps its weight."""
    for new in (1, 80):
        q, cache, kw, starts = setup([new], [300], 8, 1, 128, 16, BF, E4M3, seed=new)
        for c, s in ((cache[0], kw["k_scale"]), (cache[1], kw["v_scale"])):
            c.view(torch.uint8)[:, :, ::3] = 0
            s.view(torch.uint8)[:, :, ::3] = 27
        compare(q, cache, kw, starts, [300], shared=7)


@pytest.mark.parametrize("ct", [BF, E4M3])
@pytest.mark.parametrize("new", [3, 70])
def test_a_key_that_is_no_number_reaches_who_sees_it(new, ct):
    """A NaN among the keys: queries before it, or whose window lies behind it, keep their bits, the others are NaN."""
    for bad, window in ((298, 0), (300 - new, 2)):
        q, cache, kw, _ = setup([new], [300], 8, 2, 128, 16, BF, ct, seed=new, ragged=False)
        want, wl = L.paged_attention(q, *cache, window=window, return_lse=True, **kw)
        pg, slot = cached_row(cache[0], cache[2], 0, bad)
        cache[0][pg, 1, slot, 7] = math.nan
        out, lse = L.paged_attention(q, *cache, window=window, return_lse=True, **kw)
        pos = torch.arange(300 - new, 300, device="cuda")
        sees = (pos >= bad) & ((pos < bad + window) if window else True)
        assert torch.equal(out[:, :4], want[:, :4]) and torch.equal(lse[:, :4], wl[:, :4])  # the other kv head
        assert torch.equal(out[~sees], want[~sees]) and torch.equal(lse[~sees], wl[~sees])
        assert bool(out[sees][:, 4:].isnan().all()) and bool(lse[sees][:, 4:].isnan().all())


# ---------------------------------------------------------------------------------------------------------------------
# weights far below the largest


@pytest.mark.parametrize("strong", [0, 70000, 131071 - 70])
@pytest.mark.parametrize("ct", [HF, E4M3])
@pytest.mark.parametrize("new,batch", [(1, 600), (70, 150)])
def test_a_long_flat_tail_below_one_strong_key(new, batch, ct, strong):
    """131k keys 2^-25.3 below one, with values of 256: each alone rounds away beside a largest probability of 1, together they are
    as much as the strong key. As many sequences over the same pages as there are CTAs, so that one of them meets all of the keys."""
    n, page = 131072, 128
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(batch, 1)
    kc, vc = torch.zeros(2, n // page, 1, page, 64, device="cuda").unbind(0)
    kc[strong // page, 0, strong % page, 0] = 1.0
    vc[...] = -256.0
    vc[strong // page, 0, strong % page] = 1.0
    kw = dict(k_scale=None, v_scale=None)
    if ct == E4M3:
        kw = {k: torch.full((n // page, 1, page), 127, dtype=torch.uint8, device="cuda").view(E8M0) for k in kw}
    q = torch.zeros(batch * new, 1, 64, dtype=HF, device="cuda")
    q[:, 0, 0] = 25.3 * math.log(2.0)
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out = L.paged_attention(q, kc.to(ct), vc.to(ct), table, lens, scale=1.0, **kw).view(batch, new, 1, 64)
    want, _, tol = expected(q[:new], kc.to(ct), vc.to(ct), kw["k_scale"], kw["v_scale"], table, [n], [0, new], scale=1.0)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"error {err.max().item():.3e}, {(err / tol).max().item():.2f} of its bound"


# ---------------------------------------------------------------------------------------------------------------------
# scale bytes that kv_append never writes


@pytest.mark.parametrize("ot", [torch.float32, BF])
def test_read_of_the_smallest_and_largest_scale_bytes(ot):
    """value * 2^(byte - 127) from byte 0 to 254, NaN for byte 255."""
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    values = torch.arange(256, dtype=torch.uint8, device="cuda").view(E4M3)
    kc = values.view(1, 1, 1, 256).expand(1, 1, 16, 256).contiguous()
    byte = torch.tensor([0, 1, 2, 26, 27, 100, 127, 200, 246, 247, 253, 254, 255, 255, 0, 254], dtype=torch.uint8, device="cuda")
    ks = byte.view(1, 1, 16).view(E8M0)
    k, v = L.kv_read(kc, kc, table, torch.tensor([16], dtype=torch.int32, device="cuda"), 16, k_scale=ks, v_scale=ks, out_dtype=ot)
    want = values.double()[None] * torch.exp2(byte.double() - 127)[:, None]
    want[byte == 255] = math.nan
    want = want.float().to(ot)  # the product is exact in fp32 up to its largest value
    for x in (k, v):
        assert torch.equal(x[0, :, 0].isnan(), want.isnan()) and torch.equal(x[0, :, 0].nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_scale_byte_that_is_no_number(new, which):
    """255 is NaN: queries that see the row get NaN (the row sum only where it is a key's), others what they got without it."""
    length, late = 300, 299 if new == 1 else 290
    q, cache, kw, starts = setup([new], [length], 8, 2, 128, 16, BF, E4M3, seed=new)
    want, wl = L.paged_attention(q, *cache, return_lse=True, **kw)
    pg, slot = cached_row(cache[0], cache[2], 0, late)
    kw[which + "_scale"].view(torch.uint8)[pg, :, slot] = 255
    out, lse = L.paged_attention(q, *cache, return_lse=True, **kw)
    sees = torch.arange(length - new, length, device="cuda") >= late
    assert bool(out[sees].isnan().all())
    assert bool(out[~sees].isfinite().all())
    if which == "k":
        assert bool(lse[sees].isnan().all())
    else:
        assert bool(((lse - wl)[sees].abs() <= 2.0 ** -18 * (1 + wl[sees].abs() + 128)).all())
    # another reference power of two, but the values of each row are exact either way: a rounding of P and of the result each
    assert bool(((out.double() - want.double())[~sees].abs() <= 2.0 ** -7 * (want.double().abs() + 4.0)[~sees]).all())
    assert bool(((lse - wl)[~sees].abs() <= 2.0 ** -18 * (1 + wl[~sees].abs() + 128)).all())


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("k_byte,v_byte", [(0, 127), (127, 227), (127, 0), (0, 0)])
def test_attention_over_the_smallest_and_largest_scale_bytes(new, k_byte, v_byte):
    """Every row has the same extreme power of two."""
    q, cache, kw, starts = setup([new], [300], 8, 2, 128, 16, BF, E4M3, seed=9)
    kw["k_scale"].view(torch.uint8)[:] = k_byte
    kw["v_scale"].view(torch.uint8)[:] = v_byte
    out, lse = L.paged_attention(q, *cache, return_lse=True, **kw)
    want, wl, tol = expected(q, cache[0], cache[1], kw["k_scale"], kw["v_scale"], cache[2], [300], starts, shared=7)
    # rows of less than 2^-100 may count as zeros
    assert bool(((out.double() - want).abs() <= tol + 448 * 2.0 ** -100).all())
    assert bool(((lse.double() - wl).abs() <= 2.0 ** -18 * (1 + wl.abs() + 128)).all())


def test_large_queries_at_right_angles_to_large_keys():
    """Factors of a row of q and of a row of K beyond fp32 together: a product of zero stays zero."""
    for new in (1, 70):
        q, cache, kw, starts = setup([new], [300], 8, 2, 128, 16, BF, E4M3, seed=3)
        q.zero_()
        q[..., 0] = 2.0 ** 100
        cache[0].view(torch.uint8)[..., 0] = 0
        kw["k_scale"].view(torch.uint8)[:] = 230
        compare(q, cache, kw, starts, [300])


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("byte,alone", [(87, True), (87, False), (246, True), (246, False)])
def test_factors_at_both_ends_of_the_range(byte, alone, new):
    """Queries of 2^115 over keys of 2^-40, queries of 1 over keys as large as a saturated infinity: the one key with a score has all
    of the weight, and its score is the lse. `alone`: only that key's power of two is extreme."""
    q, cache, kw, _ = setup([new], [300], 8, 2, 128, 16, BF, E4M3, seed=byte, ragged=False)
    q.zero_()
    q[..., 0] = 2.0 ** 115 if byte == 87 else 1.0
    pg, slot = cached_row(cache[0], cache[2], 0, 17)
    cache[0].view(torch.uint8)[:] = 0
    cache[0][pg, :, slot, 0] = 448.0
    ks = kw["k_scale"].view(torch.uint8)
    if not alone:
        ks[:] = byte
    ks[pg, :, slot] = byte
    out, lse = L.paged_attention(q, *cache, return_lse=True, **kw)
    want = rows_of(cache[1], kw["v_scale"], cache[2], 0, 300)[17].repeat_interleave(4, 0).expand(new, 8, 128)
    # half a step of the result; a largest weight of 1 and a row sum of 1 are exact up to the exponential's 2^-21 and fp32's 2^-24 each
    assert bool(((out.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -20) * want.abs()).all())
    score = q[0, 0, 0].double() * 448 * 2.0 ** (byte - 127) / 128 ** 0.5
    assert bool(((lse.double() - score).abs() <= 2.0 ** -18 * score).all())


@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("v_byte", [121, 137, 151, 190])
@pytest.mark.parametrize("k_byte", [135, 151, 200])
def test_a_row_far_above_the_others_is_the_result_of_who_sees_it(k_byte, v_byte, new):
    """A key of a huge score whose value has a large power of two, too: neither drowns the other. Queries before it are their own."""
    length, late = 300, 300 - (new + 1) // 2
    q, cache, kw, starts = setup([new], [length], 8, 2, 128, 16, BF, E4M3, seed=k_byte, ragged=False)
    q[..., 0] = 8.0
    pg, slot = cached_row(cache[0], cache[2], 0, late)
    cache[0].view(torch.uint8)[pg, :, slot] = 0
    cache[0][pg, :, slot, 0] = 448.0
    kw["k_scale"].view(torch.uint8)[pg, :, slot], kw["v_scale"].view(torch.uint8)[pg, :, slot] = k_byte, v_byte
    out, lse = L.paged_attention(q, *cache, return_lse=True, **kw)
    want, wl, tol = expected(q, cache[0], cache[1], kw["k_scale"], kw["v_scale"], cache[2], [length], starts, shared=7)
    sees = torch.arange(length - new, length, device="cuda") >= late
    v = rows_of(cache[1], kw["v_scale"], cache[2], 0, length)[late].repeat_interleave(4, 0)
    score = 8.0 * 448 * 2.0 ** (k_byte - 127) / 128 ** 0.5  # 2^16 and more, the others' at most 2^10
    assert bool(((out.double() - v)[sees].abs() <= (2.0 ** -7 + 2.0 ** -20) * v.abs()).all())  # the result's and the one weight's rounding
    assert bool(((lse.double() - score)[sees].abs() <= 2.0 ** -18 * score).all())
    assert bool(((out.double() - want).abs() <= tol)[~sees].all())
    assert bool(((lse.double() - wl)[~sees].abs() <= 2.0 ** -18 * (1 + wl[~sees].abs() + 128)).all())


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("qt,ct,size", [(HF, HF, 8000.0), (BF, BF, 2.0 ** 20), (BF, BF, 2.0 ** 45), (BF, E4M3, 2.0 ** 45), (HF, E4M3, 2.0 ** 15)])
def test_scores_beyond_what_a_rounding_of_fp32_leaves(new, qt, ct, size):
    """Scores of 2^25 and far more, where the last bit of a product is worth powers of two: the largest still has all of the weight."""
    q, cache, kw, _ = setup([new], [300], 8, 2, 128, 16, qt, ct, seed=new, ragged=False)
    g = torch.Generator().manual_seed(31)
    q.copy_(size * (1 + 0.25 * torch.rand(q.shape, generator=g)))
    k = cache[0].view(torch.uint8) if ct == E4M3 else cache[0]
    j = torch.arange(300, device="cuda")
    pg, slot = cache[2][0].long()[j // 16], j % 16
    rows = -(1 + 0.25 * torch.rand(300, 2, 128, generator=g)).cuda()  # all far below
    rows[17] = 1 + 0.25 * torch.rand(2, 128, generator=g).cuda()
    if ct == E4M3:
        k[pg, :, slot] = (256 * rows).to(E4M3).view(torch.uint8)
        kw["k_scale"].view(torch.uint8)[:] = min(127 + int(math.log2(size)), 190)
    else:
        k[pg, :, slot] = (size * rows).to(ct)
    out, lse = L.paged_attention(q, *cache, return_lse=True, **kw)
    want = rows_of(cache[1], kw["v_scale"], cache[2], 0, 300)[17].repeat_interleave(4, 0).expand(new, 8, 128)
    key = rows_of(cache[0], kw["k_scale"], cache[2], 0, 300)[17].repeat_interleave(4, 0)
    half = torch.finfo(qt).eps / 2
    # half a step of the result and of the one weight, whose exponential is off by 2^-21
    assert bool(((out.double() - want).abs() <= (2 * half + 2.0 ** -20) * want.abs() + torch.finfo(qt).tiny).all())
    score = (q.double() * key).sum(-1) / 128 ** 0.5
    # 128 products and sums of one sign, the scale, log2 and back: 2^-24 each of the score
    assert bool(((lse.double() - score).abs() <= 136 * 2.0 ** -24 * score).all())


# ---------------------------------------------------------------------------------------------------------------------
# scratch


def test_scratch_stays_within_the_documented_bounds():
    """Of every row count, head dimension and type: 39.5 MB for many query rows, 7.5 MB for few, 47 MB for both, on 148 SMs."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    most = {}
    for dtype in (1, 4):
        for dim in (64, 128):
            for group in (1, 5, 8, 16, 24, 32):
                for new, starts in ((1, False), (2, False), (3, False), (4, False), (24, False), (32, False), (300, False), (1, True), (300, True)):
                    a = N.AttnArgs()
                    c = a.kv
                    c.k, c.v, c.k_scale, c.v_scale = 4096, 8192, *((4096, 4096) if dtype == 4 else (None, None))
                    c.k_stride = c.v_stride = (C.c_int64 * 3)(16 * dim, 16 * dim, dim)
                    c.page_table, c.table_stride, c.kv_lens, c.q_starts = 4096, 4096, 4096, 4096 if starts else None
                    c.dtype, c.pages, c.kv_heads, c.page_size, c.head_dim, c.table_width, c.batch = dtype, 64, 1, 16, dim, 4096, 64
                    c.tokens = 64 * new
                    a.q, a.out, a.q_dtype, a.heads, a.scale = 4096, 4096, 1, group, 0.1
                    a.q_stride = a.out_stride = (C.c_int64 * 2)(group * dim, dim)
                    need = N.lib.llg_paged_attention_ws(C.byref(a))
                    assert need > 0
                    kind = "both" if starts else "many" if new * group > 32 else "few" if new * group <= 24 else "either"
                    most[kind] = max(most.get(kind, 0), need)
    assert most["few"] <= 7.5e6 * sms / 148 and max(most["many"], most["either"]) <= 39.5e6 * sms / 148 and most["both"] <= 47e6 * sms / 148, most
    assert most["both"] > 39.5e6 * sms / 148  # the sum is reached
