"""Paged key/value cache and attention on the GPU against plain 64-bit implementations of the same formulas."""
import math

import pytest
import torch

import lowlat_gemm as L
from lowlat_gemm import _native as N

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BF, HF = torch.bfloat16, torch.float16


def pages_for(lens, page, seed, extra=3, width=None):
    """A page table whose pages lie anywhere in the cache; unused entries name no page at all."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=g).tolist()
    width = width or max(max(need), 1)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda(), total


def make_cache(pages, heads, page, dim, dtype, seed, slots_first=False):
    """Random cache rows; slots_first: stored [pages, page_size, heads, head_dim] and passed as a transposed view."""
    g = torch.Generator().manual_seed(seed)
    shape = (pages, page, heads, dim) if slots_first else (pages, heads, page, dim)
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        if dtype == E4M3:
            c = (x * 64).clamp(-448, 448).to(E4M3).cuda()
            s = torch.randint(118, 124, shape[:3], generator=g).to(torch.uint8).cuda().view(E8M0)
        else:
            c, s = x.to(dtype).cuda(), None
        if slots_first:
            c, s = c.transpose(1, 2), None if s is None else s.view(torch.uint8).transpose(1, 2).view(E8M0)
        out += [c, s]
    return out[0], out[2], out[1], out[3]


def rows_of(cache, scale, table, i, n):
    """float64 [n, heads, dim]: tokens 0..n of sequence i; pages that do not exist read as zeros."""
    pages, heads, page, dim = cache.shape
    j = torch.arange(n, device=cache.device)
    pg = table[i].long()[j // page]
    ok = (pg >= 0) & (pg < pages)
    x = cache.view(torch.uint8)[pg.clamp(0, pages - 1), :, j % page].view(cache.dtype).double() if cache.dtype == E4M3 \
        else cache[pg.clamp(0, pages - 1), :, j % page].double()
    if scale is not None:
        x = x * torch.exp2(scale.view(torch.uint8)[pg.clamp(0, pages - 1), :, j % page].double() - 127)[..., None]
    return torch.where(ok[:, None, None], x, 0.0)


def reference(q, kc, vc, ks, vs, table, lens, starts, scale, causal, window):
    """(o, lse, tolerance of o): float64, rows of no sequence are NaN."""
    tokens, heads, dim = q.shape
    group = heads // kc.shape[1]
    half = torch.finfo(q.dtype).eps / 2
    o = torch.full((tokens, heads, dim), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, heads), math.nan, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    for i, length in enumerate(lens):
        t0, t1 = starts[i], starts[i + 1]
        n = t1 - t0
        length = min(length, table.shape[1] * kc.shape[2])
        if n == 0:
            continue
        k, v = rows_of(kc, ks, table, i, length), rows_of(vc, vs, table, i, length)
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        qq = q[t0:t1].double()
        s = torch.einsum("thd,jhd->thj", qq, k) * scale
        pos = length - n + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        s = torch.where(seen[:, None], s, -math.inf)
        top = s.amax(-1, keepdim=True) if length else torch.full((n, heads, 1), -math.inf, dtype=torch.float64, device="cuda")
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        w = p / torch.where(total == 0, 1.0, total)
        o[t0:t1] = torch.einsum("thj,jhd->thd", w, v)
        lse[t0:t1] = (top + torch.log(total)).squeeze(-1)
        # one rounding of the result (half a step of |o|), one of each probability (half a step of the weighted |v|, the fp32
        # products and sums over keys 2^-24 each), and the error of a score - a dot product of dim fp32 products and sums,
        # 2^-24 each of sum |q||k| - which moves a weight by twice its size; exp2 adds 2^-21
        mass = torch.einsum("thj,jhd->thd", w, v.abs())
        score = (torch.einsum("thd,jhd->thj", qq.abs(), k.abs()) * abs(scale)).amax(-1, keepdim=True) if length else torch.zeros_like(top)
        delta = score * (dim + 4) * 2.0 ** -24 + 2.0 ** -21
        tol[t0:t1] = half * o[t0:t1].abs() + mass * (half + 2 * delta + length * 2.0 ** -24) + torch.finfo(q.dtype).tiny
    return o, lse, tol


def check(news, lens, heads, kvh, dim, page, qt, ct, *, causal=True, window=0, scale=None, seed=0, slots_first=False, ragged=None, tail=0,
          width=None, loud=1.0):
    table, pages = pages_for(lens, page, seed, width=width)
    kc, vc, ks, vs = make_cache(pages, kvh, page, dim, ct, seed + 1, slots_first)
    g = torch.Generator().manual_seed(seed + 2)
    tokens = sum(news) + tail
    # queries as the qkv projection leaves them: a strided view
    wide = (torch.randn(tokens, (heads + 2 * kvh) * dim, generator=g) * loud).to(qt).cuda()
    q = wide[:, :heads * dim].view(tokens, heads, dim)
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    ragged = (len(set(news)) > 1 or tail > 0) if ragged is None else ragged
    st = torch.tensor(starts, dtype=torch.int32, device="cuda") if ragged else None
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((tokens, heads, dim), 7.0, dtype=qt, device="cuda")
    got, lse = L.paged_attention(q, kc, vc, table, ln, q_starts=st, k_scale=ks, v_scale=vs, scale=scale, causal=causal, window=window,
                                 out=out, return_lse=True)
    assert got is out
    want, wl, tol = reference(q, kc, vc, ks, vs, table, lens, starts, dim ** -0.5 if scale is None else scale, causal, window)
    body = slice(0, sum(news))
    err = (out[body].double() - want[body]).abs()
    assert bool((err <= tol[body]).all()), f"error {err.max().item():.3e}, {(err / tol[body]).max().item():.2f} of its bound"
    fin = torch.isfinite(wl[body])
    assert torch.equal(fin, torch.isfinite(lse[body]))
    assert bool((lse[body][~fin] == -math.inf).all())
    # a score is off by its dot product's error (bounded by |lse| and dim here), the sum by 2^-21
    assert bool(((lse[body].double() - wl[body])[fin].abs() <= 2.0 ** -18 * (1 + wl[body][fin].abs() + loud * loud)).all())
    assert bool((out[sum(news):] == 7.0).all())
    assert N.device_status() == 0
    return out


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("qt", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kvh", [(8, 1), (8, 8), (5, 1), (32, 2), (32, 1), (14, 2)])
def test_one_token(heads, kvh, dim, qt, ct):
    check([1] * 5, [1, 17, 64, 65, 777], heads, kvh, dim, 16, qt, E4M3 if ct == "e4m3" else qt, seed=heads)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("page", [1, 3, 16, 48, 256])
def test_pages_end_anywhere(page, ct):
    check([1, 1, 1], [130, 1, 259], 8, 2, 128, page, BF, E4M3 if ct == "e4m3" else BF, seed=page)
    check([3, 3], [61, 200], 8, 2, 64, page, HF, E4M3 if ct == "e4m3" else HF, seed=page + 1)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("news,lens", [
    ([5] * 4, [5, 6, 300, 1000]), ([4, 1, 0, 7], [900, 33, 12, 7]), ([17], [400]), ([100, 1, 33], [100, 2000, 640]), ([257], [700]),
    ([129, 0, 1, 300], [129, 0, 513, 1500])])
def test_chunks(news, lens, ct):
    for qt, dim, heads, kvh in ((BF, 128, 16, 2), (HF, 64, 10, 2)):
        check(news, lens, heads, kvh, dim, 32, qt, E4M3 if ct == "e4m3" else qt, seed=len(news) + dim)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 200])
def test_sliding_window(window, ct):
    check([1, 1, 1], [500, 40, 64], 8, 2, 128, 16, BF, E4M3 if ct == "e4m3" else BF, window=window, seed=window)
    check([90, 3, 1], [190, 3, 400], 8, 2, 128, 16, BF, E4M3 if ct == "e4m3" else BF, window=window, seed=window)
    check([130], [300], 16, 1, 64, 16, HF, E4M3 if ct == "e4m3" else HF, window=window, causal=False, seed=window)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
def test_without_causal_mask(ct):
    check([40, 2], [100, 70], 8, 2, 128, 16, BF, E4M3 if ct == "e4m3" else BF, causal=False)


@pytest.mark.parametrize("news,lens", [([3, 2], [0, 1]), ([70, 1], [40, 0]), ([1], [0]), ([300], [10])])
def test_rows_that_see_nothing(news, lens):
    """Fewer cached tokens than new ones: the first queries stand before the first key."""
    for ct in (BF, E4M3):
        out = check(news, lens, 8, 2, 128, 16, BF, ct, width=4)
        at = 0
        for n, length in zip(news, lens):
            assert bool((out[at:at + max(0, n - length)] == 0).all())
            at += n


def test_rows_behind_the_last_sequence_stay():
    check([1, 2, 1], [50, 9, 130], 8, 2, 128, 16, BF, E4M3, tail=5)
    check([100, 2, 1], [150, 9, 130], 8, 2, 128, 16, BF, BF, tail=200)


def test_heads_behind_slots_and_wide_tables():
    for ct in (BF, E4M3):
        check([1, 1], [300, 77], 8, 4, 128, 16, BF, ct, slots_first=True, width=4000)
        check([150, 1], [300, 77], 8, 4, 128, 16, BF, ct, slots_first=True, width=4000)


def test_equal_counts_given_as_offsets_agree():
    a = check([2, 2, 2], [40, 300, 2], 8, 2, 128, 16, BF, E4M3, ragged=True)
    b = check([2, 2, 2], [40, 300, 2], 8, 2, 128, 16, BF, E4M3, ragged=False)
    assert torch.equal(a, b)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
def test_long_cache_few_heads(ct):
    """One sequence shared by every SM: many partial results per row."""
    check([1], [33333], 8, 1, 128, 64, BF, E4M3 if ct == "e4m3" else BF)
    check([9], [20001], 4, 1, 64, 64, HF, E4M3 if ct == "e4m3" else HF)
    check([40], [9000], 4, 1, 128, 64, BF, E4M3 if ct == "e4m3" else BF)


def test_many_sequences():
    lens = [(37 * i) % 311 + 1 for i in range(300)]
    check([1] * 300, lens, 4, 1, 64, 16, BF, BF)
    news = [(i % 5) if i % 7 else 40 for i in range(300)]
    check(news, [n + x for n, x in zip(news, lens)], 4, 1, 64, 16, BF, E4M3)


def test_large_scores_and_growing_maxima():
    """Scores of hundreds: one key takes all of the weight, the running maximum moves through the whole walk."""
    check([1, 1], [700, 5000], 8, 1, 128, 16, BF, BF, loud=30.0, scale=1.0)
    check([200], [700], 8, 1, 128, 16, HF, E4M3, loud=30.0, scale=0.7)


def test_smallest_and_largest_row_scales():
    """e4m3 rows whose powers of two span the range a bf16 model meets, subnormal e4m3 values among them."""
    table, pages = pages_for([200], 16, 5)
    kc, vc, ks, vs = make_cache(pages, 1, 16, 128, E4M3, 6)
    g = torch.Generator().manual_seed(7)
    kc.view(torch.uint8)[:, :, ::2] &= 0x87  # subnormal values only
    ks.view(torch.uint8)[:, :, ::2] = 130
    vs.view(torch.uint8).copy_(torch.randint(90, 160, vs.shape, generator=g).to(torch.uint8))
    q = torch.randn(1, 8, 128, generator=g).to(BF).cuda()
    out = L.paged_attention(q, kc, vc, table, torch.tensor([200], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)
    want, _, tol = reference(q, kc, vc, ks, vs, table, [200], [0, 1], 128 ** -0.5, True, 0)
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales_that_are_not_positive(scale, ct):
    for news, lens in (([1, 1], [70, 500]), ([90, 2], [300, 150])):
        check(news, lens, 8, 1, 128, 16, BF, E4M3 if ct == "e4m3" else BF, scale=scale)
        check(news, lens, 8, 2, 64, 16, HF, E4M3 if ct == "e4m3" else HF, scale=scale)


@pytest.mark.parametrize("loud", [0.0, 1e-30, 1e-12])
def test_queries_of_zeros_and_near_them(loud):
    """The factors of a bf16 row of q and of a quarter tile without rows are tiny together; masked keys stay masked."""
    for news, lens in (([1, 1], [70, 500]), ([90, 2], [301, 150]), ([40], [3001])):
        for ct in (BF, E4M3):
            check(news, lens, 8, 1, 128, 16, BF, ct, loud=loud)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("page", [8, 24, 40, 96])
def test_chunks_over_pages_of_any_size(page, ct):
    """Boxes of 8 and 32 rows, and pages that no box fits."""
    check([70, 1], [300, 90], 8, 2, 128, page, BF, E4M3 if ct == "e4m3" else BF, seed=page)
    check([33], [1500], 4, 1, 64, page, HF, E4M3 if ct == "e4m3" else HF, seed=page)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
def test_rows_between_the_kernels(ct):
    """9 to 32 query rows per kv head, uniform and ragged, and groups of 32."""
    for new in (2, 3, 4, 5):
        check([new] * 3, [30, 300, 1000], 8, 1, 128, 16, BF, E4M3 if ct == "e4m3" else BF, seed=new)
        check([new] * 3, [30, 300, 1000], 8, 1, 64, 16, HF, E4M3 if ct == "e4m3" else HF, ragged=True, seed=new)
    check([1, 5, 40], [100, 300, 90], 32, 1, 128, 16, BF, E4M3 if ct == "e4m3" else BF)
    check([2, 3], [100, 300], 48, 2, 128, 16, BF, E4M3 if ct == "e4m3" else BF)


def test_more_sequences_than_threads():
    news = [(i % 3) if i % 97 else 45 for i in range(700)]
    check(news, [n + (31 * i) % 157 for i, n in enumerate(news)], 8, 1, 64, 16, BF, BF)


def test_windows_wider_than_any_cache():
    for news, lens in (([5], [2]), ([90], [20]), ([1, 60], [300, 400])):
        for window in (2 ** 31 - 1, 2 ** 30, 2 ** 30 - 1):
            check(news, lens, 8, 1, 128, 16, BF, BF, window=window, width=32)


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("news,lens", [([1], [20000]), ([2, 70], [900, 9000]), ([40], [9000]), ([300, 1], [700, 40])])
def test_a_nan_query_stays_a_nan_and_alone(news, lens, ct):
    """Also where several CTAs share its sequence and no part has a maximum."""
    ct = E4M3 if ct == "e4m3" else BF
    table, pages = pages_for(lens, 16, 11)
    kc, vc, ks, vs = make_cache(pages, 1, 16, 128, ct, 12)
    g = torch.Generator().manual_seed(13)
    q = torch.randn(sum(news), 4, 128, generator=g).to(BF).cuda()
    starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, wl = L.paged_attention(q, kc, vc, table, ln, q_starts=starts, k_scale=ks, v_scale=vs, return_lse=True)
    bad = q.clone()
    bad[-1, 2, 5] = math.nan
    got, gl = L.paged_attention(bad, kc, vc, table, ln, q_starts=starts, k_scale=ks, v_scale=vs, return_lse=True)
    assert bool(got[-1, 2].isnan().all()) and bool(gl[-1, 2].isnan())
    want[-1, 2], wl[-1, 2] = got[-1, 2], gl[-1, 2]
    assert torch.equal(want.view(torch.int16), got.view(torch.int16)) and torch.equal(wl.view(torch.int32), gl.view(torch.int32))


@pytest.mark.parametrize("ct", ["same", "e4m3"])
def test_queries_of_other_sequences_stay_apart(ct):
    """Rows of the tile that belong to no token of it may hold anything: the next sequence's NaN, rows behind the last sequence."""
    ct = E4M3 if ct == "e4m3" else BF
    news, lens = [70, 3, 45], [300, 40, 2000]
    table, pages = pages_for(lens, 16, 51)
    kc, vc, ks, vs = make_cache(pages, 1, 16, 128, ct, 52)
    g = torch.Generator().manual_seed(53)
    q = torch.randn(sum(news) + 9, 8, 128, generator=g).to(BF).cuda()
    starts = torch.tensor([0, 70, 73, 118], dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = L.paged_attention(q, kc, vc, table, ln, q_starts=starts, k_scale=ks, v_scale=vs)
    bad = q.clone()
    bad[70:73], bad[118:] = math.nan, math.inf
    got = L.paged_attention(bad, kc, vc, table, ln, q_starts=starts, k_scale=ks, v_scale=vs)
    assert torch.equal(got[:70], want[:70]) and torch.equal(got[73:118], want[73:118]) and bool(got[70:73].isnan().all())


@pytest.mark.parametrize("ct", ["same", "e4m3"])
@pytest.mark.parametrize("news,lens", [([1, 1], [70, 500]), ([90, 2], [300, 150])])
def test_keys_and_values_in_one_allocation(news, lens, ct):
    """Strided views of one tensor, scale rows that are not contiguous, and a strided output: the same results."""
    ct = E4M3 if ct == "e4m3" else BF
    table, pages = pages_for(lens, 16, 21)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 128, ct, 22)
    both = torch.stack([kc.view(torch.uint8), vc.view(torch.uint8)], 1)
    kv = [both[:, i].view(ct) for i in range(2)]
    scales = [None, None]
    if ks is not None:
        s = torch.stack([ks.view(torch.uint8), vs.view(torch.uint8)], 3)
        scales = [s[..., i].view(E8M0) for i in range(2)]
    g = torch.Generator().manual_seed(23)
    q = torch.randn(sum(news), 8, 128, generator=g).to(BF).cuda()
    starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = L.paged_attention(q, kc, vc, table, ln, q_starts=starts, k_scale=ks, v_scale=vs)
    wide = torch.full((sum(news), 10, 128), 7.0, dtype=BF, device="cuda")
    L.paged_attention(q, *kv, table, ln, q_starts=starts, k_scale=scales[0], v_scale=scales[1], out=wide[:, 1:9])
    assert torch.equal(wide[:, 1:9], want) and bool((wide[:, ::9] == 7.0).all())


@pytest.mark.parametrize("qt", [BF, HF])
@pytest.mark.parametrize("new", [1, 70])
def test_row_scales_far_apart(new, qt):
    """Neighbouring rows whose powers of two differ by up to 2^16: the tile kernel keeps a row's value times 2^-d, d up to 16 below
    the quarter's largest, in f16, whose smallest step is 2^-24 - an error of 2^-25 of the quarter's power of two per element."""
    table, pages = pages_for([700], 16, 31)
    kc, vc, ks, vs = make_cache(pages, 1, 16, 128, E4M3, 32)
    g = torch.Generator().manual_seed(33)
    for s in (ks, vs):
        s.view(torch.uint8).copy_(torch.randint(108, 125, s.shape, generator=g).to(torch.uint8))
    q = torch.randn(new, 4, 128, generator=g).to(qt).cuda()
    out = L.paged_attention(q, kc, vc, table, torch.tensor([700], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)
    want, _, tol = reference(q, kc, vc, ks, vs, table, [700], [0, new], 128 ** -0.5, True, 0)
    # 2^-3 is the largest power (byte 124): a score is off by sum|q| 2^-28 / sqrt(128), which moves a weight by twice that; V by 2^-28
    shift = q.double().abs().sum(-1, keepdim=True) * 2.0 ** -28 / 128 ** 0.5
    v = rows_of(vc, vs, table, 0, 700).abs().amax()
    tol = tol + 2 * shift * v + 2.0 ** -28
    assert bool(((out.double() - want).abs() <= tol).all())


# ---------------------------------------------------------------------------------------------------------------------
# the cache itself


def plain_quantised(x):
    """(e4m3 values, exponents) of rows x by the definition, in float64."""
    x = x.double()
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 9 + (m > 0.875)).clamp(-100, 119), -100)
    return torch.ldexp(x, -e[..., None]).clamp(-448, 448).to(torch.float32).to(E4M3), e


def run_append(news, lens, kvh, dim, page, it, ct, *, ragged=None, tail=0, seed=0, slots_first=False, table=None, spread=1.0):
    auto, pages = pages_for(lens, page, seed)
    table = auto if table is None else table
    kc, vc, ks, vs = make_cache(pages, kvh, page, dim, ct, seed + 1, slots_first)
    before = [None if t is None else t.view(torch.uint8).clone() if t.dtype in (E4M3, E8M0) else t.clone() for t in (kc, vc, ks, vs)]
    g = torch.Generator().manual_seed(seed + 2)
    tokens = sum(news) + tail
    rows = torch.exp2(torch.randint(-20, 15, (tokens, 2 * kvh, 1), generator=g).float() * spread)
    kv = (torch.randn(tokens, 2 * kvh, dim, generator=g) * rows).to(it).cuda()
    if tokens > 2:
        kv[1, 0] = 0  # a row of zeros
    k, v = kv[:, :kvh], kv[:, kvh:]
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    ragged = (len(set(news)) > 1 or tail > 0) if ragged is None else ragged
    st = torch.tensor(starts, dtype=torch.int32, device="cuda") if ragged else None
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    L.kv_append(k, v, kc, vc, table, ln, q_starts=st, k_scale=ks, v_scale=vs)
    status = N.device_status()
    for x, cache, scale, was, swas in ((k, kc, ks, before[0], before[2]), (v, vc, vs, before[1], before[3])):
        want, wscale = was.clone(), None if swas is None else swas.clone()
        for i, n in enumerate(news):
            for j in range(n):
                pos = lens[i] - n + j
                if pos < 0 or pos // page >= table.shape[1]:
                    continue
                pg = int(table[i, pos // page])
                if not 0 <= pg < pages:
                    continue
                row = x[starts[i] + j]
                if ct == E4M3:
                    val, e = plain_quantised(row)
                    want[pg, :, pos % page] = val.view(torch.uint8)
                    wscale[pg, :, pos % page] = (e + 127).to(torch.uint8)
                else:
                    want[pg, :, pos % page] = row
        assert torch.equal(cache.view(torch.uint8) if ct == E4M3 else cache, want)
        if scale is not None:
            assert torch.equal(scale.view(torch.uint8), wscale)
    return status


@pytest.mark.parametrize("it,ct", [(BF, E4M3), (HF, E4M3), (torch.float32, E4M3), (BF, BF), (HF, HF)])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128, 256])
def test_append(dim, it, ct):
    assert run_append([1, 1, 1], [1, 40, 33], 3, dim, 16, it, ct) == 0
    assert run_append([4, 0, 9, 1], [4, 7, 100, 33], 2, dim, 16, it, ct, tail=3, seed=1) == 0
    assert run_append([37], [70], 1, dim, 5, it, ct, seed=2, slots_first=True) == 0


def test_append_extremes():
    """Rows of the largest and smallest floats: exponents end at 119 and -100, infinities saturate, NaN stays."""
    table, pages = pages_for([6], 16, 0)
    kc, vc, ks, vs = make_cache(pages, 1, 16, 16, E4M3, 1)
    k = torch.zeros(6, 1, 16, device="cuda")
    k[0, 0, 0], k[0, 0, 1] = 3.4e38, 1.0
    k[1, 0, 0] = 1e-40
    k[2, 0, 0], k[2, 0, 1] = math.inf, 1e38
    k[3, 0, 0], k[3, 0, 1] = math.nan, 2.0
    k[4, 0, 0], k[4, 0, 1] = 448.0, 2.0 ** -9
    k[5, 0, 0] = 448.0000305
    L.kv_append(k, k, kc, vc, table, torch.tensor([6], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)
    pg = int(table[0, 0])
    e = ks.view(torch.uint8)[pg, 0, :6].int().cpu() - 127
    assert e.tolist() == [119, -100, 119, -7, 0, 1]
    x = kc[pg, 0, :6].float().cpu()
    assert x[0, 0] == 448 and x[1, 0] == 0 and x[2, 0] == 448 and math.isnan(x[3, 0]) and x[3, 1] == 256 and x[4, 0] == 448
    assert x[4, 1] == 2.0 ** -9 and x[5, 0] == 224


def test_append_many_sequences_and_short_lengths():
    lens = [(13 * i) % 50 + 1 for i in range(1100)]
    assert run_append([1] * 1100, lens, 1, 64, 16, BF, BF, ragged=True) == 0
    # more new tokens than the length says: those before position 0 are not in the cache
    assert run_append([5, 3], [2, 20], 2, 64, 16, BF, E4M3, ragged=True) == 0


def test_pages_that_do_not_exist():
    """Entries that name no page: nothing is written there, they read as zeros, and the device status says so."""
    lens = [40, 40]
    table, pages = pages_for(lens, 16, 3)
    table[0, 2], table[1, 0] = pages, -5
    for ct in (BF, E4M3):
        assert run_append([20, 20], lens, 2, 64, 16, BF, ct, seed=3, table=table) == 32
        kc, vc, ks, vs = make_cache(pages, 2, 16, 64, ct, 1)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        k, v = L.kv_read(kc, vc, table, ln, 40, k_scale=ks, v_scale=vs)
        assert N.device_status() == 32
        assert bool((k[0, 32:] == 0).all()) and bool((v[1, :16] == 0).all()) and not bool((k[0, :32] == 0).all())
        for news in ([1, 1], [30, 30]):
            q = torch.randn(sum(news), 8, 64, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
            out = L.paged_attention(q, kc, vc, table, ln, k_scale=ks, v_scale=vs)
            assert N.device_status() == 32
            want, _, tol = reference(q, kc, vc, ks, vs, table, lens, [0, news[0], sum(news)], 64 ** -0.5, True, 0)
            assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("ot,ct", [(BF, E4M3), (HF, E4M3), (torch.float32, E4M3), (BF, BF), (HF, HF)])
@pytest.mark.parametrize("dim", [16, 80, 64, 128, 256])
def test_read(dim, ot, ct):
    lens = [33, 0, 1, 70]
    for page, slots_first in ((16, False), (7, True)):
        table, pages = pages_for(lens, page, 4)
        kc, vc, ks, vs = make_cache(pages, 3, page, dim, ct, 5, slots_first)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for most in (64, 1, 71):
            got = L.kv_read(kc, vc, table, ln, most, k_scale=ks, v_scale=vs, out_dtype=ot)
            for x, cache, scale in ((got[0], kc, ks), (got[1], vc, vs)):
                assert x.shape == (4, most, 3, dim) and x.dtype == ot
                for i, n in enumerate(lens):
                    n = min(n, most)
                    assert torch.equal(x[i, :n], rows_of(cache, scale, table, i, n).to(ot)), (dim, most, i)
                    assert bool((x[i, n:] == 0).all())
    assert N.device_status() == 0


def test_append_then_read_returns_the_values():
    """bf16 rows of four significant bits pass through an e4m3 cache unchanged."""
    table, pages = pages_for([50], 16, 0)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 64, E4M3, 1)
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(8, 16, (50, 2, 64), generator=g) * torch.exp2(torch.randint(-6, 6, (50, 2, 1), generator=g).float())).to(BF).cuda()
    ln = torch.tensor([50], dtype=torch.int32, device="cuda")
    L.kv_append(x, -x, kc, vc, table, ln, k_scale=ks, v_scale=vs)
    k, v = L.kv_read(kc, vc, table, ln, 50, k_scale=ks, v_scale=vs)
    assert torch.equal(k[0], x) and torch.equal(v[0], -x)


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, refusals


def test_captured_call_follows_lengths_and_page_tables():
    lens = [100, 5]
    table, pages = pages_for([400, 400], 16, 0)
    for ct in (BF, E4M3):
        kc, vc, ks, vs = make_cache(pages, 2, 16, 128, ct, 1)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        kv = torch.randn(2, 2, 2, 128, device="cuda").to(BF)
        q = torch.randn(2, 8, 128, device="cuda").to(BF)
        out = torch.empty_like(q)

        def step():
            L.kv_append(kv[:, 0], kv[:, 1], kc, vc, table, ln, k_scale=ks, v_scale=vs)
            L.paged_attention(q, kc, vc, table, ln, k_scale=ks, v_scale=vs, out=out)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for now in ([101, 6], [399, 1], [64, 128]):
            ln.copy_(torch.tensor(now, dtype=torch.int32))
            kv.normal_()
            q.normal_()
            out.zero_()
            graph.replay()
            want, _, tol = reference(q, kc, vc, ks, vs, table, now, [0, 1, 2], 128 ** -0.5, True, 0)
            assert bool(((out.double() - want).abs() <= tol).all())


def test_two_graphs_and_two_streams_share_nothing():
    lens = [3000, 2500, 2000]
    table, pages = pages_for(lens, 16, 0)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 128, E4M3, 1)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = [torch.randn(3, 16, 128, device="cuda").to(BF), torch.randn(90, 16, 128, device="cuda").to(BF)]
    want = [L.paged_attention(q, kc, vc, table, ln, k_scale=ks, v_scale=vs) for q in qs]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(L.paged_attention(q, kc, vc, table, ln, k_scale=ks, v_scale=vs))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    eager = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            eager.append(L.paged_attention(qs[i % 2], kc, vc, table, ln, k_scale=ks, v_scale=vs))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], want[i])  # the order of every sum is fixed: same bits
    for i, e in enumerate(eager):
        assert torch.equal(e, want[i % 2])


def test_with_programmatic_dependent_launch():
    """The whole chain - projection, append, attention, projection - with early launches gives the bits it gives without."""
    heads, kvh, dim, hidden = 8, 1, 128, 1024
    lens = [70, 300, 9]
    table, pages = pages_for([n + 8 for n in lens], 16, 0)
    g = torch.Generator().manual_seed(3)
    w_qkv = (torch.randn((heads + 2 * kvh) * dim, hidden, generator=g) * 0.05).to(BF).cuda()
    w_o = (torch.randn(hidden, heads * dim, generator=g) * 0.05).to(BF).cuda()
    x0 = torch.randn(3, hidden, generator=g).to(BF).cuda()

    def steps():
        kc, vc, ks, vs = make_cache(pages, kvh, 16, dim, E4M3, 1)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        x = x0
        for _ in range(4):
            ln += 1
            qkv = L.gemm(x, w_qkv)
            q, k, v = (t.view(3, -1, dim) for t in qkv.split([heads * dim, kvh * dim, kvh * dim], dim=1))
            L.kv_append(k, v, kc, vc, table, ln, k_scale=ks, v_scale=vs)
            y = L.paged_attention(q, kc, vc, table, ln, k_scale=ks, v_scale=vs)
            x = L.gemm(y.view(3, -1), w_o)
        return x, kc.view(torch.uint8).clone()

    want = steps()
    L.set_pdl(True)
    try:
        got = steps()
        torch.cuda.synchronize()
    finally:
        L.set_pdl(False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert N.device_status() == 0


def test_empty_calls():
    table = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    ln = torch.zeros(0, dtype=torch.int32, device="cuda")
    kc = torch.zeros(2, 2, 16, 128, dtype=BF, device="cuda")
    q = torch.zeros(0, 8, 128, dtype=BF, device="cuda")
    assert L.paged_attention(q, kc, kc, table, ln).shape == (0, 8, 128)
    L.kv_append(q[:, :2], q[:, :2], kc, kc, table, ln)
    assert L.kv_read(kc, kc, table, ln, 5)[0].shape == (0, 5, 2, 128)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    none = torch.zeros(1, 0, dtype=torch.int32, device="cuda")
    out = L.paged_attention(torch.ones(1, 8, 128, dtype=BF, device="cuda"), kc, kc, none, one)
    assert bool((out == 0).all())
    assert bool((L.kv_read(kc, kc, none, one, 3)[0] == 0).all())


def test_refusals():
    kc = torch.zeros(4, 2, 16, 128, dtype=BF, device="cuda")
    f8 = kc.to(E4M3)
    sc = torch.zeros(4, 2, 16, dtype=torch.uint8, device="cuda").view(E8M0)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    ln = torch.ones(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(3, 8, 128, dtype=BF, device="cuda")
    k = q[:, :2]

    def refused(text, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=text):
            fn(*args, **kw)

    att, app, rd = L.paged_attention, L.kv_append, L.kv_read
    refused("k_scale is needed", att, q, f8, f8, table, ln)
    refused("v_scale is needed", att, q, f8, f8, table, ln, k_scale=sc)
    refused("k_scale belongs", att, q, kc, kc, table, ln, k_scale=sc, v_scale=sc)
    refused("must be a float8_e8m0fnu", att, q, f8, f8, table, ln, k_scale=sc[:3], v_scale=sc)
    refused("a 16-bit cache must have q's type", att, q.half(), kc, kc, table, ln)
    refused("q must be bf16 or f16", att, q.float(), f8, f8, table, ln, k_scale=sc, v_scale=sc)
    refused("1 to 32 times", att, q[:, :7], kc, kc, table, ln)
    refused("1 to 32 times", att, torch.zeros(3, 66, 128, dtype=BF, device="cuda"), kc, kc, table, ln)
    refused("head_dim must be 64 or 128", att, q[:, :, :96], kc[..., :96], kc[..., :96], table, ln)
    refused("q has head_dim", att, q[:, :, :64], kc, kc, table, ln)
    refused("multiple of the 3 sequences", att, torch.cat([q, q[:1]]), kc, kc, table, ln)
    refused("q_starts must be", att, q, kc, kc, table, ln, q_starts=ln)
    refused("page_table must be int32", att, q, kc, kc, table.long(), ln)
    refused("page_table must be int32", att, q, kc, kc, table[:2], ln)
    refused("kv_lens must be", att, q, kc, kc, table, ln.long())
    refused("window", att, q, kc, kc, table, ln, window=-1)
    refused("one shape", att, q, kc, kc[:3], table, ln)
    refused("16-byte aligned", att, torch.zeros(3, 8, 132, dtype=BF, device="cuda")[..., 4:], kc, kc, table, ln)
    refused("cache rows must be 16-byte aligned", att, q, torch.zeros(4, 2, 16, 132, dtype=BF, device="cuda")[..., :128],
            torch.zeros(4, 2, 16, 132, dtype=BF, device="cuda")[..., :128], table, ln)
    refused("out must have q's type", att, q, kc, kc, table, ln, out=q.half())
    refused("takes keys and values of its own type", app, k.half(), k.half(), kc, kc, table, ln)
    refused("the cache holds", app, q, q, kc, kc, table, ln)
    refused("bfloat16, float16 or float32", app, k.to(E4M3), k.to(E4M3), f8, f8, table, ln, k_scale=sc, v_scale=sc)
    refused("16-bit cache's type", rd, kc, kc, table, ln, 4, out_dtype=HF)
    refused("must be on", att, q, kc, kc, table.cpu(), ln)
    refused("must be on", app, k.cpu(), k, kc, kc, table, ln)
    with pytest.raises(ValueError, match="max_len"):
        rd(kc, kc, table, ln, -1)
    refused("must both be bfloat16", att, q, kc.float(), kc.float(), table, ln)
    assert N.device_status() == 0


@pytest.mark.parametrize("ct", [BF, E4M3])
def test_offsets_beyond_32_bits(ct):
    """Pages more than 4 GiB into the cache: the same bits as from a small one."""
    heads, page, dim = 2, 64, 128
    row = dim * ct.itemsize
    pages = (5 << 30) // (heads * page * row)
    far = torch.tensor([[pages - 1, pages - 5, pages - 2], [pages - 4, 1, pages - 3]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([150, 131], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(41)
    kv = torch.randn(2 * 131, 2 * heads, dim, generator=g).to(BF).cuda()
    q = torch.randn(2 * 131, 8, dim, generator=g).to(BF).cuda()
    results = []
    for table, n in ((near, 6), (far, pages)):
        kc, vc = (torch.zeros if n == 6 else torch.empty)((2, n, heads, page, dim), dtype=ct, device="cuda").unbind(0)
        scales = {}
        if ct == E4M3:
            ks, vs = torch.empty(2, n, heads, page, dtype=torch.uint8, device="cuda").view(E8M0).unbind(0)
            scales = dict(k_scale=ks, v_scale=vs)
        first = torch.full((2,), 19, dtype=torch.int32, device="cuda")  # then 131 new ones reach lengths of 150 and 131
        L.kv_append(kv[:38, :heads], kv[:38, heads:], kc, vc, table, first, **scales)
        L.kv_append(kv[:, :heads], kv[:, heads:], kc, vc, table, lens, **scales)
        results.append([L.paged_attention(q, kc, vc, table, lens, **scales), L.paged_attention(q[:2], kc, vc, table, lens, **scales),
                        *L.kv_read(kc, vc, table, lens, 150, **scales)])
        del kc, vc, scales
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert N.device_status() == 0
