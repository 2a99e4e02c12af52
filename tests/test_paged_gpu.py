"""GPU parity of the paged cache's operators against their definitions in float64
(oracle/paged.py).

Tolerances, from the number formats: the result is rounded once to its type, by at most 2^-8 of
it in bf16, 2^-11 in fp16 and nothing in fp32, and a weight enters the product with the values
as one fp16 number (2^-11 of it) or as two bf16 numbers (less than 2^-16): u_p + u_out with
u = 2^-9 for bf16 and 2^-11 for fp16 covers both, and what one bf16 number per weight would lose
(2^-8) it does not. Scores are fp32 sums of exact 16-bit products: with sum |q k| scale <= 64
and at most 16 chained additions their error is below 64 * 16 * 2^-23 = 1.3e-4, which is also
the relative error of a weight and, with the sum of exponentials, the absolute one of the
logarithm: SCORE = 2^-12 covers both.
    |out - ref| <= (u_p + u_out + SCORE) sum p |v|,  |lse - ref| <= SCORE,
    |mass - ref| <= 2 SCORE * weight + 2^-22 mass.
Everything else (append, select, move) is exact.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu
SCORE = 2.0 ** -12
UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11, torch.float32: 0.0}


def _np(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def make(seed, lengths, h, kv, d, page, dtype, device, *, width=None, nhd=False, stale=float("nan"), spare=3):
    """A cache whose sequences' pages are scattered over the pool, with `stale` in every row that
    belongs to no sequence, and ids outside the pool in the table's unused places."""
    from pseudobrain_b200.paged_cache import PagedCache
    g = torch.Generator(device="cpu").manual_seed(seed)
    b = len(lengths)
    used = [-(-n // page) for n in lengths]
    m = max(max(used), 1) + 1 if width is None else width
    pool = sum(used) + spare
    ids = torch.randperm(pool, generator=g)
    table = torch.full((b, m), -7, dtype=torch.int32)
    table[:, ::2] = 2 ** 30
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = ids[at:at + n].to(torch.int32)
        at += n
    shape = (pool, page, kv, d) if nhd else (pool, kv, page, d)
    kp, vp = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if nhd:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    mass = torch.rand(pool, kv, page, generator=g)
    pos = torch.randint(0, 1 << 20, (pool, kv, page), generator=g, dtype=torch.int32)
    dead = torch.ones(pool, page, dtype=torch.bool)
    for i, n in enumerate(lengths):
        e = torch.arange(n)
        dead[table[i, e // page].long(), e % page] = False
    kp.masked_fill_(dead[:, None, :, None], stale)
    vp.masked_fill_(dead[:, None, :, None], stale)
    q = torch.randn(b, h, d, generator=g).to(dtype)
    dev = lambda t: t.to(device)  # noqa: E731
    if nhd:
        kp, vp = (dev(t.transpose(1, 2).contiguous()).transpose(1, 2) for t in (kp, vp))
    cache = PagedCache(dev(kp), dev(vp), dev(mass), dev(pos))
    return cache, dev(table), dev(torch.tensor(lengths, dtype=torch.int32)), dev(q)


def used_table(table, lengths, page):
    t = _np(table).copy()
    for i, n in enumerate(lengths):
        t[i, -(-n // page):] = 0
    return t


def check_attend(cache, table, lengths, q, out, lse, before, window=None, sinks=0, scale=None, accumulate=False):
    lens = _np(lengths)
    page = cache.page
    t = used_table(table, lens, page)
    kp, vp = _np(cache.k_pages), _np(cache.v_pages)
    ref, ref_lse, weights = op.attend(_np(q), kp, vp, t, lens, window, sinks, scale)
    big, _, _ = op.attend(_np(q), kp, np.abs(vp), t, lens, window, sinks, scale)
    tol = (UNIT[cache.k_pages.dtype] + UNIT[out.dtype] + SCORE) * big + 1e-30
    err = np.abs(_np(out) - ref)
    assert np.isfinite(_np(out)).all() and (err <= tol).all(), float((err / tol).max())
    empty = np.isinf(ref_lse)
    assert (np.isneginf(_np(lse)) == empty).all()
    assert (np.abs(_np(lse)[~empty] - ref_lse[~empty]) <= SCORE).all()
    want, slack = before.copy(), np.zeros_like(before)
    if accumulate:
        for i, w in enumerate(weights):
            p, r = op.entry(t, page, i, np.arange(w.shape[1]))
            for h in range(w.shape[0]):
                want[p, h, r] += w[h]
                slack[p, h, r] += 2 * SCORE * w[h] + 2.0 ** -22 * want[p, h, r]
    got = _np(cache.mass)
    assert (np.abs(got - want) <= slack).all()


CASES = [
    # lengths, h, kv, d, page, window, sinks
    ([1], 8, 2, 128, 16, None, 0),
    ([2, 1, 0, 3], 4, 4, 64, 8, None, 0),
    ([15, 16, 17, 31, 32, 33], 32, 8, 128, 16, None, 0),
    ([517], 32, 8, 128, 16, None, 0),
    ([1000, 1, 0, 255, 64], 24, 4, 256, 64, None, 0),
    ([300, 7], 5, 5, 128, 32, None, 0),              # one query head per key head
    ([129, 513], 17, 1, 64, 128, None, 0),           # 17 query rows: more than two tiles of eight
    ([700], 64, 1, 128, 16, None, 0),                # 64 query heads on one key head
    ([100], 66, 2, 256, 8, None, 0),                 # 33 rows
    ([5000, 2500], 10, 2, 128, 256, None, 0),
    ([1000, 50, 4, 0, 131], 32, 8, 128, 16, 64, 4),  # window and sinks, shorter and longer sequences
    ([1000, 333], 24, 4, 256, 8, 1, 0),              # the new token alone
    ([1000, 40, 77], 12, 3, 64, 32, 50, 33),         # sinks that end inside a tile; that meet the window
    ([640, 90], 8, 1, 128, 16, 96, 600),             # sinks past most of the sequence
    ([333], 8, 8, 128, 16, 4096, 4),                 # a window wider than the cache
    ([3] * 300, 4, 2, 64, 8, None, 0),               # many short sequences
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attend_matches_definition(cuda_device, case, dtype):
    from pseudobrain_b200.paged_cache import paged_attend
    lengths, h, kv, d, page, window, sinks = CASES[case]
    cache, table, lens, q = make(case, lengths, h, kv, d, page, dtype, cuda_device)
    before = _np(cache.mass)
    out, lse = paged_attend(cache, q, table, lens, window, sinks)
    assert out.dtype == dtype and out.shape == q.shape and lse.dtype == torch.float32
    check_attend(cache, table, lens, q, out, lse, before, window, sinks)
    again = paged_attend(cache, q, table, lens, window, sinks, accumulate=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])  # the sums' order is fixed
    check_attend(cache, table, lens, q, *again, before, window, sinks, accumulate=True)


def test_attend_fp32_output_scale_and_strides(cuda_device):
    """Entry-major pools, queries as a slice of a packed projection, a wider strided table, out
    into a slice of a larger fp32 buffer, a scale of the caller's."""
    from pseudobrain_b200.paged_cache import paged_attend
    lengths = [400, 0, 77]
    cache, table, lens, q = make(3, lengths, 12, 4, 128, 16, torch.bfloat16, cuda_device, nhd=True)
    packed = torch.zeros(3, 20, 128, dtype=torch.bfloat16, device=cuda_device)
    packed[:, 5:17] = q
    wide = torch.full((3, table.shape[1] + 9), -1, dtype=torch.int32, device=cuda_device)
    wide[:, : table.shape[1]] = table
    buf = torch.full((3, 16, 128), 7.0, device=cuda_device)
    out, lse = paged_attend(cache, packed[:, 5:17], wide[:, : table.shape[1]], lens, scale=0.21, out=buf[:, 2:14])
    check_attend(cache, table, lens, q, out, lse, _np(cache.mass), scale=0.21)
    assert bool((buf[:, :2] == 7).all()) and bool((buf[:, 14:] == 7).all())


def test_attend_values_interleaved_with_keys(cuda_device):
    """k_pages and v_pages as halves of one [P, 2, KV, page, hd] pool."""
    from pseudobrain_b200.paged_cache import PagedCache, paged_attend
    cache, table, lens, q = make(5, [260, 31], 8, 2, 64, 16, torch.float16, cuda_device)
    both = torch.stack((cache.k_pages, cache.v_pages), 1)
    halves = PagedCache(both[:, 0], both[:, 1], cache.mass, cache.pos)
    a, b = paged_attend(cache, q, table, lens), paged_attend(halves, q, table, lens)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attend_sharp_and_flat_rows(cuda_device):
    """Scores that rise along the entries (the running maximum changes in every tile), and one
    entry that outweighs 20000 others by 2^20 each: in fp16 too, the light ones' share survives."""
    from pseudobrain_b200.paged_cache import paged_attend
    for dtype in (torch.bfloat16, torch.float16):
        cache, table, lens, q = make(9, [3000], 8, 2, 128, 16, dtype, cuda_device)
        ramp = torch.zeros_like(cache.k_pages)
        t = table[0, : -(-3000 // 16)].long()
        ramp[t] = (torch.arange(t.numel() * 16, device=cuda_device).view(-1, 1, 16, 1) / 3000 * 3).to(dtype)
        cache.k_pages.copy_(torch.where(cache.k_pages.isnan(), cache.k_pages, ramp + 0.01 * cache.k_pages))
        q.abs_()
        out, lse = paged_attend(cache, q, table, lens, scale=0.02)
        check_attend(cache, table, lens, q, out, lse, _np(cache.mass), scale=0.02)
        n = 20001
        cache, table, lens, q = make(10, [n], 1, 1, 64, 64, dtype, cuda_device)
        cache.k_pages.copy_(torch.where(cache.k_pages.isnan(), cache.k_pages, torch.zeros_like(cache.k_pages)))
        q.fill_(1.0)
        cache.k_pages[table[0, 0].long(), 0, 0] = 1.0  # entry 0 scores 64 * scale
        cache.v_pages.copy_(torch.where(cache.v_pages.isnan(), cache.v_pages, torch.ones_like(cache.v_pages)))
        cache.v_pages[table[0, 0].long(), 0, 0] = 0.0  # the result is the light entries' share
        scale = 20 * np.log(2.0) / 64
        out, _ = paged_attend(cache, q, table, lens, scale=scale, out=torch.empty(1, 1, 64, device=cuda_device))
        share = (n - 1) * 2.0 ** -20 / (1 + (n - 1) * 2.0 ** -20)
        # every light weight rounds alike (u); its value 2^-20 is a power of two up to the exponent's error
        assert abs(float(out[0, 0, 0]) / share - 1) < UNIT[dtype] + SCORE


def test_attend_infinite_scores(cuda_device):
    """Keys that score -inf have no weight; a NaN query gives NaN and leaves the others alone."""
    from pseudobrain_b200.paged_cache import paged_attend
    cache, table, lens, q = make(11, [70, 70], 4, 1, 64, 16, torch.bfloat16, cuda_device)
    q.abs_()
    for e in (0, 17, 69):
        cache.k_pages[table[0, e // 16].long(), 0, e % 16] = -float("inf")
    q[1, 2, 5] = float("nan")
    out, lse = paged_attend(cache, q, table, lens)
    keep = [e for e in range(70) if e not in (0, 17, 69)]
    k = torch.stack([cache.k_pages[table[0, e // 16].long(), 0, e % 16] for e in keep]).double()
    v = torch.stack([cache.v_pages[table[0, e // 16].long(), 0, e % 16] for e in keep]).double()
    p = torch.softmax(q[0].double() @ k.T / 8, -1)
    tol = (2 * UNIT[torch.bfloat16] + SCORE) * (p @ v.abs())
    assert bool(((out[0].double() - p @ v).abs() <= tol).all())
    assert bool(out[1, 2].isnan().all()) and bool(lse[1, 2].isnan())
    assert bool(out[1, [0, 1, 3]].isfinite().all()) and bool(lse[1, [0, 1, 3]].isfinite().all())


def test_attend_lengths_and_page_ids_out_of_range(cuda_device):
    """A negative length is 0, one above the table's capacity is the capacity; entries on a page
    id outside the pool read as zeros and take no mass."""
    from pseudobrain_b200.paged_cache import paged_attend
    cache, table, lens, q = make(13, [48, 48, 48], 4, 2, 128, 16, torch.bfloat16, cuda_device, width=3)
    want = paged_attend(cache, q, table, lens)
    lens2 = torch.tensor([-5, 1 << 30, 48], dtype=torch.int32, device=cuda_device)
    out, lse = paged_attend(cache, q, table, lens2)
    assert bool((out[0] == 0).all()) and bool(lse[0].isneginf().all())
    assert torch.equal(out[1:], want[0][1:]) and torch.equal(lse[1:], want[1][1:])
    bad = table.clone()
    bad[2, 1] = 1 << 30
    before = _np(cache.mass)
    out, lse = paged_attend(cache, q, bad, lens, accumulate=True)
    zero = cache.k_pages.clone()
    zeros = _np(zero)
    vals = _np(cache.v_pages)
    page = int(table[2, 1])
    zeros[page], vals[page] = 0, 0
    ref, ref_lse, w = op.attend(_np(q), zeros, vals, _np(table), [48, 48, 48])
    big = op.attend(_np(q), zeros, np.abs(vals), _np(table), [48, 48, 48])[0]
    assert (np.abs(_np(out) - ref) <= (2 * UNIT[torch.bfloat16] + SCORE) * big).all()
    assert (np.abs(_np(lse) - ref_lse) <= SCORE).all()
    assert (_np(cache.mass)[page] == before[page]).all()


def test_attend_shared_pages_other_stream_and_graph(cuda_device):
    """Two sequences over the same pages; a call on a stream of its own; a captured graph whose
    replays follow the lengths."""
    from pseudobrain_b200.paged_cache import paged_append_, paged_attend
    cache, table, lens, q = make(15, [200, 200], 8, 2, 128, 16, torch.bfloat16, cuda_device)
    shared = table.clone()
    shared[1] = table[0]
    lens2 = torch.tensor([200, 90], dtype=torch.int32, device=cuda_device)
    out, lse = paged_attend(cache, q, shared, lens2)
    check_attend(cache, shared, lens2, q, out, lse, _np(cache.mass))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2, lse2 = paged_attend(cache, q, shared, lens2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    k = torch.randn(2, 2, 128, device=cuda_device).to(torch.bfloat16)
    n = lens.clone()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            paged_append_(cache, k, k, table, n)
            n += 1
            out3, lse3 = paged_attend(cache, q, table, n)
    torch.cuda.synchronize()
    for _ in range(3):
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check_attend(cache, table, n, q, out3, lse3, _np(cache.mass))
    assert n.tolist() == [203, 203]


def test_long_cache_past_32_bit_offsets(cuda_device):
    """A pool whose byte and element offsets pass 2^32: pages spread over 4.3e9 elements."""
    from pseudobrain_b200.paged_cache import (PagedCache, move_entries_, paged_append_, paged_attend, paged_observe_)
    page, d, n = 16, 64, 300
    pages = 65
    stride = (2 ** 32 + 2 ** 20) // pages // 8 * 8
    big = torch.empty(2, stride * pages, dtype=torch.bfloat16, device=cuda_device)
    kp, vp = (t.as_strided((pages, 1, page, d), (stride, page * d, d, 1)) for t in (big[0], big[1]))
    g = torch.Generator(device=cuda_device).manual_seed(4)
    for t in (kp, vp):
        t.copy_(torch.randn(pages, 1, page, d, generator=g, device=cuda_device))
    cache = PagedCache(kp, vp, torch.zeros(pages, 1, page, device=cuda_device),
                       torch.zeros(pages, 1, page, dtype=torch.int32, device=cuda_device))
    table = torch.arange(pages - 1, pages - 21, -1, dtype=torch.int32, device=cuda_device)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    q = torch.randn(1, 4, d, generator=g, device=cuda_device).to(torch.bfloat16)
    small = PagedCache(kp.contiguous(), vp.contiguous(), cache.mass.clone(), cache.pos.clone())
    k = torch.randn(1, 1, d, generator=g, device=cuda_device).to(torch.bfloat16)
    src, dst = (torch.tensor([[[x]]], dtype=torch.int32, device=cuda_device) for x in (299, 0))
    got = []
    for c in (cache, small):
        paged_append_(c, k, k, table, lens)
        move_entries_(c, table, src, dst, torch.ones(1, 1, dtype=torch.int32, device=cuda_device))
        out = paged_attend(c, q, table, lens + 1, accumulate=True)
        paged_observe_(c, q[:, None], table, lens + 1)
        got.append((*out, c.mass, c.k_pages.contiguous(), c.v_pages.contiguous()))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert bool((got[0][3][pages - 1, 0, 0] == got[0][3][int(table[0, 18]), 0, 11]).all())


OBSERVE = [
    # lengths, w, h, kv, d, page
    ([1], 1, 4, 2, 64, 8),
    ([40, 3, 0, 16, 17], 16, 12, 12, 64, 16),   # shorter than the queries, empty
    ([700, 129], 32, 32, 8, 128, 16),           # 128 rows per key head
    ([300, 301], 20, 24, 4, 256, 64),           # 120 rows
    ([513, 100], 7, 5, 1, 128, 32),             # 35 rows
    ([1030], 64, 24, 1, 128, 8),                # 1536 rows
    ([257, 256, 255], 3, 64, 1, 64, 128),
    ([2000], 33, 8, 2, 256, 16),                # 132 rows
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(OBSERVE)))
def test_observe_matches_definition(cuda_device, case, dtype):
    from pseudobrain_b200.paged_cache import paged_observe_
    lengths, w, h, kv, d, page = OBSERVE[case]
    cache, table, lens, _ = make(50 + case, lengths, h, kv, d, page, dtype, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(case)
    q = torch.randn(len(lengths), h, w, d, generator=g, device=cuda_device).to(dtype).transpose(1, 2)
    before = _np(cache.mass)
    start = cache.mass.clone()
    paged_observe_(cache, q, table, lens)
    t = used_table(table, lengths, page)
    want, slack = before.copy(), np.zeros_like(before)
    for i, add in enumerate(op.observe(_np(q), _np(cache.k_pages), t, lengths)):
        p, r = op.entry(t, page, i, np.arange(add.shape[1]))
        for j in range(kv):
            want[p, j, r] += add[j]
            slack[p, j, r] += 2 * SCORE * add[j] + 2.0 ** -22 * want[p, j, r]
    assert (np.abs(_np(cache.mass) - want) <= slack).all()
    first = cache.mass.clone()
    cache.mass.copy_(start)
    paged_observe_(cache, q, table, lens)
    assert torch.equal(cache.mass, first)


def test_observe_of_one_query_is_attend(cuda_device):
    from pseudobrain_b200.paged_cache import paged_attend, paged_observe_
    cache, table, lens, q = make(70, [400, 23], 16, 2, 128, 16, torch.bfloat16, cuda_device)
    cache.mass.zero_()
    paged_attend(cache, q, table, lens, accumulate=True)
    a = cache.mass.clone()
    cache.mass.zero_()
    paged_observe_(cache, q[:, None], table, lens)
    assert bool(((cache.mass - a).abs() <= 4 * SCORE * a).all())
    assert abs(float(a.double().sum()) - 2 * 16) < 32 * SCORE  # the weights of a row sum to one


@pytest.mark.parametrize("kv,d,page,dtype,counts,lengths,nhd", [
    (2, 128, 16, torch.bfloat16, [1, 1, 1], [0, 15, 16], False),
    (1, 64, 8, torch.float16, [9, 0, 1, 30], [7, 3, 0, 8], False),
    (4, 256, 64, torch.bfloat16, [100, 65], [63, 1], True),
    (3, 128, 32, torch.bfloat16, [0, 0], [4, 4], False),
    (2, 64, 16, torch.float16, [40, 5], [30, 0], False),  # the first passes the table's capacity
])
def test_append_is_exact(cuda_device, kv, d, page, dtype, counts, lengths, nhd):
    from pseudobrain_b200.paged_cache import paged_append_
    after = [n + c for n, c in zip(lengths, counts)]
    cap = 48 if counts == [40, 5] else None
    cache, table, lens, _ = make(20 + kv + d, [min(n, cap or n) for n in after], kv, kv, d, page, dtype, cuda_device,
                                 nhd=nhd, stale=5.0, width=None if cap is None else cap // page)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    seen = lens + 1000
    packed = torch.randn(sum(counts), 3 * kv, d, device=cuda_device).to(dtype)
    k, v = packed[:, :kv], packed[:, kv:2 * kv]
    cu = torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device=cuda_device)
    pools = [_np(x).copy() for x in (cache.k_pages, cache.v_pages, cache.mass, cache.pos)]
    op.append(pools, _np(table), lengths, _np(seen), _np(k), _np(v), counts)
    one = all(c == 1 for c in counts)
    paged_append_(cache, k, v, table, lens, seen, None if one else cu)
    for got, want in zip((cache.k_pages, cache.v_pages, cache.mass, cache.pos), pools):
        assert np.array_equal(_np(got), want)


def test_append_without_mass_and_with_page_ids_outside_the_pool(cuda_device):
    from pseudobrain_b200.paged_cache import PagedCache, paged_append_
    k_pages = torch.zeros(4, 1, 8, 64, dtype=torch.bfloat16, device=cuda_device)
    cache = PagedCache(k_pages, torch.zeros_like(k_pages))
    table = torch.tensor([[3, 1 << 30], [-1, 2]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([7, 6], dtype=torch.int32, device=cuda_device)
    k = torch.arange(1, 7, device=cuda_device, dtype=torch.bfloat16)[:, None, None].expand(6, 1, 64).contiguous()
    paged_append_(cache, k, k, table, lens, cu_seqlens=torch.tensor([0, 2, 6], dtype=torch.int32, device=cuda_device))
    want = torch.zeros_like(k_pages)
    want[3, 0, 7] = 1
    want[2, 0, 0], want[2, 0, 1] = 5, 6
    assert torch.equal(cache.k_pages, want) and torch.equal(cache.v_pages, want)


def _select_cache(mass, pos, page, seed, device):
    """Pools that hold mass / pos [B, KV, n] through a scattered table."""
    from pseudobrain_b200.paged_cache import PagedCache
    b, kv, n = mass.shape
    m = -(-n // page)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(b * m + 2, generator=g)[: b * m].view(b, m).to(torch.int32)
    mp = torch.full((b * m + 2, kv, page), 9e9)
    pp = torch.full((b * m + 2, kv, page), 1 << 30, dtype=torch.int32)
    e = torch.arange(n)
    for i in range(b):
        mp[table[i, e // page].long(), :, e % page] = mass[i].T
        pp[table[i, e // page].long(), :, e % page] = pos[i].T
    return PagedCache(None, None, mp.to(device), pp.to(device)), table.to(device)


@pytest.mark.parametrize("n,lengths,kv,page,budget,recent,sinks,levels", [
    (200, [200, 64, 65, 0], 2, 8, 64, 8, 4, 0),
    (5000, [5000, 4097], 3, 16, 4096, 100, 4, 0),
    (3000, [3000], 2, 64, 16, 0, 0, 0),
    (4112, [4112, 4100, 4096], 2, 16, 4096, 256, 4, 7),   # seven different masses: ties everywhere
    (33000, [33000, 20001], 1, 128, 1000, 500, 500, 3),   # every place protected
    (1024, [1024] * 5, 1, 32, 1, 0, 1, 0),
    (70000, [70000], 4, 16, 8192, 512, 4, 0),
    (131, [131], 1, 8, 130, 3, 0, 1),
    (64, [64, 10], 2, 8, 100, 3, 2, 1),                   # nothing to do: no moves at all
])
def test_select_matches_sorting(cuda_device, n, lengths, kv, page, budget, recent, sinks, levels):
    from pseudobrain_b200.paged_cache import select_evictions
    rng = np.random.default_rng(n + budget)
    b = len(lengths)
    mass = rng.random((b, kv, n)).astype(np.float32) ** 8 if not levels else \
        rng.integers(0, levels, (b, kv, n)).astype(np.float32) - 1
    pos = np.argsort(rng.random((b, kv, n)), -1).astype(np.int32)
    if n == 5000:  # what a sum of weights never is, ordered all the same
        mass[0, 0, ::7], mass[0, 1, ::11], mass[0, 2, ::3], mass[0, 0, 5::50] = np.nan, np.inf, -np.inf, -0.0
    seen = np.asarray(lengths, np.int32) + 3
    cache, table = _select_cache(torch.from_numpy(mass), torch.from_numpy(pos), page, n, cuda_device)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    src, dst, count = select_evictions(cache, table, dev(lengths), dev(seen), budget, recent, sinks)
    moves = max(0, min(budget, table.shape[1] * page - budget))
    assert src.shape == dst.shape == (b, kv, moves) and count.shape == (b, kv)
    t = _np(table)
    for i, row in enumerate(op.select(_np(cache.mass).astype(np.float32), _np(cache.pos), t, lengths, seen, budget,
                                      recent, sinks)):
        for j, (s, d) in enumerate(row):
            assert int(count[i, j]) == len(s) == len(d)
            pad = [-1] * (moves - len(s))
            assert src[i, j].tolist() == s + pad and dst[i, j].tolist() == d + pad


@pytest.mark.parametrize("kv,d,page,dtype,nhd", [(2, 128, 16, torch.bfloat16, False), (1, 64, 8, torch.float16, True),
                                                 (3, 256, 32, torch.bfloat16, False)])
def test_evict_keeps_what_the_choice_says(cuda_device, kv, d, page, dtype, nhd):
    """paged_evict_ moves the kept entries and touches nothing else; the attention over what is
    left is that over the kept entries."""
    from pseudobrain_b200.paged_cache import paged_attend, paged_evict_
    lengths, budget, recent, sinks = [900, 128, 130, 5, 0], 128, 16, 4
    cache, table, lens, q = make(80 + d, lengths, 4 * kv, kv, d, page, dtype, cuda_device, nhd=nhd, stale=3.0)
    rng = np.random.default_rng(d)
    for i, n in enumerate(lengths):  # positions of their own
        p, r = op.entry(_np(table), page, i, np.arange(n))
        for j in range(kv):
            cache.pos[torch.from_numpy(p).long(), j, torch.from_numpy(r).long()] = torch.from_numpy(
                rng.permutation(n).astype(np.int32)).to(cuda_device)
    t = used_table(table, lengths, page)
    pools = [_np(x).copy() for x in (cache.k_pages, cache.v_pages, cache.mass, cache.pos)]
    for i, row in enumerate(op.select(pools[2].astype(np.float32), pools[3], t, lengths, lengths, budget, recent, sinks)):
        for j, (s, e) in enumerate(row):
            for a, z in zip(s, e):
                (pa, ra), (pz, rz) = op.entry(t, page, i, a), op.entry(t, page, i, z)
                for x in pools:
                    x[pz, j, rz] = x[pa, j, ra]
    paged_evict_(cache, table, lens, lens, budget, recent, sinks)
    for got, want in zip((cache.k_pages, cache.v_pages, cache.mass, cache.pos), pools):
        assert np.array_equal(_np(got), want)
    lens.clamp_(max=budget)
    out, lse = paged_attend(cache, q, table, lens)
    check_attend(cache, table, lens, q, out, lse, pools[2])


def test_a_bounded_cache_over_many_tokens(cuda_device):
    """Prompt, observation, then decoding with an eviction every page: the cache stays within its
    budget plus a page, keeps the sinks and the recent tokens, and each step's result is the
    attention over what is kept."""
    from pseudobrain_b200.paged_cache import (PagedCache, paged_append_, paged_attend, paged_evict_, paged_observe_)
    kv, h, d, page, budget, recent, sinks, prompt = 2, 8, 64, 8, 64, 16, 4, 150
    g = torch.Generator(device=cuda_device).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda_device).to(torch.bfloat16)  # noqa: E731
    cache = PagedCache.allocate(25, kv, page, d, device=cuda_device)
    cache.k_pages.fill_(float("nan"))
    cache.v_pages.fill_(float("nan"))
    table = torch.randperm(25, generator=torch.Generator().manual_seed(2)).to(torch.int32)[None, :20].to(cuda_device)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    seen = lens.clone()
    paged_append_(cache, rnd(prompt, kv, d), rnd(prompt, kv, d), table, lens, seen,
                  torch.tensor([0, prompt], dtype=torch.int32, device=cuda_device))
    lens += prompt
    seen += prompt
    paged_observe_(cache, rnd(1, 16, h, d), table, lens)
    paged_evict_(cache, table, lens, seen, budget, recent, sinks)
    lens.clamp_(max=budget)
    for step in range(30):
        paged_append_(cache, rnd(1, kv, d), rnd(1, kv, d), table, lens, seen)
        lens += 1
        seen += 1
        before = _np(cache.mass)
        q = rnd(1, h, d)
        out, lse = paged_attend(cache, q, table, lens, accumulate=True)
        check_attend(cache, table, lens, q, out, lse, before, accumulate=True)
        if step % page == page - 1:
            paged_evict_(cache, table, lens, seen, budget, recent, sinks)
            lens.clamp_(max=budget)
    n, last = int(lens[0]), int(seen[0])
    assert n <= budget + page and last == prompt + 30
    for j in range(kv):
        pos = set(op.entries(_np(cache.pos), _np(table), 0, j, n).tolist())
        assert len(pos) == n and set(range(sinks)) <= pos and set(range(last - recent, last)) <= pos


def test_refusals(cuda_device):
    from pseudobrain_b200 import _capi
    from pseudobrain_b200 import paged_cache as P
    cache, table, lens, q = make(90, [20, 3], 4, 2, 64, 16, torch.bfloat16, cuda_device)
    z = torch.zeros
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.PagedCache(z(2, 1, 8, 64), z(2, 1, 8, 64))
    with pytest.raises(TypeError, match="bf16 or fp16"):
        P.PagedCache(z(2, 1, 8, 64, device=cuda_device), z(2, 1, 8, 64, device=cuda_device))
    with pytest.raises(ValueError, match="alike"):
        P.PagedCache(cache.k_pages, cache.v_pages[:1])
    with pytest.raises(ValueError, match="mass"):
        P.PagedCache(cache.k_pages, cache.v_pages, cache.mass.double())
    with pytest.raises(ValueError, match="no mass"):
        P.paged_attend(P.PagedCache(cache.k_pages, cache.v_pages), q, table, lens, accumulate=True)
    with pytest.raises(ValueError, match="block_table"):
        P.paged_attend(cache, q, table.long(), lens)
    with pytest.raises(ValueError, match="lengths"):
        P.paged_attend(cache, q, table, lens[:1])
    with pytest.raises(ValueError, match="q:"):
        P.paged_attend(cache, q.float(), table, lens)
    with pytest.raises(ValueError, match="window"):
        P.paged_attend(cache, q, table, lens, window=0)
    with pytest.raises(_capi.PbkError, match="invalid argument"):
        P.paged_attend(cache, q, table, lens, window=4, sinks=-1)
    with pytest.raises(_capi.PbkError, match="unsupported shape"):
        P.paged_attend(cache, q[:, :3], table, lens)       # 3 query heads over 2 key heads
    with pytest.raises(_capi.PbkError, match="unsupported shape"):
        P.paged_attend(cache, z(2, 130, 64, device=cuda_device, dtype=torch.bfloat16), table, lens)
    with pytest.raises(_capi.PbkError, match="misaligned"):
        P.paged_attend(cache, z(2, 4 * 64 + 1, device=cuda_device, dtype=torch.bfloat16)[:, 1:].unflatten(1, (4, 64)),
                       table, lens)
    odd = [z(3, 1, 12, 64, device=cuda_device, dtype=torch.bfloat16) for _ in range(2)]
    with pytest.raises(_capi.PbkError, match="unsupported shape"):
        P.paged_attend(P.PagedCache(*odd), q[:, :1], table, lens)  # pages of 12
    wide = [z(3, 1, 16, 96, device=cuda_device, dtype=torch.bfloat16) for _ in range(2)]
    with pytest.raises(_capi.PbkError, match="unsupported shape"):
        P.paged_attend(P.PagedCache(*wide), z(2, 1, 96, device=cuda_device, dtype=torch.bfloat16), table, lens)
    with pytest.raises(ValueError, match="cu_seqlens"):
        P.paged_append_(cache, q[:1, :2].contiguous(), q[:1, :2].contiguous(), table, lens)
    with pytest.raises(ValueError, match="recent"):
        P.select_evictions(cache, table, lens, lens, 8, recent=8, sinks=1)
    with pytest.raises(ValueError, match="no pos"):
        P.select_evictions(P.PagedCache(cache.k_pages, cache.v_pages, cache.mass), table, lens, lens, 8)
    src = z(2, 2, 1, dtype=torch.int32, device=cuda_device)
    with pytest.raises(ValueError, match="dst must be"):
        P.move_entries_(cache, table, src, src.long(), z(2, 2, dtype=torch.int32, device=cuda_device))
    many = z(1, 1025, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    with pytest.raises(_capi.PbkError, match="unsupported shape"):
        P.paged_observe_(cache, many, table[:1], lens[:1])
    # nothing to do is no error
    none = z(0, dtype=torch.int32, device=cuda_device)
    out, lse = P.paged_attend(cache, q[:0], table[:0], none)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    P.paged_observe_(cache, many[:, :0], table[:1], lens[:1])
    assert _capi.device_error() == 0


def test_example_keeps_its_budget_and_agrees_where_nothing_leaves(cuda_device):
    """The example: with a budget that holds everything the bounded stream is the whole one's (the
    weights change no result), with a smaller one the cache stays within it plus a page."""
    from examples.bounded_decode import main
    common = ["--batch", "2", "--prompt", "90", "--tokens", "20", "--layers", "2", "--hidden", "256", "--heads", "4",
              "--kv", "2", "--observe", "8", "--recent", "8"]
    same = main(common + ["--budget", "112"])
    assert same["bounded"] == same["whole"] == 110 and max(abs(d) for d in same["drift"]) < 1e-5
    small = main(common + ["--budget", "48"])
    assert 48 <= small["bounded"] <= 48 + 16


@pytest.mark.parametrize("batch", [2, 200])
def test_a_pool_without_pages_and_a_table_without_columns(cuda_device, batch):
    """Nothing to read is no error: attention gives zeros, the other calls do nothing."""
    from pseudobrain_b200 import paged_cache as P
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda_device)  # noqa: E731
    q = torch.ones(batch, 4, 64, dtype=torch.bfloat16, device=cuda_device)
    for pages, width in ((0, 3), (5, 0)):
        cache = P.PagedCache.allocate(pages, 2, 16, 64, device=cuda_device)
        table, lens = i32(batch, width), i32(batch) + 40
        for accumulate in (False, True):
            out, lse = P.paged_attend(cache, q, table, lens, accumulate=accumulate)
            assert bool((out == 0).all()) and bool(lse.isneginf().all())
        P.paged_append_(cache, q[:, :2].contiguous(), q[:, :2].contiguous(), table, lens)
        P.paged_observe_(cache, q[:, None], table, lens)
        P.paged_evict_(cache, table, lens, lens, 8)
        src, dst, count = P.select_evictions(cache, table, lens, lens, 8)
        assert bool((count == 0).all()) and bool((src == -1).all()) and bool((dst == -1).all())
        assert bool((cache.mass == 0).all())


@pytest.mark.parametrize("d,h", [(64, 4), (128, 4), (128, 16), (256, 6)])
def test_attend_long_runs_do_not_lose_their_sum(cuda_device, d, h):
    """1200 sequences over the same 131072 entries, so that a warp walks some 8192 units of a head:
    with values of 1 the result is 1. The weights in two bf16 numbers are within 2^-16; each unit's
    addition rounds by at most 2^-24 of the sum so far, either way, which in 8192 steps is
    2^-24 sqrt(8192 / 3) / sqrt(3) at one standard deviation, 1.1e-5 < 2^-16 at six."""
    from pseudobrain_b200.paged_cache import PagedCache, paged_attend
    n, page, b = 131072, 64, 1200
    g = torch.Generator(device=cuda_device).manual_seed(d + h)
    k = torch.randn(n // page, 1, page, d, generator=g, device=cuda_device).to(torch.bfloat16)
    cache = PagedCache(k, torch.ones_like(k))
    table = torch.arange(n // page, dtype=torch.int32, device=cuda_device)[None].expand(b, -1)
    lens = torch.full((b,), n, dtype=torch.int32, device=cuda_device)
    q = torch.randn(b, h, d, generator=g, device=cuda_device).to(torch.bfloat16)
    out, _ = paged_attend(cache, q, table, lens, out=torch.empty(b, h, d, device=cuda_device))
    assert float((out - 1).abs().max()) <= 2.0 ** -15


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,h,d", [(1, 1, 64), (1, 12, 128), (2, 5, 256), (300, 1, 64), (300, 12, 256), (300, 33, 128)])
def test_attend_weights_have_both_their_16_bit_numbers(cuda_device, b, h, d, dtype):
    """Entry e scores -4 e / d exactly and its value is 1 at place e, so out[e] is its weight. In
    fp32 arithmetic the exponent errs by less than 6 (2^-24 + 2^-25) + 14 * 2^-24 < 1.4e-6, the
    weight by ln 2 of that and 2^-22 for the power, their sum by as much again and the division by
    2^-23: less than 2^-18 in all. Held in two numbers, a weight has 2^-16 (bf16) or 2^-22 (fp16)."""
    from pseudobrain_b200.paged_cache import PagedCache, paged_attend
    page = 16
    e = torch.arange(d, device=cuda_device)
    k = (-e.float())[:, None].expand(d, d).to(dtype).view(d // page, 1, page, d).contiguous()
    v = torch.eye(d, device=cuda_device, dtype=dtype).view(d // page, 1, page, d)
    table = torch.arange(d // page, dtype=torch.int32, device=cuda_device)[None].expand(b, -1)
    lens = torch.full((b,), d, dtype=torch.int32, device=cuda_device)
    q = torch.ones(b, h, d, dtype=dtype, device=cuda_device)
    out, lse = paged_attend(PagedCache(k, v), q, table, lens, scale=4 / d ** 2, out=torch.empty(b, h, d, device=cuda_device))
    x = -4 * e.double() / d
    want = torch.softmax(x, -1)
    assert float((out.double() / want - 1).abs().max()) <= (2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -22) + 2.0 ** -18
    assert float((lse.double() - torch.logsumexp(x, -1)).abs().max()) <= 2.0 ** -18


def spread(seed, count, top, *first):
    """`count` lengths: those given, then some from 0 to `top`."""
    return (list(first) + np.random.default_rng(seed).integers(0, top + 1, count).tolist())[:count]


RUNS = [
    # lengths, h, kv, d, page, window, sinks: more units than a warp's ring holds, heads cut over runs
    (spread(1, 40, 3000, 3000, 0, 1, 0), 32, 8, 64, 16, None, 0),     # joined by runs (1280 query heads, 1184 runs)
    (spread(2, 30, 1500, 1500, 0, 699, 700, 701, 740), 40, 8, 128, 8, 700, 37),    # window and sinks over runs
    (spread(3, 40, 600, 600, 17), 24, 4, 256, 64, None, 0),           # 960 query heads, 888 runs
    (spread(4, 30, 1500, 1400, 3), 96, 8, 64, 32, 260, 600),          # sinks up to the window
    (spread(5, 160, 2000, 2000, 0, 16), 2, 1, 128, 32, None, 0),      # joined by heads on 256 threads
    (spread(6, 160, 900, 900, 0, 16), 10, 1, 256, 8, 300, 4),         # the same, 10 rows, a window
    ([30000], 4, 1, 256, 16, None, 0),                                # by heads on 1024 threads
    ([60001], 12, 1, 64, 128, 31000, 100),
    ([0, 41003, 5], 8, 2, 128, 8, None, 0),
    (spread(7, 12, 9000, 9000, 0), 40, 2, 64, 16, None, 0),           # two row tiles of ten
    (spread(8, 12, 4000, 4000), 66, 2, 128, 256, 2000, 33),           # three row tiles
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(RUNS)))
def test_attend_by_equal_runs(cuda_device, case, dtype):
    """The path of ragged batches and of long sequences. A workspace without weights to add says that
    a call takes it (clusters need none)."""
    from pseudobrain_b200 import _capi
    from pseudobrain_b200 import paged_cache as P
    lengths, h, kv, d, page, window, sinks = RUNS[case]
    cache, table, lens, q = make(200 + case, lengths, h, kv, d, page, dtype, cuda_device)
    desc = _capi.PbkPagedAttendDesc(h, window or 0, sinks, 0, 0.1, _capi.PBK_F32, 16, d, d, 16, d, d, 16)
    assert P.LIB.pbk_paged_attend_workspace(cache._ref, P._batch(cache, table, lens), desc) > 0
    before = _np(cache.mass)
    out, lse = P.paged_attend(cache, q, table, lens, window, sinks)
    check_attend(cache, table, lens, q, out, lse, before, window, sinks)
    again = P.paged_attend(cache, q, table, lens, window, sinks, accumulate=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    check_attend(cache, table, lens, q, *again, before, window, sinks, accumulate=True)
    assert _capi.device_error() == 0


OBSERVE_RUNS = [
    # lengths, w, h, kv, d, page, tiles per CTA: more key tiles per CTA than two turns of its ring
    ([23000, 17003, 0, 12011, 7189], 32, 32, 8, 64, 8, 25),                 # 128 rows, long heads
    (spread(21, 61, 2100, 2100, 1, 0, 19), 20, 24, 4, 128, 16, 13),         # 120 rows, heads of 0 to 17 tiles
    ([30011, 3, 27000, 5000], 5, 6, 2, 256, 256, 6),                        # 15 rows
    (spread(22, 700, 300, 300, 0, 1, 0), 7, 12, 4, 64, 16, 25),             # many heads of one to three tiles
    ([60000, 45003, 20], 40, 16, 2, 64, 64, 11),                            # 3 row tiles
    (spread(23, 70, 2000, 2000, 0, 49, 50, 51), 50, 12, 2, 128, 16, 7),     # 3 row tiles, a sequence as long as the queries
    (spread(24, 40, 3900, 3900, 63, 0), 64, 6, 1, 256, 32, 4),              # 4 row tiles, one stage of keys
    (spread(25, 30, 4000, 4000), 70, 24, 1, 64, 16, 3),                     # 14 row tiles: two launches a pass
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(OBSERVE_RUNS)))
def test_observe_over_many_key_tiles(cuda_device, case, dtype):
    """The pipeline at work: rings and accumulators in their second turns, runs over several heads and
    sequences, heads over several runs."""
    from pseudobrain_b200 import _capi
    from pseudobrain_b200.paged_cache import paged_observe_
    lengths, w, h, kv, d, page, each = OBSERVE_RUNS[case]
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    assert kv * sum(-(-n // 128) for n in lengths) > (each - 1) * sms
    cache, table, lens, _ = make(300 + case, lengths, h, kv, d, page, dtype, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(case)
    q = torch.randn(len(lengths), w, h, d, generator=g, device=cuda_device).to(dtype)
    start, before = cache.mass.clone(), _np(cache.mass)
    paged_observe_(cache, q, table, lens)
    t = used_table(table, lengths, page)
    want, slack = before.copy(), np.zeros_like(before)
    for i, add in enumerate(op.observe(_np(q), _np(cache.k_pages), t, lengths)):
        p, r = op.entry(t, page, i, np.arange(add.shape[1]))
        for j in range(kv):
            want[p, j, r] += add[j]
            slack[p, j, r] += 2 * SCORE * add[j] + 2.0 ** -22 * want[p, j, r]
    assert (np.abs(_np(cache.mass) - want) <= slack).all()
    first = cache.mass.clone()
    cache.mass.copy_(start)
    paged_observe_(cache, q, table, lens)
    assert torch.equal(cache.mass, first) and _capi.device_error() == 0


def choose(mass, pos, seen, budget, recent, sinks):
    """The moves (src, dst) of one row of n entries, by sorting."""
    n = len(mass)
    safe = ((pos >= 0) & (pos < sinks)) | (pos.astype(np.int64) >= seen - recent)
    nan = np.isnan(mass) & ~safe
    value = np.where(safe | nan, np.float32(0), mass)
    order = np.lexsort((np.arange(n), -value, ~nan, ~safe))
    kept = np.zeros(n, bool)
    kept[order[:budget]] = True
    at = np.arange(n)
    return at[kept & (at >= budget)], at[~kept & (at < budget)]


@pytest.mark.parametrize("lengths,kv,page,budget,recent,sinks,kind,width", [
    ([131072], 8, 16, 4096, 512, 4, "weights", None),                     # 16 CTAs of 512 threads
    ([131072], 2, 64, 130000, 3, 0, "near", None),                        # all three digits count
    ([131072, 4097, 70001, 4096, 0], 3, 16, 4096, 512, 4, "five", None),  # ties, shorter than the shares
    (spread(31, 25, 20000, 20000, 4099), 8, 16, 4096, 64, 4, "near", None),      # one CTA of 512 threads each
    (spread(32, 25, 30000, 30000, 9000), 8, 32, 9000, 64, 4, "weights", None),   # clusters of two
    ([24576, 24000], 80, 8, 12000, 0, 0, "five", None),                   # the longest share that is kept
    ([24577, 100, 24576], 60, 8, 24000, 9, 9, "odd", None),
    ([400003, 393217, 100], 2, 128, 4096, 512, 4, "weights", None),       # keys read again in every pass
    ([400003, 25000], 1, 8, 300000, 0, 7, "five", None),
    ([600001, 30], 2, 256, 100000, 1000, 4, "near", 1 << 15),             # a table of 2^23 entries
    ([1 << 23], 1, 256, 1 << 20, 1 << 19, 4, "odd", None),                # the most that a row may hold
])
def test_select_of_long_rows_matches_sorting(cuda_device, lengths, kv, page, budget, recent, sinks, kind, width):
    """Shares of over 4608 entries (512 threads) and of over 24576 (not kept in shared memory)."""
    from pseudobrain_b200 import _capi
    from pseudobrain_b200.paged_cache import PagedCache, select_evictions
    rng = np.random.default_rng(sum(lengths) + budget)
    n, b = max(lengths), len(lengths)
    m = -(-n // page)
    mass = {"weights": lambda: rng.random((b, kv, m * page), np.float32) ** 8 * 50,
            "near": lambda: (1 + rng.integers(0, 3000, (b, kv, m * page)) * 2.0 ** -23).astype(np.float32),
            "five": lambda: rng.integers(-1, 4, (b, kv, m * page)).astype(np.float32),
            "odd": lambda: rng.standard_normal((b, kv, m * page), np.float32)}[kind]()
    if kind == "odd":
        mass[..., ::97], mass[..., 5::101], mass[..., 7::103], mass[..., 11::89] = np.nan, np.inf, -np.inf, -0.0
    pos = rng.permuted(np.broadcast_to(np.arange(m * page, dtype=np.int32), mass.shape), axis=-1)
    seen = np.asarray(lengths, np.int64) + 3
    table = rng.permutation(b * m).reshape(b, m).astype(np.int32)
    pools = [torch.zeros(b * m, kv, page, dtype=dt, device=cuda_device) for dt in (torch.float32, torch.int32)]
    t = torch.from_numpy(table).long().to(cuda_device)
    for pool, x in zip(pools, (mass, pos)):
        pool[t] = torch.from_numpy(x).to(cuda_device).view(b, kv, m, page).transpose(1, 2)
    wide = torch.full((b, width or m), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :m] = t
    dev = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=cuda_device)  # noqa: E731
    got = select_evictions(PagedCache(None, None, *pools), wide, dev(lengths), dev(seen), budget, recent, sinks)
    src, dst, count = (x.cpu().numpy() for x in got)
    assert src.shape[2] == dst.shape[2] == max(0, min(budget, (width or m) * page - budget))
    for i, length in enumerate(lengths):
        for j in range(kv):
            s, d = choose(mass[i, j, :length], pos[i, j, :length], int(seen[i]), budget, recent, sinks) \
                if length > budget else ([], [])
            assert count[i, j] == len(s) == len(d)
            assert np.array_equal(src[i, j, :len(s)], s) and np.array_equal(dst[i, j, :len(d)], d)
            assert (src[i, j, len(s):] == -1).all() and (dst[i, j, len(d):] == -1).all()
    assert _capi.device_error() == 0
