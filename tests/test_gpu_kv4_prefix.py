"""Attention over the 4-bit cache behind beginnings that sequences share, on a B200 against 64 bits.

Tolerances: those of test_gpu_kv4.py, and for the join of up to 17 parts (the prefix's splits and the sequence's own) an exp2 (2^-22) and
three roundings (2^-24 each) a part, 2^-17.5 in all, twice as it enters values and sums: 2 vmax 2^-17 more.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_kv4 import TYPES, attended, contents, filled, rows_of, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[0, 600_000], ids=["walked", "passed"])
def room(request):
    """Few rows walk a beginning on their own where its capacity is small, and have a pass over it where it is large."""
    return request.param


def device(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device="cuda")


def queries(rows, heads, dim, dtype, seed=7):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, heads, dim, generator=gen, device="cuda") * 1.5).to(dtype)


def check(cache, prefix, lengths, groups, q, at, starts, dtype, scale=None, window=0, sinks=0, out=None):
    """One call against 64 bits; lengths, groups, at, starts as lists (groups, starts None)."""

    got = cache.attention(q.clone() if out is q else q, device(at), None if starts is None else device(starts, torch.int32), scale=scale, window=window,
                          sinks=sinks, out=out if out is not q else None, prefix=prefix, prefix_lengths=device(lengths),
                          prefix_groups=None if groups is None else device(groups, torch.int32))
    scale = cache.head_dim**-0.5 if scale is None else scale
    k, v, par = contents(cache.data, cache.head_dim)
    held = 2 * ((min(max(max(lengths), 1), prefix.max_len) + 31) // 32)
    pk, pv, ppar = contents(prefix.data[:, :, :held].contiguous(), cache.head_dim)
    bounds = list(range(cache.batch + 1)) if starts is None else starts
    for b in range(cache.batch):
        r0, r1 = bounds[b], bounds[b + 1]
        if r1 == r0:
            continue
        mine = [g for g in range(prefix.batch) if (0 if groups is None else groups[g]) <= b < (cache.batch if groups is None else groups[g + 1])]
        n = min(max(lengths[mine[0]], 0), prefix.max_len) if mine else 0
        own = torch.arange(r1 - r0) + at[b]
        rows = torch.where((own >= 0) & (own < cache.max_len), own + n, -1)
        kk, vv, pp = k[b], v[b], par[b]
        if n:
            kk, vv, pp = (torch.cat([x[mine[0]][:, :n], y], 1) for x, y in ((pk, kk), (pv, vv), (ppar, pp)))
        want = attended(q[r0:r1], kk, vv, rows, scale, window, sinks)
        end = max(int(rows.max()) + 1, 1)
        vmax = float(vv[:, :end].nan_to_num(0).abs().max())
        most = float((pp[:, :end, 1].abs() + 15 * pp[:, :end, 0]).nan_to_num(0, 0, 0).max())
        tol = tolerance(q[r0:r1], most, vmax, scale, want, dtype) + 2 * vmax * 2.0**-17
        diff = (got[r0:r1].double().cpu() - want).abs()
        assert bool((diff <= tol).all()), (b, float((diff - tol).max()), float(diff.max()))
    return got


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("group,window,sinks", [(1, 0, 0), (4, 0, 0), (3, 40, 4), (8, 1, 0), (16, 164, 133)])
def test_single_tokens(dim, dtype, group, window, sinks, room) -> None:
    from ivonar_inference_b200 import KV4Cache

    own = [1, 15, 16, 17, 33, 64, 65, 0, 100]
    cache, prefix = KV4Cache(len(own), 2, dim, 100), KV4Cache(1, 2, dim, 300 + room)
    filled(cache, own, seed=dim + group)
    filled(prefix, [300], seed=3)
    q = queries(len(own), 2 * group, dim, TYPES[dtype])
    for n in (1, 16, 128, 129, 300):
        got = check(cache, prefix, [n], None, q, [m - 1 for m in own], None, TYPES[dtype], window=window, sinks=sinks)
        assert bool((got[own.index(0)] == 0).all())   # an idle row
    cache.check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,group,window,sinks", [(64, 1, 0, 0), (128, 4, 0, 0), (32, 2, 50, 3), (64, 3, 217, 140), (128, 1, 100, 0)])
def test_prompts_drafts_and_single_tokens_in_one_call(dim, dtype, group, window, sinks, room) -> None:
    from ivonar_inference_b200 import KV4Cache

    first, counts = [0, 30, 7, 100, 0, 61, 0, 3], [150, 1, 5, 33, 0, 129, 1, 2]
    cache, prefix = KV4Cache(8, 2, dim, 256), KV4Cache(1, 2, dim, 140 + room)
    filled(cache, [a + n for a, n in zip(first, counts)], seed=dim)
    filled(prefix, [140], seed=5)
    starts = rows_of(8, first, counts)[1].tolist()
    q = queries(sum(counts), 2 * group, dim, TYPES[dtype])
    for n in (1, 127, 140):
        check(cache, prefix, [n], None, q, first, starts, TYPES[dtype], window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_groups(dtype, window, sinks, room) -> None:
    """Prefixes of other lengths, an empty group, one of length zero and one below, sequences of none, idle rows."""
    from ivonar_inference_b200 import KV4Cache

    groups, lengths = [1, 4, 4, 6, 8, 9], [200, 77, 0, 33, -3]
    own = [20, 5, 0, 31, 8, 1, 90, 40, 12, 50, 3]
    cache, prefix = KV4Cache(11, 2, 64, 90), KV4Cache(5, 2, 64, 200 + room)
    filled(cache, own, seed=3)
    filled(prefix, [200] * 5, seed=4)
    T = TYPES[dtype]
    check(cache, prefix, lengths, groups, queries(11, 6, 64, T), [n - 1 for n in own], None, T, window=window, sinks=sinks)
    counts = [3, 1, 0, 70, 2, 1, 50, 0, 4, 1, 2]
    first = [max(0, n - c) for n, c in zip(own, counts)]
    starts = rows_of(11, first, counts)[1].tolist()
    filled(cache, [max(n, a + c) for n, a, c in zip(own, first, counts)], seed=3)
    check(cache, prefix, lengths, groups, queries(sum(counts), 6, 64, T), first, starts, T, window=window, sinks=sinks)
    cache.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("batch,kv_heads,group,length,dim", [(2, 1, 1, 3001, 64), (70, 2, 4, 2500, 32), (300, 1, 1, 900, 64), (5, 3, 8, 1281, 128),
                                                                (40, 1, 3, 700, 128), (17, 2, 2, 1500, 64)])
def test_long_beginnings_are_split_and_joined(batch, kv_heads, group, length, dim, dtype, room) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(batch, kv_heads, dim, 40), KV4Cache(1, kv_heads, dim, length + 3 + room)
    own = [1 + 7 * b % 40 for b in range(batch)]
    filled(cache, own, seed=length)
    filled(prefix, [length], seed=1)
    q = queries(batch, kv_heads * group, dim, TYPES[dtype])
    check(cache, prefix, [length], None, q, [n - 1 for n in own], None, TYPES[dtype])
    check(cache, prefix, [length], None, q, [n - 1 for n in own], None, TYPES[dtype], window=600, sinks=5)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("batch,group,length", [(9, 1, 301), (9, 4, 1281), (70, 4, 1000), (300, 3, 130)])
def test_single_tokens_weights_keep_their_remainder(batch, group, length, dim, dtype, room) -> None:
    """16-bit single tokens of up to four query heads a key/value head, whose weights are not rounded, walked or passed: half the positions
    have the values of the other half with the other sign, so that what is left of them shows a rounding of the weights (2^-11, of values of 1).
    The tolerance is that of fp32 queries, and half a step of the output: tanh(0.03 / 2), and 1 / 131 where one half has a position more, times
    1.01 is under 2^-5."""
    from ivonar_inference_b200 import KV4Cache

    T = TYPES[dtype]
    cache, prefix = KV4Cache(batch, 2, dim, 20), KV4Cache(1, 2, dim, length + room)
    channel = (1.0 - 2.0 * (torch.arange(dim, device="cuda") % 3 == 0)).expand(2, dim)
    for to, n in ((prefix, length), (cache, 20)):
        k = (torch.arange(n, device="cuda") % 2).float()[:, None, None].expand(n, 2, dim)
        at, starts = rows_of(to.batch, [0] * to.batch, [n] * to.batch)
        to.append(k.repeat(to.batch, 1, 1), ((2 * k - 1) * channel).repeat(to.batch, 1, 1), at, starts)
    gen = torch.Generator(device="cuda").manual_seed(batch)
    q = (0.06 * torch.rand(batch, 2 * group, 1, generator=gen, device="cuda") - 0.03).expand(batch, 2 * group, dim).to(T) * dim**-0.5
    own = [b % 20 for b in range(batch)]
    got = cache.attention(q, device(own), prefix=prefix, prefix_lengths=device([length]))
    k, v, par = contents(cache.data, dim)
    pk, pv, _ = contents(prefix.data[:, :, : 2 * ((length + 31) // 32)].contiguous(), dim)
    for b in range(batch):
        kk, vv = torch.cat([pk[0][:, :length], k[b]], 1), torch.cat([pv[0][:, :length], v[b]], 1)
        want = attended(q[b:b + 1], kk, vv, [length + own[b]], dim**-0.5, 0, 0)
        assert float(want.abs().max()) < 2.0**-5
        tol = tolerance(q[b:b + 1], 1.0, 1.01, dim**-0.5, want, torch.float32) + 2 * 2.0**-17 + torch.finfo(T).eps / 2 * want.abs()
        diff = (got[b:b + 1].double().cpu() - want).abs()
        assert bool((diff <= tol).all()), (b, float((diff - tol).max()), float(diff.max()))


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_a_lone_sequence(dtype, room) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(1, 2, 64, 200), KV4Cache(1, 2, 64, 90 + room)
    filled(cache, [200])
    filled(prefix, [90], seed=1)
    for first, n in ((0, 200), (150, 3), (199, 1), (0, 1)):
        for window, sinks in ((0, 0), (64, 100)):
            check(cache, prefix, [83], None, queries(n, 4, 64, TYPES[dtype]), [first], [0, n], TYPES[dtype], window=window, sinks=sinks)
    check(cache, prefix, [83], None, queries(1, 4, 64, TYPES[dtype]), [77], None, TYPES[dtype])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("sizes", [[1, 2] * 35, [200, 1, 1, 3], [0, 90, 5], [300, 290]])
def test_many_and_uneven_groups(sizes, dtype, room) -> None:
    """More groups than a warp has lanes, and groups of other sizes than the even ones that the tiles are chosen by."""
    from ivonar_inference_b200 import KV4Cache

    batch, many = sum(sizes), len(sizes)
    lengths = [37 * (g + 3) % 300 for g in range(many)]
    cache, prefix = KV4Cache(batch, 1, 32, 20), KV4Cache(many, 1, 32, 300 + room // 8)
    own = [1 + b % 20 for b in range(batch)]
    filled(cache, own, seed=1)
    filled(prefix, [300] * many, seed=2)
    groups = [sum(sizes[:g]) for g in range(many + 1)]
    for group in (1, 4):
        check(cache, prefix, lengths, groups, queries(batch, group, 32, TYPES[dtype]), [n - 1 for n in own], None, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts", [None, [1, 70, 3]])
def test_masked_places_may_hold_anything(dtype, counts, room) -> None:
    """NaN scales and infinities behind the beginning's end, behind the last position and outside the window."""
    from ivonar_inference_b200 import KV4Cache

    T = TYPES[dtype]
    cache, prefix = KV4Cache(3, 2, 64, 160), KV4Cache(1, 2, 64, 150 + room)
    n = [1, 70, 3] if counts is None else counts
    first, length, window, sinks = [0, 71, 10], 141, 60, 2
    filled(cache, [160] * 3, seed=2)
    filled(prefix, [150], seed=3)
    rows = 3 if counts is None else sum(n)
    q = queries(rows, 4, 64, T)
    at, starts = rows_of(3, first, n)
    starts = None if counts is None else starts
    args = dict(window=window, sinks=sinks, prefix=prefix, prefix_lengths=device([length]))
    want = cache.attention(q, at, starts, **args)
    bad = torch.tensor([math.nan, math.inf, -math.inf, -65504.0], dtype=torch.float16).view(torch.uint8).to("cuda")
    lowest = min(length + a - window for a in first)
    for p in range(150):
        if p >= length or sinks <= p <= lowest:
            prefix.data[:, :, p // 16, 1024 + 8 * (p % 16):1032 + 8 * (p % 16)] = bad.roll(2 * (p % 4))
    for b in range(3):
        last = first[b] + (1 if counts is None else n[b]) - 1
        for p in range(160):
            if p > last or length + p <= length + first[b] - window:
                cache.data[b, :, p // 16, 1024 + 8 * (p % 16):1032 + 8 * (p % 16)] = bad.roll(2 * (p % 4))
    assert torch.equal(cache.attention(q, at, starts, **args), want)
    assert bool(torch.isfinite(want).all())


def test_a_visible_nan_reaches_its_rows_only(room) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(4, 2, 64, 64), KV4Cache(2, 2, 64, 64 + room)
    filled(cache, [64] * 4)
    filled(prefix, [64] * 2)
    x = torch.randn(2, 2, 64, device="cuda")
    x[0, 1, 5] = math.nan
    prefix.append(x, x.abs(), device([40, 40]))
    q = queries(4, 4, 64, torch.float32)
    args = dict(prefix=prefix, prefix_lengths=device([64, 64]), prefix_groups=device([0, 2, 4], torch.int32))
    got = cache.attention(q, device([5, 6, 7, 8]), **args)
    assert bool(got[:2, 2:].isnan().all()) and bool(torch.isfinite(got[:2, :2]).all()) and bool(torch.isfinite(got[2:]).all())
    q[3, 0, 3] = math.inf
    got = cache.attention(q, device([5, 6, 7, 8]), **args)
    assert bool(got[3, 0].isnan().all()) and bool(torch.isfinite(got[3, 1:]).all()) and bool(torch.isfinite(got[2]).all())


def test_rows_outside_are_zero_or_left_alone_and_reported(room) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(4, 2, 64, 50), KV4Cache(1, 2, 64, 60 + room)
    filled(cache, [50] * 4)
    filled(prefix, [60], seed=2)
    q = queries(12, 4, 64, torch.float32)
    at, starts = rows_of(4, [-2, 48, 2**62, -(2**62)], [3, 4, 1, 1])
    out = torch.full((12, 4, 64), 9.0, device="cuda")
    args = dict(prefix=prefix, prefix_lengths=device([60]))
    cache.attention(q, at, starts, out=out, **args)
    with pytest.raises(ValueError, match="capacity"):
        cache.check()
    assert bool((out[[0, 1, 5, 6, 7, 8]] == 0).all()) and bool((out[9:] == 9.0).all())
    check(cache, prefix, [60], None, q[2:5].repeat(2, 1, 1)[:4], [0, 48, 49, -1], None, torch.float32)
    want = cache.attention(q[2:5], device([0, 48, 50, -1]), device([0, 1, 3, 3, 3], torch.int32), **args)
    assert torch.equal(out[2:5], want)
    # rows before and behind the call's own
    part = cache.attention(q[3:5], device([0, 48, 50, -1]), device([-1, 0, 2, 2, 2], torch.int32), **args)
    assert torch.equal(part, want[1:])
    part = cache.attention(q[2:4], device([0, 48, 50, -1]), device([0, 1, 3, 3, 3], torch.int32), **args)
    assert torch.equal(part, want[:2])
    cache.check()
    if room:   # more positions than were written
        return
    # lengths beyond the capacity count as that and are reported
    for first, counts in (([5] * 4, None), ([0] * 4, [1, 1, 50, 2])):
        where = (device(first), None) if counts is None else rows_of(4, first, counts)
        x = queries(4 if counts is None else sum(counts), 4, 64, torch.float32)
        long = cache.attention(x, *where, prefix=prefix, prefix_lengths=device([2**40]))
        with pytest.raises(ValueError, match="capacity"):
            cache.check()
        assert torch.equal(long, cache.attention(x, *where, **args))
        short = cache.attention(x, *where, prefix=prefix, prefix_lengths=device([-(2**40)]))
        assert torch.equal(short, cache.attention(x, *where, prefix=prefix, prefix_lengths=device([0])))
    cache.check()


def test_a_beginning_of_nothing_is_the_plain_attention(room) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(3, 2, 64, 300), KV4Cache(1, 2, 64, 60 + room)
    filled(cache, [300] * 3)
    for first, counts in (([5, 100, 299], None), ([0, 30, 250], [200, 1, 30])):
        where = (device(first), None) if counts is None else rows_of(3, first, counts)
        q = queries(3 if counts is None else sum(counts), 4, 64, torch.float32)
        for window, sinks in ((0, 0), (50, 3)):
            got = cache.attention(q, *where, window=window, sinks=sinks, prefix=prefix, prefix_lengths=device([0]))
            # (the few rows' warps may share a history otherwise)
            want = cache.attention(q, *where, window=window, sinks=sinks)
            assert float((got - want).abs().max()) <= 2.0**-18 * float(want.abs().max())


def test_scale_strides_alignment_and_in_place(room) -> None:
    from ivonar_inference_b200 import KV4Cache

    for dtype in TYPES.values():
        for dim in (32, 64, 128):
            cache, prefix = KV4Cache(3, 2, dim, 40), KV4Cache(1, 2, dim, 130 + room)
            filled(cache, [40] * 3)
            filled(prefix, [130], seed=2)
            n = [30, 3, 1]
            starts = [0, 30, 33, 34]
            fused = torch.randn(34, 4 * dim + 1, device="cuda").to(dtype)[:, 1:]
            q = fused.unflatten(1, (4, dim))
            want = check(cache, prefix, [130], None, q, [0, 7, 39], starts, dtype, scale=0.31)
            turned = torch.empty(4, sum(n), dim, dtype=dtype, device="cuda").transpose(0, 1)
            odd = torch.empty(34, 4 * dim + 1, dtype=dtype, device="cuda")[:, 1:].unflatten(1, (4, dim))
            args = dict(scale=0.31, prefix=prefix, prefix_lengths=device([130]))
            for out in (turned, odd):
                assert torch.equal(cache.attention(q, device([0, 7, 39]), device(starts, torch.int32), out=out, **args), want)
            assert torch.equal(cache.attention(q.contiguous(), device([0, 7, 39]), device(starts, torch.int32), **args), want)
            here = q.contiguous()
            assert torch.equal(cache.attention(here, device([0, 7, 39]), device(starts, torch.int32), out=here, **args), want)
            tokens = queries(3, 4, dim, dtype)
            want = check(cache, prefix, [130], None, tokens, [0, 7, 39], None, dtype, scale=-0.2)
            assert torch.equal(cache.attention(tokens, device([0, 7, 39]), out=tokens, **dict(args, scale=-0.2)), want)


def test_offsets_beyond_32_bits() -> None:
    from ivonar_inference_b200 import KV4Cache

    length = 1 << 24
    prefix, cache = KV4Cache(3, 1, 128, length), KV4Cache(3, 1, 128, 50)   # 2.3 GB a sequence
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(60, 1, 128, generator=gen, device="cuda")
    prefix.append(x, -x, *rows_of(3, [length - 20] * 3, [20, 20, 20]))
    filled(cache, [50] * 3)
    pk, pv = prefix.read(*rows_of(3, [length - 20] * 3, [20, 20, 20]), rows=60)
    k, v, par = contents(cache.data, 128)
    for first, counts in (([9] * 3, None), ([0, 5, 5], [40, 2, 1])):
        where = (device(first), None) if counts is None else rows_of(3, first, counts)
        n = [1] * 3 if counts is None else counts
        q = queries(sum(n), 2, 128, torch.float32)
        got = cache.attention(q, *where, window=20 + min(first), prefix=prefix, prefix_lengths=device([length] * 3),
                              prefix_groups=device([0, 1, 2, 3], torch.int32))
        r = 0
        for b in range(3):
            kk = torch.cat([pk[20 * b:20 * b + 20].double().cpu().transpose(0, 1), k[b]], 1)
            vv = torch.cat([pv[20 * b:20 * b + 20].double().cpu().transpose(0, 1), v[b]], 1)
            want = attended(q[r:r + n[b]], kk, vv, [20 + first[b] + i for i in range(n[b])], 128**-0.5, 20 + min(first), 0)
            tol = tolerance(q[r:r + n[b]], float(kk.abs().max()) * 3, float(vv.abs().max()), 128**-0.5, want, torch.float32)
            assert bool(((got[r:r + n[b]].double().cpu() - want).abs() <= tol + 2 * float(vv.abs().max()) * 2.0**-17).all()), (b, n)
            r += n[b]


def test_captured_on_two_streams_and_repeated(room) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(40, 2, 64, 64), KV4Cache(1, 2, 64, 2000 + room)
    filled(cache, [64] * 40)
    filled(prefix, [2000], seed=2)
    first, counts = [3] * 40, [1] * 38 + [60, 2]
    at, starts = rows_of(40, first, counts)
    q, tokens = queries(sum(counts), 8, 64, torch.bfloat16), queries(40, 8, 64, torch.bfloat16, 8)
    lengths = device([2000])

    def both():
        return (cache.attention(q, at, starts, prefix=prefix, prefix_lengths=lengths), cache.attention(tokens, at, prefix=prefix, prefix_lengths=lengths))

    want = both()
    for a, b in zip(both(), want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            found = both()
        graphs.append((graph, found))
    sides = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):   # two graphs and an eager call at the same time
        for side, (graph, _) in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        with torch.cuda.stream(sides[2]):
            eager = both()
    torch.cuda.synchronize()
    for found in [f for _, f in graphs] + [eager]:
        for a, b in zip(found, want):
            assert torch.equal(a, b)
    lengths.fill_(100)   # read when the graph runs
    graphs[0][0].replay()
    torch.cuda.synchronize()
    for a, b in zip(graphs[0][1], both()):
        assert torch.equal(a, b)


def test_a_shared_beginning_is_what_each_sequence_could_have_held(room) -> None:
    """The same histories held by each sequence on its own: forked, with their own tokens behind."""
    from ivonar_inference_b200 import KV4Cache

    cache, prefix, whole = KV4Cache(5, 2, 64, 64), KV4Cache(1, 2, 64, 96 + room), KV4Cache(5, 2, 64, 160)
    filled(prefix, [96], seed=2)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(5 * 20, 2, 64, generator=gen, device="cuda")
    at, starts = rows_of(5, [0] * 5, [20] * 5)
    cache.append(x, x, at, starts)
    whole.fork(device([0] * 5), device([96] * 5), source=prefix)
    whole.append(x, x, at + 96, starts)
    q = queries(100, 4, 64, torch.float32)
    got = cache.attention(q, at, starts, prefix=prefix, prefix_lengths=device([96]))
    assert float((got - whole.attention(q, at + 96, starts)).abs().max()) < 1e-5
    got = cache.attention(q[:5], at + 19, prefix=prefix, prefix_lengths=device([96]))
    assert float((got - whole.attention(q[:5], at + 115)).abs().max()) < 1e-5


@pytest.mark.parametrize("dtype,dim,heads", [("fp32", 64, 4), ("bf16", 128, 4), ("fp32", 128, 2), ("fp16", 64, 96)])
def test_waits_of_a_pass_that_run_out_are_reported_and_the_gpu_stays_usable(dtype, dim, heads) -> None:
    """No products are issued, so that every wait for them gives up after 1 ms: NaN for the rows behind the beginning, and the error word."""
    import ctypes

    from ivonar_inference_b200 import KernelError, KV4Cache
    from ivonar_inference_b200 import _native as native

    cache, prefix = KV4Cache(6, 2, dim, 64), KV4Cache(1, 2, dim, 600_000)
    filled(cache, [64] * 6)
    filled(prefix, [900], seed=1)
    q, at, lengths, groups = queries(6, heads, dim, TYPES[dtype]), device([5, 9, 63, 0, -1, 7]), device([900]), device([0, 5], torch.int32)
    args = dict(prefix=prefix, prefix_lengths=lengths, prefix_groups=groups)
    want = cache.attention(q, at, **args)
    out = torch.empty_like(q)
    shared = native.IvbKv4Prefix(prefix._desc, lengths.data_ptr(), groups.data_ptr())
    lib, T = native.library(), {"fp32": native.IVB_F32, "fp16": native.IVB_F16, "bf16": native.IVB_BF16}[dtype]
    nbytes = lib.ivb_kv4_prefix_workspace_bytes(cache._ref, ctypes.byref(shared), T, heads, None, 6)
    assert nbytes > 0
    workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    rc = lib.ivb_probe_kv4_prefix_timeout(
        cache._ref, ctypes.byref(shared), q.data_ptr(), T, q.stride(0), q.stride(1), heads, None, at.data_ptr(), 6, dim**-0.5, 0, 0, out.data_ptr(),
        out.stride(0), out.stride(1), workspace.data_ptr(), nbytes, cache.error.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == native.IVB_OK
    with pytest.raises(KernelError, match="error"):
        cache.check()
    assert bool(out[:4].isnan().all()) and bool((out[4] == 0).all()) and torch.equal(out[5], want[5])
    assert torch.equal(cache.attention(q, at, **args), want)
    cache.check()


def test_refusals() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache, prefix = KV4Cache(3, 2, 64, 64), KV4Cache(2, 2, 64, 96)
    q, at, n, g = queries(3, 4, 64, torch.float32), device([1, 2, 3]), device([5, 6]), device([0, 1, 3], torch.int32)

    def refused(match, **kwargs):
        with pytest.raises(ValueError, match=match):
            cache.attention(q, at, **kwargs)

    refused("need a prefix", prefix_lengths=n)
    refused("need a prefix", prefix_groups=g)
    refused("needs prefix_lengths", prefix=prefix, prefix_groups=g)
    refused("need prefix_groups", prefix=prefix, prefix_lengths=n)
    for bad in (n.int(), n[:1], n.cpu(), device([1, 2, 3, 4])[::2]):
        refused("prefix_lengths must be", prefix=prefix, prefix_lengths=bad, prefix_groups=g)
    for bad in (g.long(), g[:2], g.cpu()):
        refused("prefix_groups must be", prefix=prefix, prefix_lengths=n, prefix_groups=bad)
    for other in (KV4Cache(2, 1, 64, 96), KV4Cache(2, 2, 32, 96)):
        refused("prefix must be", prefix=other, prefix_lengths=n, prefix_groups=g)
    cache.attention(q[:0], at, device([0, 0, 0, 0], torch.int32), prefix=prefix, prefix_lengths=n, prefix_groups=g)
    # a cache may be its own prefix: its first sequence read by the others
    filled(cache, [64] * 3)
    own = cache.sequence(0)
    check(cache, own, [64], None, q, [1, 2, 3], None, torch.float32)
