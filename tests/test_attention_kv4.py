"""The 4-bit cache's attention where its kernels and calls meet: grids beside one another, rows of any size beside one another,
waits that run out, outputs and strides that are refused or put right, and its rounding against 64 bits row by row.

Tolerances are those of test_gpu_kv4.py unless a test derives its own."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_kv4 import TYPES, contents, filled, held, rows_of, tolerance

gpu = pytest.mark.gpu


# ---- few rows beside prompts --------------------------------------------------------------------
# Cases in which the few rows' kernel takes one warp a tile (over 4736 tiles, or a cache of up to 32 positions): sequence 0 is one
# of few rows, and a prompt is in the call.
ONE_WARP = [
    ("fp32", 64, 32, 160, 4, 1, {60: 400}),
    ("bf16", 64, 32, 160, 4, 1, {60: 400, 159: 65}),
    ("fp16", 128, 32, 150, 300, 1, {3: 300}),
    ("fp32", 64, 2, 3, 0, 4, {1: 20}),
    ("bf16", 32, 2, 4, 0, 8, {2: 31}),
]


@gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype,dim,kv_heads,batch,first,group,prompts", ONE_WARP)
def test_calls_that_follow_a_mixed_call_of_one_warp_a_tile(dtype, dim, kv_heads, batch, first, group, prompts, captured) -> None:
    """Each call's inputs are the last one's outputs, and the cache is written over between: as with a wait after every call."""
    from ivonar_inference_b200 import KV4Cache

    T = TYPES[dtype]
    counts = [prompts.get(b, 1) for b in range(batch)]
    rows, length = sum(counts), first + max(counts)
    at, starts = rows_of(batch, [first] * batch, counts)
    gen = torch.Generator(device="cuda").manual_seed(21)
    start = torch.randn(rows, kv_heads * group, dim, generator=gen, device="cuda").to(T)
    results = []
    for wait in (True, False):
        cache = KV4Cache(batch, kv_heads, dim, max(length, 32 if first == 0 else 0))
        filled(cache, [first] * batch, seed=4)
        x, history = start.clone(), []

        def pause():
            if wait:
                torch.cuda.synchronize()

        def step():
            cache.append(x[:, :kv_heads], x[:, -kv_heads:], at, starts)
            pause()
            y = cache.attention(x, at, starts)
            pause()
            cache.append(y[:, :kv_heads], y[:, -kv_heads:], at, starts)     # over what the attention read
            pause()
            k, v = cache.read(at, starts, rows, dtype=T)
            pause()
            cache.attention(y, at, starts, out=x)
            pause()
            return y, k, v

        if captured and not wait:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            for _ in range(4):
                graph.replay()
                history.append([t.clone() for t in (*out, x)])
        else:
            for _ in range(4):
                history.append([t.clone() for t in (*step(), x)])
        torch.cuda.synchronize()
        cache.check()
        results.append(history)
    for waited, free in zip(*results):
        for a, b in zip(waited, free):
            assert torch.isfinite(a).all() and torch.equal(a, b)


# ---- rows beside rows of another size -----------------------------------------------------------
SHAPES = [  # dim, kv_heads, group, batch, first position, counts (None: one row each)
    (64, 2, 4, 3, 39, None),
    (128, 1, 8, 2, 50, None),
    (32, 1, 16, 2, 33, None),
    (64, 1, 2, 2, 30, [7, 3]),
    (128, 2, 1, 1, 20, [150]),
    (64, 2, 2, 2, 10, [200, 5]),
    (32, 1, 4, 1, 40, [100]),
]


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,kv_heads,group,batch,first,counts", SHAPES)
def test_rows_do_not_depend_on_the_size_of_others(dim, kv_heads, group, batch, first, counts, dtype) -> None:
    """Queries of a call 2^33 (fp16: 2^12) apart, the scale for the small ones, so that the large ones see the key of their largest
    score only: small rows within the bound of their own size, large rows that value."""
    from ivonar_inference_b200 import KV4Cache

    T, k = TYPES[dtype], 12 if dtype == "fp16" else 33
    counts_ = [1] * batch if counts is None else counts
    total = [first + n for n in counts_]
    cache = KV4Cache(batch, kv_heads, dim, max(total))
    filled(cache, total, seed=dim + batch)
    gen = torch.Generator(device="cuda").manual_seed(9)
    rows, H = sum(counts_), kv_heads * group
    q = torch.randn(rows, H, dim, generator=gen, device="cuda") * 1.5
    # every third head of a group, or every third token
    large = (torch.arange(rows)[:, None] + torch.arange(H)[None]) % 3 == 1
    q = torch.where(large[..., None].cuda(), q, q * 2.0**-k).to(T)
    scale = 2.0**k * dim**-0.5
    at, starts = rows_of(batch, [first] * batch, counts_)
    got = cache.attention(q, at, None if counts is None else starts, scale=scale).double().cpu()
    kk, vv, par = contents(cache.data, dim)
    tested, r0 = 0, 0
    for b in range(batch):
        n = counts_[b]
        x = q[r0:r0 + n].double().cpu().unflatten(1, (kv_heads, group))
        score = torch.einsum("nhgd,hjd->nhgj", x, kk[b, :, :total[b]]) * scale
        hidden = torch.arange(total[b])[None] > first + torch.arange(n)[:, None]
        score = score.masked_fill(hidden[:, None, None], -math.inf).flatten(1, 2)
        weight = torch.softmax(score, -1).unflatten(1, (kv_heads, group))
        want = torch.einsum("nhgj,hjd->nhgd", weight, vv[b, :, :total[b]]).flatten(1, 2)
        most = float((par[b, :, :total[b], 1].abs() + 15 * par[b, :, :total[b], 0]).max())
        vmax = float(vv[b, :, :total[b]].abs().max())
        small = ~large[r0:r0 + n]
        tol = tolerance(q[r0:r0 + n][small.cuda()], most, vmax, scale, want, T)
        diff = (got[r0:r0 + n] - want).abs()
        assert bool((diff[small] <= tol[small]).all()), (b, float(diff[small].max()))
        # a large row: scores are off by A 2^-18 at most, so a gap of twice that and 40 leaves the others weights below e^-40
        A = scale * float(q[r0:r0 + n].double().abs().sum(-1).max()) * most
        two = score.topk(2, -1).values
        clear = ~small & (two[..., 0] - two[..., 1] > 2 * A * 2.0**-18 + 40)
        tested += int(clear.sum())
        tol = 2 * vmax * (2.0**-17 + (0 if T == torch.float32 else 2.0**-11)) + (0 if T == torch.float32 else torch.finfo(T).eps / 2) * want.abs()
        assert bool((diff[clear] <= tol[clear]).all()), (b, float(diff[clear].max()))
        r0 += n
    assert tested >= int(large.sum()) // 2
    cache.check()


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,group,counts,idle", [(64, 1, [9], 4), (64, 4, [3, 6], 2), (128, 2, [150], 40), (32, 1, [300, 5], 3), (64, 3, [100, 1], 30)])
def test_idle_rows_may_hold_any_query(dim, group, counts, idle, dtype) -> None:
    """Rows before position 0 and beyond the capacity: the others' results to the last bit whatever they hold."""
    from ivonar_inference_b200 import KV4Cache

    T, batch = TYPES[dtype], len(counts)
    length = max(counts)
    cache = KV4Cache(batch, 2, dim, length - idle - 1)    # the longest sequence's last row is beyond it
    filled(cache, [length - idle - 1] * batch, seed=dim)
    gen = torch.Generator(device="cuda").manual_seed(9)
    at, starts = rows_of(batch, [-idle] * batch, counts)
    q = (torch.randn(sum(counts), 2 * group, dim, generator=gen, device="cuda") * 1.5).to(T)
    live = torch.cat([(torch.arange(n) >= idle) & (torch.arange(n) - idle < cache.max_len) for n in counts]).cuda()
    want = cache.attention(q, at, starts)
    assert bool((want[~live] == 0).all()) and bool((want[live] != 0).any()) and 0 < int(live.sum()) < sum(counts)
    for value in (0.0, 1e30, torch.finfo(T).max, math.inf, math.nan):
        q[~live] = torch.tensor(value).to(T).cuda()
        assert torch.equal(cache.attention(q, at, starts), want)


# ---- waits that run out -------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,kv_heads,counts", [(64, 2, [300, 1, 5]), (128, 40, [90] * 5 + [2]), (32, 1, [400]), (128, 1, [1, 1, 500])])
def test_rows_whose_wait_ran_out_are_nan_and_reported(dim, kv_heads, counts, dtype) -> None:
    """One CTA a tile of rows and clusters: no row of a prompt looks like a result, few rows are what they were, and the next call is."""
    import ctypes

    from ivonar_inference_b200 import KernelError, KV4Cache
    from ivonar_inference_b200 import _native as native

    T, batch = TYPES[dtype], len(counts)
    cache = KV4Cache(batch, kv_heads, dim, 700)
    filled(cache, [100 + n for n in counts], seed=dim)
    at, starts = rows_of(batch, [100] * batch, counts)
    q = torch.randn(sum(counts), kv_heads, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(T)
    want = cache.attention(q, at, starts)
    out = torch.full_like(q, 3.0)
    rc = native.library().ivb_probe_kv4_timeout(
        ctypes.byref(native.IvbKv4Cache(cache.data.data_ptr(), batch, kv_heads, dim, 700)), q.data_ptr(), list(TYPES).index(dtype), *q.stride()[:2],
        kv_heads, starts.data_ptr(), at.data_ptr(), q.shape[0], dim**-0.5, 0, 0, out.data_ptr(), *out.stride()[:2], cache.error.data_ptr(),
        torch.cuda.current_stream().cuda_stream)
    assert rc == native.IVB_OK
    with pytest.raises(KernelError, match=str(native.IVB_ETIMEOUT)):
        cache.check()
    r0 = 0
    for n in counts:
        if n > 64:
            assert bool(out[r0:r0 + n].isnan().all())
        else:
            assert torch.equal(out[r0:r0 + n], want[r0:r0 + n])
        r0 += n
    assert torch.equal(cache.attention(q, at, starts), want)
    cache.check()


# ---- outputs whose rows share memory ------------------------------------------------------------
def _shared(x: torch.Tensor) -> bool:
    """By the places of every value."""
    rows, heads, dim = x.shape
    row, head, channel = x.stride()
    at = (torch.arange(rows)[:, None, None] * row + torch.arange(heads)[:, None] * head + torch.arange(dim) * channel).flatten()
    return at.unique().numel() < at.numel()


def test_overlapping_outputs_are_found() -> None:
    """Every pair of strides of small outputs, and pairs of outputs, against the places of every value."""
    from ivonar_inference_b200.kv4 import _apart, _writable

    memory = torch.zeros(4096)
    for rows, heads in ((1, 1), (1, 3), (3, 1), (2, 2), (3, 4), (4, 3)):
        for row in (0, 1, 4, 7, 8, 9, 16, 24, 25, 32, 40, 64):
            for head in (0, 1, 4, 7, 8, 9, 16, 24, 25, 32, 40, 64):
                x = memory.as_strided((rows, heads, 8), (row, head, 1))
                if _shared(x):
                    with pytest.raises(ValueError, match="overlap"):
                        _writable(x)
                else:
                    _writable(x)
    for rows, heads in ((1, 1), (3, 2), (2, 3)):
        for strides in ((8 * heads, 8), (16 * heads, 8), (8, 8 * rows), (16, 16 * rows), (24 * heads, 24)):
            for other in (strides, (8 * heads, 8), (32 * heads, 16)):
                for gap in (0, 1, 7, 8, 9, 16, 8 * heads, 8 * rows, 8 * rows * heads, 1000):
                    a = memory.as_strided((rows, heads, 8), (*strides, 1))
                    b = memory.as_strided((rows, heads, 8), (*other, 1), gap)
                    places = torch.cat([torch.arange(4096).as_strided(t.shape, t.stride(), t.storage_offset()).flatten() for t in (a, b)])
                    for pair in ((a, b), (b, a)):
                        if places.unique().numel() < places.numel():
                            with pytest.raises(ValueError, match="overlap"):
                                _apart(*pair, "outputs")
                        else:
                            _apart(*pair, "outputs")
    _writable(memory[:0].view(0, 2, 8))
    _apart(memory[:0].view(0, 2, 8), memory[:0].view(0, 2, 8), "outputs")


@gpu
def test_overlapping_outputs_are_refused() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(3, 2, 64, 16)
    at = torch.tensor([4, 5, 6], device="cuda")
    memory = torch.zeros(4096, device="cuda")
    q = torch.zeros(3, 2, 64, device="cuda")
    for strides in ((64, 64, 1), (0, 64, 1), (128, 32, 1), (96, 64, 1)):
        wrong = memory.as_strided((3, 2, 64), strides)
        with pytest.raises(ValueError, match="overlap"):
            cache.attention(q, at, out=wrong)
        with pytest.raises(ValueError, match="overlap"):
            cache.read(at, out=(q, wrong))
        with pytest.raises(ValueError, match="overlap"):
            cache.read(at, out=(wrong, q))
    with pytest.raises(ValueError, match="overlap"):
        cache.read(at, out=(q, q))
    with pytest.raises(ValueError, match="overlap"):
        cache.read(at, out=(memory[:384].view(3, 2, 64), memory[64:448].view(3, 2, 64)))
    filled(cache, [10] * 3)
    want = cache.read(at)
    # rows within the step of heads, and keys and values side by side
    turned = memory.as_strided((3, 2, 64), (64, 192, 1)), memory.as_strided((3, 2, 64), (64, 192, 1), 1024)
    fused = memory[2048:].as_strided((3, 2, 64), (256, 64, 1)), memory[2048:].as_strided((3, 2, 64), (256, 64, 1), 2048 + 128)
    for out in (turned, fused):
        cache.read(at, out=out)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


# ---- queries whose rows overlap -----------------------------------------------------------------
@gpu
@pytest.mark.parametrize("rows,strides", [(4, (1, 64, 1)), (100, (1, 256, 1)), (100, (64, 1, 1)), (3, (2, 2, 1)), (100, (0, 0, 1)), (70, (64, 64, 1))])
def test_queries_that_overlap(rows, strides) -> None:
    """Sliding windows over one tensor: the result's channels are contiguous and its values those of the copied queries."""
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(1, 2, 64, 128)
    filled(cache, [128])
    memory = torch.randn(8192, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    q = memory.as_strided((rows, 2, 64), strides)
    at, starts = rows_of(1, [5], [rows])
    got, want = cache.attention(q, at, starts), cache.attention(q.contiguous(), at, starts)
    assert got.stride(2) == 1 and torch.equal(got, want) and bool((want != 0).all())


@gpu
@pytest.mark.parametrize("rows", [3, 90])
def test_an_output_is_the_queries_or_apart_from_them(rows) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(1, 2, 64, 128)
    filled(cache, [128])
    at, starts = rows_of(1, [20], [rows])
    gen = torch.Generator(device="cuda").manual_seed(2)
    memory = torch.randn(rows + 2, 8, 64, generator=gen, device="cuda")
    q = memory[:rows, :4]
    want = cache.attention(q, at, starts)
    for wrong in (memory[1:rows + 1, :4], memory[:rows, 1:5], memory[:rows, 3:7], memory[:rows, :4].transpose(0, 1).reshape(-1)[:0]):
        with pytest.raises(ValueError):
            cache.attention(q, at, starts, out=wrong)
    narrow = torch.randn(rows * 4 * 64 + 64, generator=gen, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        cache.attention(narrow[:-64].view(rows, 4, 64), at, starts, out=narrow[64:].view(rows, 4, 64))
    # an input whose own rows overlap, and an output beside it
    assert cache.attention(narrow[:256].view(1, 4, 64).expand(rows, 4, 64), at, starts, out=memory[:rows, 4:]).data_ptr() == memory[:, 4:].data_ptr()
    for out in (memory[:rows, 4:], q):
        assert torch.equal(cache.attention(q, at, starts, out=out), want) and torch.equal(out, want)


# ---- positions and rows at the ends of their ranges ---------------------------------------------
@gpu
@pytest.mark.parametrize("rows", [3, 100])
@pytest.mark.parametrize("position", [2**63 - 1, 2**63 - 2, 2**62, 2**31 - 1, -(2**63)])
def test_positions_at_the_ends_of_their_range(position, rows) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(2, 2, 64, 128)
    filled(cache, [128, 128])
    before = cache.data.clone()
    at, starts = rows_of(2, [position, 20], [rows, 2])
    x = torch.randn(rows + 2, 2, 64, device="cuda")
    want = cache.attention(x[rows:], torch.tensor([200, 20], device="cuda"), torch.tensor([0, 0, 2], dtype=torch.int32, device="cuda"))
    cache.check()

    def reported():
        if position < 0:
            cache.check()
        else:
            with pytest.raises(ValueError, match="capacity"):
                cache.check()

    y = cache.attention(x, at, starts)
    reported()
    assert bool((y[:rows] == 0).all()) and torch.equal(y[rows:], want)
    out = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    cache.read(at, starts, out=out)
    reported()
    assert all(bool((o[:rows] == 9.0).all()) and bool((o[rows:] != 9.0).any()) for o in out)
    cache.append(x, x, at, starts)
    reported()
    assert torch.equal(cache.data[0], before[0])


@gpu
@pytest.mark.parametrize("counts,cuts", [([3, 1, 5], [2, 6]), ([200, 1, 150, 40], [70, 201, 230, 300]), ([400], [1, 300])])
def test_a_call_in_parts(counts, cuts) -> None:
    """Slices of a call's rows with starts less the rows before: every part is what the whole call has there."""
    from ivonar_inference_b200 import KV4Cache

    batch, rows = len(counts), sum(counts)
    whole, parts = (KV4Cache(batch, 2, 64, 600) for _ in range(2))
    at, starts = rows_of(batch, [50] * batch, counts)
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = torch.randn(3, rows, 2, 64, generator=gen, device="cuda")
    for cache in (whole, parts):
        filled(cache, [50] * batch)
    whole.append(k, v, at, starts)
    bounds = list(zip([0] + cuts, cuts + [rows]))
    for a, b in bounds:
        parts.append(k[a:b], v[a:b], at, starts - a)
    assert torch.equal(parts.data, whole.data)
    want, held_ = whole.attention(q, at, starts), whole.read(at, starts, rows)
    kk, vv, par = contents(whole.data, 64)
    most, vmax = float((par[..., 1].abs() + 15 * par[..., 0]).max()), float(vv.abs().max())
    for a, b in bounds:
        for got, expected in zip(parts.read(at, starts - a, b - a), held_):
            assert torch.equal(got, expected[a:b])
        got = parts.attention(q[a:b], at, starts - a)
        # other kernels and splits: both within the tolerance of the exact result
        tol = tolerance(q, most, vmax, 0.125, want[a:b].double().cpu(), torch.float32)
        assert bool(((got - want[a:b]).abs().double().cpu() <= 2 * tol).all())
    whole.check()
    parts.check()


@gpu
def test_more_rows_than_32_bits_count_are_refused() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(1, 1, 64, 16)
    at, starts = rows_of(1, [0], [5])
    x = torch.ones(1, 1, 64, device="cuda")
    for rows in (2**31, 2**32 + 1):
        many = x.expand(rows, 1, 64)
        with pytest.raises(ValueError, match="rows"):
            cache.append(many, many, at, starts)
    assert bool((cache.data == 0).all())


@gpu
def test_dual_tensors_are_refused() -> None:
    """Forward-mode tangents would be lost; transforms of torch.func have no storage to read."""
    from torch.autograd import forward_ad

    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(2, 2, 64, 16)
    at = torch.tensor([0, 0], device="cuda")
    x = torch.ones(2, 2, 64, device="cuda")
    with forward_ad.dual_level():
        cache.append(x, x, at)
        before = cache.data.clone()
        dual = forward_ad.make_dual(x, x)
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                for call in (lambda: cache.append(dual, x, at), lambda: cache.append(x, dual, at), lambda: cache.attention(dual, at)):
                    with pytest.raises(ValueError, match="tangent"):
                        call()
        assert torch.isfinite(cache.attention(x, at)).all()
    for transform in (lambda f: torch.func.jvp(f, (x,), (x,)), lambda f: torch.func.grad(lambda y: f(y).sum())(x), lambda f: torch.func.vmap(f)(x[None])):
        with pytest.raises((ValueError, RuntimeError)):
            transform(lambda y: cache.attention(y, at))
    assert torch.equal(cache.data, before)


# ---- rows at the ends of the types --------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_of_the_whole_range(dtype) -> None:
    """What is clipped and what is not: the offset to +-65504, the scale to 65504, values to offset and offset + 15 scale."""
    from ivonar_inference_b200 import KV4Cache

    T = TYPES[dtype]
    ends = [(-65504.0, 65504.0)]
    if dtype != "fp16":
        ends += [(0.0, 2.0**20), (-(2.0**20), 1.0), (1e5, 2e5), (-3e38, 3e38)]
    x = torch.stack([torch.linspace(0, 1, 64, dtype=torch.float64) * (high - low) + low for low, high in ends])[:, None].to(T).cuda()
    cache = KV4Cache(1, 1, 64, 8)
    at, starts = rows_of(1, [0], [len(ends)])
    cache.append(x, -x, at, starts)
    want = held(x)[:, 0], held(-x)[:, 0]
    assert float(want[0][0].max()) == 65536.0 and (dtype == "fp16" or float(want[0][4].max()) == 65504.0 * 14)
    for out in TYPES.values():
        for got, w in zip(cache.read(at, starts, len(ends), dtype=out), want):
            assert torch.equal(got[:, 0].cpu(), w.float().to(out))
    assert bool(cache.read(at, starts, len(ends), dtype=torch.float16)[0][0].isinf().any())


# ---- how near the result is, by its norm --------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,kv_heads,group,first,counts,window,sinks", [
    (64, 2, 1, [700, 30, 299], None, 0, 0),
    (128, 2, 4, [511, 64], None, 200, 4),
    (32, 2, 8, [400, 65, 7, 260], None, 0, 0),
    (128, 1, 16, [300, 511], None, 0, 0),
    (64, 2, 3, [200, 0, 77], [4, 7, 2], 0, 0),
    (64, 6, 2, [0, 130, 300], [250, 1, 40], 0, 0),
    (128, 2, 1, [300, 0], [150, 400], 120, 3),
    (32, 1, 4, [64], [200], 0, 0),
])
def test_errors_by_their_norm(dim, kv_heads, group, first, counts, window, sinks, dtype) -> None:
    """All outputs of a call against 64 bits. The scores here are sums of absolute products of up to about 16, each off by 2^-22 of that, in
    both directions as their parts are; with the weights' split and the sums that is 2^-18 of the output, and twice that is allowed
    (a weight held in 11 bits alone would be off by 2^-13 of it). 16 bits: a weight p_j is off by a rounding of 2^-11 at most, apart from the
    others', on values s (u - c) about the codes' middle, and the result by half a step of its type: the norms of
    2^-11 sqrt(sum_j (p_j s_j (u_j - c_j))^2) and of eps / 2 of the output are added, whose expected sizes are 0.58 of these."""
    from ivonar_inference_b200 import KV4Cache

    T, batch = TYPES[dtype], len(first)
    n = [1] * batch if counts is None else counts
    total = [a + c for a, c in zip(first, n)]
    cache = KV4Cache(batch, kv_heads, dim, max(total))
    filled(cache, total, seed=dim + group, spread=0.3)
    at, starts = rows_of(batch, first, n)
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(sum(n), kv_heads * group, dim, generator=gen, device="cuda").to(T)
    got = cache.attention(q, at, None if counts is None else starts, window=window, sinks=sinks).double().cpu()
    kk, vv, par = contents(cache.data, dim)
    error = size = rounding = 0.0
    r0 = 0
    for b in range(batch):
        L, mine = total[b], torch.arange(first[b], total[b])[:, None]
        where = torch.arange(L)
        hidden = where > mine
        if window:
            hidden |= (where <= mine - window) & (where >= sinks)
        x = q[r0:r0 + n[b]].double().cpu().unflatten(1, (kv_heads, group))
        score = torch.einsum("nhgd,hjd->hgnj", x, kk[b, :, :L]) * dim**-0.5
        weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
        value, scale, offset = vv[b, :, :L], par[b, :, :L, 2:3], par[b, :, :L, 3:4]
        want = torch.einsum("hgnj,hjd->nhgd", weight, value).flatten(1, 2)
        about = value - offset - scale * (8.0 - (where % 2)[:, None])
        error += float(((got[r0:r0 + n[b]] - want) ** 2).sum())
        size += float((want**2).sum())
        rounding += float(torch.einsum("hgnj,hjd->nhgd", weight**2, about**2).sum())
        r0 += n[b]
    bound = 2.0**-17 * size**0.5
    if T != torch.float32:
        bound += 2.0**-11 * rounding**0.5 + torch.finfo(T).eps / 2 * size**0.5
    assert error**0.5 <= bound, (error**0.5 / size**0.5, bound / size**0.5)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("group,counts", [(1, None), (8, None), (2, [3, 2]), (1, [90, 1]), (4, [100, 70])])
def test_queries_near_the_largest_of_their_type(group, counts, dtype) -> None:
    """Queries of 2^124 beside others whose products with the codes pass 32 bits while the scores do not: as the same queries and scale
    2^100 apart (the powers of two come off exactly)."""
    from ivonar_inference_b200 import KV4Cache

    T, n = TYPES[dtype], [1, 1] if counts is None else counts
    cache = KV4Cache(2, 1, 64, 120)
    gen = torch.Generator(device="cuda").manual_seed(2)
    k = torch.randn(240, 1, 64, generator=gen, device="cuda") * 1e-4
    at, starts = rows_of(2, [0, 0], [120, 120])
    cache.append(k, torch.randn(240, 1, 64, generator=gen, device="cuda"), at, starts)
    at, starts = rows_of(2, [15, 10], n)
    q = torch.randn(sum(n), group, 64, generator=gen, device="cuda").clamp(-7, 7) * 2.0**24
    q[::2, ::2] *= 2.0**-30
    q = q.to(T)
    for scale in (1e-3, 2.0**-22):
        want = cache.attention(q, at, None if counts is None else starts, scale=scale)
        got = cache.attention(q * 2.0**100, at, None if counts is None else starts, scale=scale * 2.0**-100)
        assert torch.isfinite(want).all() and torch.equal(got, want)
    # scores of 2^124 * 1e-4 * scale: finite
    assert torch.isfinite(cache.attention(q * 2.0**100, at, None if counts is None else starts, scale=0.125)).all()


# ---- the first call of a process ----------------------------------------------------------------
@gpu
@pytest.mark.parametrize("first", ["append", "read", "attention"])
def test_the_first_call_of_a_process_can_be_captured(first) -> None:
    """Before any eager call has loaded a kernel or allowed its shared memory: few rows, prompts and both in one graph."""
    import subprocess
    import sys
    from pathlib import Path

    code = f"""
import torch
from ivonar_inference_b200 import KV4Cache
cache = KV4Cache(2, 2, 64, 400)
x = torch.randn(302, 2, 64, device="cuda")
at = torch.tensor([0, 0], device="cuda")
starts = torch.tensor([0, 300, 302], dtype=torch.int32, device="cuda")
def step():
    order = ["append", "read", "attention"]
    order.remove({first!r})
    out = []
    for name in [{first!r}] + order:
        if name == "append":
            cache.append(x, x, at, starts)
        elif name == "read":
            out.append(cache.read(at, starts, 302)[0])
        else:
            out += [cache.attention(x, at, starts), cache.attention(x[:2], at), cache.attention(x[:40], at, starts)]
    return out
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
cache.check()
for a, b in zip(got, step()):
    assert torch.equal(a, b) and bool((a != 0).any())
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


# ---- refusals of the C entry points, before any launch ------------------------------------------
def test_the_queries_and_keys_of_a_step_refuse_bad_sizes() -> None:
    import ctypes

    from ivonar_inference_b200 import _native as native

    lib = native.library()
    buffer = ctypes.create_string_buffer(64)
    at = ctypes.addressof(buffer)  # never read: every call is refused before a launch
    desc = native.IvbLayerDesc()
    desc.rope = at
    good = dict(ld=256, batch=1, channels=64, latent=16, heads=2, head_dim=32, rope=16, nope=16, max_len=8)

    def call(entry=at, **kw):
        g = {**good, **kw}
        return lib.ivb_batch_qk(ctypes.byref(desc), entry, g["ld"], at, at, g["batch"], g["channels"], g["latent"], g["heads"], g["head_dim"], g["rope"],
                                g["nope"], g["max_len"], at, at, None)

    for wrong in (dict(batch=0), dict(max_len=0), dict(channels=32), dict(rope=15, nope=17), dict(rope=48, nope=-16), dict(rope=-16, nope=48), dict(ld=64 + 16 + 31),
                  dict(heads=0, channels=0), dict(heads=-2, head_dim=-32, rope=-16, nope=-16), dict(latent=-64, ld=64), dict(rope=16, nope=8),
                  dict(heads=2**26, channels=0, head_dim=64, rope=32, nope=32), dict(entry=None)):
        assert call(**wrong) == native.IVB_EINVAL and "ivb_batch_qk" in native.last_error(), wrong


def test_caches_whose_bytes_64_bits_do_not_count() -> None:
    import ctypes

    from ivonar_inference_b200 import _native as native

    lib, most = native.library(), 2**31 - 1
    for batch, heads, dim, length in ((most, most, 128, most), (most, most, 32, 4), (2**30, 2**30, 64, 1), (2**16, 2**16, 128, 2**30), (1, 1, 128, most),
                                      (2**10, 2**10, 128, most), (2**14, 1, 32, most)):
        want = batch * heads * 2 * ((length + 31) // 32) * 16 * (dim + 8)
        assert lib.ivb_kv4_bytes(batch, heads, dim, length) == (want if want < 2**63 else 0)
        buffer = ctypes.create_string_buffer(64)
        at = (ctypes.addressof(buffer) + 15) // 16 * 16  # never read: refused, or no rows
        rc = lib.ivb_kv4_append(ctypes.byref(native.IvbKv4Cache(at, batch, heads, dim, length)), at, at, native.IVB_F32, 0, 0, 0, 0, at, at, 0, None, None)
        assert rc == (native.IVB_OK if want < 2**63 else native.IVB_EINVAL)
