"""The 4-bit key/value cache on a B200: writing, reading back and attention against plain 64-bit forms.

Tolerances. Codes, scales and offsets are defined to the last bit, so what is read back has to be equal. For attention let
A = max over rows and heads of scale * sum_d |q_d| (|m| + 15 s), the largest sum of absolute products behind a score. The kernels split fp32
queries and weights in two fp16 (2^-22 of each value), sum at most 8 + 1 partial products of 16 in 32 bits on the tensor
cores (each addition off by at most 2^-22 of the partial sums, as their alignment truncates), take exp2 within 2^-22 and sum
weights in 32 bits over lanes, warps and blocks (chains of under 2^9 additions at the lengths here, 2^-24 each). A weight is
then off by at most A (2^-22 + 10 * 2^-22 + 3 * 2^-24) + 2^-22 + 2^-14 (the last for the chains, which is far from reached as they
round both ways: 2^-18 is what a chain of 2^9 gives with independent roundings, times 4), the output by twice that times the largest |v|:
    fp32: 2 vmax (A 2^-18 + 2^-17)
16-bit queries: the weights are rounded to fp16 once (2^-11 of each) and the output to its type (eps / 2 of it):
    2 vmax (A 2^-18 + 2^-17 + 2^-11) + eps / 2 |out|
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def quantised(x: torch.Tensor):
    """(offset, scale, code) of rows x in 64 bits; offset and scale are what fp16 holds."""
    x = x.double().cpu()
    m = x.amin(-1, keepdim=True).clamp(-65504, 65504).float().half().double()
    s = ((x.amax(-1, keepdim=True) - m) / 15).float().clamp(0, 65504).half().double()
    code = torch.where(s > 0, torch.round((x - m) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(x)).clamp(0, 15)
    return m, s, code


def held(x: torch.Tensor) -> torch.Tensor:
    m, s, code = quantised(x)
    y = m + s * code
    return torch.where(torch.isfinite(x.double().cpu()).all(-1, keepdim=True), y, torch.full_like(y, math.nan))


def contents(data: torch.Tensor, dim: int):
    """Keys and values [batch, heads, positions, dim] in 64 bits and the key (offset, scale), value (offset, scale) of a cache's storage."""
    raw = data.cpu().numpy()
    B, H, tiles = raw.shape[:3]
    words = raw.view("<u4").reshape(B, H, tiles, -1)
    par = np.ascontiguousarray(raw[..., 16 * dim:]).view("<f2").reshape(B, H, tiles * 16, 4).astype(np.float64)
    n, out = dim // 32, np.zeros((2, B, H, tiles * 16, dim))
    for p in range(16):
        for i in range(dim // 8):
            lane, half = (2 * (p // 4) + p % 2) * 4 + i // n, p // 2 % 2
            at = {32: 2 * lane + half, 64: 4 * lane + 2 * half + i % n, 128: 128 * half + 4 * lane + i % n}[dim]
            bt = 2 * dim + 128 * (i // 8) + (4 * (i % 8) + p // 4) * 4 + p % 4
            for ch in range(8):
                shift = 4 * (ch // 2) + 16 * (ch % 2)
                out[0, :, :, p::16, 8 * i + ch] = (words[..., at] >> shift) & 15
                out[1, :, :, p::16, 8 * i + ch] = (words[..., bt] >> shift) & 15
    k = par[..., 1:2] + par[..., 0:1] * out[0]
    v = par[..., 3:4] + par[..., 2:3] * out[1]
    return torch.from_numpy(k), torch.from_numpy(v), torch.from_numpy(par)


def attended(q, k, v, at, scale, window, sinks):
    """Attention in 64 bits of one sequence: q [n, H, D], k, v [Hkv, L, D], at [n] positions (None for idle rows: below 0)."""
    n, H, D = q.shape
    Hkv, L = k.shape[:2]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    j = torch.arange(L)
    for t in range(n):
        p = int(at[t])
        seen = (j <= p) & ((j > p - window) | (j < sinks) if window else torch.ones(L, dtype=torch.bool))
        if p < 0 or not seen.any():
            continue
        for h in range(H):
            kk, vv = k[h // (H // Hkv)][seen], v[h // (H // Hkv)][seen]
            w = torch.softmax(scale * (kk @ q[t, h].double().cpu()), 0)
            out[t, h] = w @ vv
    return out


def reach(x) -> float:
    """The largest |m| + 15 s over the rows of x."""
    m, s, _ = quantised(x)
    return float((m.abs() + 15 * s).max())


def tolerance(q, most, vmax, scale, want, dtype):
    A = abs(scale) * float(q.double().abs().sum(-1).max()) * most
    tol = 2 * vmax * (A * 2.0**-18 + 2.0**-17 + (0 if dtype == torch.float32 else 2.0**-11))
    return tol + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2) * want.abs()


def rows_of(batch, lengths, counts, device="cuda"):
    starts = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=device)
    return torch.tensor(lengths, dtype=torch.int64, device=device), starts


def filled(cache, lengths, seed=0, spread=1.0):
    """Writes positions 0 .. lengths[b] - 1 of every sequence; keys with levels of their own, values of unequal rows."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(lengths)
    if n == 0:
        return
    shape = (n, cache.kv_heads, cache.head_dim)
    k = torch.randn(shape, generator=gen, device="cuda") + torch.randn(shape[1:], generator=gen, device="cuda")
    v = torch.randn(shape, generator=gen, device="cuda") * torch.exp(spread * torch.randn(shape[:2] + (1,), generator=gen, device="cuda"))
    at, starts = rows_of(cache.batch, [0] * cache.batch, lengths)
    cache.append(k, v, at, starts)


def check_attention(cache, q, at, starts, dtype, scale=None, window=0, sinks=0, out=None):
    got = cache.attention(q, at, starts, scale=scale, window=window, sinks=sinks, out=out)
    scale = cache.head_dim**-0.5 if scale is None else scale
    k, v, par = contents(cache.data, cache.head_dim)
    first = at.cpu().tolist()
    bounds = list(range(cache.batch + 1)) if starts is None else starts.cpu().tolist()
    for b in range(cache.batch):
        r0, r1 = bounds[b], bounds[b + 1]
        if r1 == r0:
            continue
        rows = torch.arange(r1 - r0) + first[b]
        rows = torch.where(rows < cache.max_len, rows, -1)
        want = attended(q[r0:r1], k[b], v[b], rows, scale, window, sinks)
        vmax = float(v[b][:, : max(int(rows.max()) + 1, 1)].nan_to_num(0).abs().max())
        most = float((par[b][..., 1].abs() + 15 * par[b][..., 0]).nan_to_num(0, 0, 0).max())
        tol = tolerance(q[r0:r1], most, vmax, scale, want, dtype)
        diff = (got[r0:r1].double().cpu() - want).abs()
        assert bool((diff <= tol).all()), (b, float((diff - tol).max()), float(diff.max()))
    return got


# ---- writing and reading back -------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_rows_read_back_as_defined(dim, dtype) -> None:
    from ivonar_inference_b200 import KV4Cache

    T = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(dim)
    counts, first = [1, 0, 37, 16, 5], [3, 9, 0, 15, 58]
    cache = KV4Cache(5, 3, dim, 63)
    n = sum(counts)
    both = torch.randn(n + 2, 2, 3, dim, generator=gen, device="cuda")
    both *= torch.exp(2 * torch.randn(n + 2, 2, 3, 1, generator=gen, device="cuda"))
    both += torch.randn(n + 2, 2, 3, 1, generator=gen, device="cuda") * 3
    both[4] = 0.0                     # a row of zeros
    both[5] = -1.7                    # a constant
    both[6] *= 1e-6                   # scales below fp16's normal range
    both[7, 0, 1, 3] = 3e38 if dtype != "fp16" else 65504.0
    both[8, 1, 0, 2] = math.inf
    both[9, 0, 2, dim - 1] = math.nan
    both[10] = torch.arange(dim, device="cuda") * 1.0   # every quotient on or near a border
    both = both.to(T)
    k, v = both[:n, 0], both[:n, 1]   # strided rows
    at, starts = rows_of(5, first, counts)
    cache.append(k, v, at, starts)
    for out_dtype in TYPES.values():
        got_k, got_v = cache.read(at, starts, rows=n, dtype=out_dtype)
        for got, x in ((got_k, k), (got_v, v)):
            want = held(x).float().to(out_dtype)
            assert torch.equal(got.cpu().nan_to_num(-7.5), want.nan_to_num(-7.5))
            assert torch.equal(got.cpu().isnan(), want.isnan())
    # the storage is laid out as documented
    ck, cv, _ = contents(cache.data, dim)
    r = 0
    for b, (p, c) in enumerate(zip(first, counts)):
        for mine, x in ((ck, k), (cv, v)):
            want = held(x[r:r + c]).transpose(0, 1)
            assert torch.equal(mine[b][:, p:p + c].nan_to_num(-7.5), want.nan_to_num(-7.5))
        r += c
    cache.check()


def test_codes_are_the_real_quotients_rounded() -> None:
    """Many rows whose quotients come near the borders between codes, against 64 bits."""
    from ivonar_inference_b200 import KV4Cache

    gen = torch.Generator(device="cuda").manual_seed(1)
    n = 4096
    cache = KV4Cache(1, 8, 64, n)
    x = torch.randint(0, 31, (n, 8, 64), generator=gen, device="cuda") * 0.5
    x[..., 0], x[..., 1] = 0.0, 15.0
    x = x * torch.exp2(torch.randint(-3, 4, (n, 8, 1), generator=gen, device="cuda").float())
    x += x * torch.randint(-1, 2, x.shape, generator=gen, device="cuda") * 2.0**-23
    at, starts = rows_of(1, [0], [n])
    cache.append(x, -x, at, starts)
    k, v = cache.read(at, starts, rows=n)
    assert torch.equal(k.cpu(), held(x).float()) and torch.equal(v.cpu(), held(-x).float())


def test_rows_outside_are_left_alone_and_reported() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(4, 2, 64, 50)
    cache.data.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(3))
    before = cache.data.clone()
    at, starts = rows_of(4, [-2, 48, 2**40, -(2**62)], [3, 4, 1, 1])
    x = torch.randn(12, 2, 64, device="cuda")
    out = (torch.full((12, 2, 64), 9.0, device="cuda"), torch.full((12, 2, 64), 9.0, device="cuda"))
    cache.append(x, x, at, starts)
    with pytest.raises(ValueError, match="capacity"):
        cache.check()
    cache.check()
    k, _, _ = contents(cache.data, 64)
    assert torch.equal(k[0][:, 0], held(x[2])) and torch.equal(k[1][:, 48:50].transpose(0, 1), held(x[3:5]))
    # everything else is as it was: positions 50..63 of the storage too
    a, b = contents(before, 64), contents(cache.data, 64)
    for old, new in zip(a, b):
        same = (old == new) | (old.isnan() & new.isnan())
        same[0][:, 0] = True
        same[1][:, 48:50] = True
        assert bool(same.all())
    cache.read(at, starts, out=out)
    for o in out:
        left = torch.ones(12, dtype=torch.bool, device="cuda")
        left[2:5] = False
        assert bool((o[left] == 9.0).all()) and torch.equal(o[2:5].cpu(), held(x[2:5]).float())
    y = torch.full((12, 2, 64), 9.0, device="cuda")
    cache.attention(x, at, starts, out=y)
    with pytest.raises(ValueError, match="capacity"):
        cache.check()
    assert bool((y[[0, 1, 5, 6, 7, 8]] == 0.0).all()) and bool((y[9:] == 9.0).all()) and bool((y[2:5] != 9.0).all())


# ---- attention ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("group,window,sinks", [(1, 0, 0), (4, 0, 0), (3, 40, 4), (8, 1, 0), (16, 64, 33), (24, 33, 2)])
def test_single_tokens(dim, dtype, group, window, sinks) -> None:
    from ivonar_inference_b200 import KV4Cache

    lengths = [1, 15, 16, 17, 31, 32, 33, 64, 65, 200, 0]
    cache = KV4Cache(len(lengths), 2, dim, 200)
    filled(cache, lengths, seed=dim + group)
    gen = torch.Generator(device="cuda").manual_seed(7)
    q = (torch.randn(len(lengths), 2 * group, dim, generator=gen, device="cuda") * 1.5).to(TYPES[dtype])
    at = torch.tensor([n - 1 for n in lengths], device="cuda")
    got = check_attention(cache, q, at, None, TYPES[dtype], window=window, sinks=sinks)
    assert bool((got[-1] == 0).all())  # an idle row
    cache.check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,group,window,sinks", [(64, 1, 0, 0), (128, 4, 0, 0), (32, 2, 50, 3), (64, 3, 17, 0), (128, 1, 100, 40)])
def test_prompts_drafts_and_single_tokens_in_one_call(dim, dtype, group, window, sinks) -> None:
    from ivonar_inference_b200 import KV4Cache

    first, counts = [0, 30, 7, 100, 0, 61, 0], [150, 1, 5, 33, 0, 129, 1]
    total = [a + n for a, n in zip(first, counts)]
    cache = KV4Cache(7, 2, dim, 256)
    filled(cache, total, seed=dim)
    gen = torch.Generator(device="cuda").manual_seed(9)
    at, starts = rows_of(7, first, counts)
    q = (torch.randn(sum(counts), 2 * group, dim, generator=gen, device="cuda") * 1.5).to(TYPES[dtype])
    check_attention(cache, q, at, starts, TYPES[dtype], window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("batch,kv_heads,group,length", [(1, 1, 1, 3001), (1, 2, 8, 4097), (3, 1, 2, 2048), (40, 4, 1, 301)])
def test_long_axes_are_split_and_joined(batch, kv_heads, group, length, dtype) -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(batch, kv_heads, 64, length + 3)
    lengths = [max(1, length - 97 * b % length) for b in range(batch)]
    filled(cache, lengths, seed=length)
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = (torch.randn(batch, kv_heads * group, 64, generator=gen, device="cuda") * 2).to(TYPES[dtype])
    check_attention(cache, q, torch.tensor([n - 1 for n in lengths], device="cuda"), None, TYPES[dtype])
    check_attention(cache, q, torch.tensor([n - 1 for n in lengths], device="cuda"), None, TYPES[dtype], window=100, sinks=5)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts", [None, [1, 70, 3]])
def test_masked_places_may_hold_anything(dtype, counts) -> None:
    """NaN scales, infinities and the type's lowest value behind the last position and outside the window."""
    from ivonar_inference_b200 import KV4Cache

    T = TYPES[dtype]
    cache = KV4Cache(3, 2, 64, 160)
    n = [1, 70, 3] if counts is None else counts
    first = [0, 101, 40]
    filled(cache, [160] * 3, seed=2)
    clean = cache.data.clone()
    gen = torch.Generator(device="cuda").manual_seed(4)
    rows = 3 if counts is None else sum(n)
    q = torch.randn(rows, 4, 64, generator=gen, device="cuda").to(T)
    at, starts = rows_of(3, first, n)
    starts = None if counts is None else starts
    want = cache.attention(q, at, starts, window=20, sinks=2)
    bad = torch.tensor([math.nan, math.inf, -math.inf, -65504.0], dtype=torch.float16).view(torch.uint8)
    par = cache.data.view(3, 2, -1, 16 * 72)
    for b in range(3):
        last = first[b] + (1 if counts is None else n[b]) - 1
        low = first[b] - 19
        for p in range(160):
            if p > last or 2 <= p < low:
                par[b, :, p // 16, 1024 + 8 * (p % 16):1032 + 8 * (p % 16)] = bad.to("cuda").roll(2 * (p % 4))
    assert not torch.equal(clean, cache.data)
    assert torch.equal(cache.attention(q, at, starts, window=20, sinks=2), want)
    assert bool(torch.isfinite(want).all())


def test_a_visible_nan_reaches_its_rows_only() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(2, 2, 64, 64)
    filled(cache, [64, 64])
    x = torch.randn(2, 2, 64, device="cuda")
    x[0, 1, 5] = math.nan
    cache.append(x, x.abs(), torch.tensor([40, 40], device="cuda"))
    q = torch.randn(2, 4, 64, device="cuda")
    got = cache.attention(q, torch.tensor([50, 50], device="cuda"))
    assert bool(got[0, 2:].isnan().all()) and bool(torch.isfinite(got[0, :2]).all()) and bool(torch.isfinite(got[1]).all())
    q[1, 0, 3] = math.inf
    got = cache.attention(q, torch.tensor([39, 50], device="cuda"))
    assert bool(torch.isfinite(got[0]).all()) and bool(got[1, 0].isnan().all()) and bool(torch.isfinite(got[1, 1:]).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_scales_of_every_size(dtype) -> None:
    """Value rows from 1e-5 to 1e4, a dominant token with small values (an attention sink), rows without any range."""
    from ivonar_inference_b200 import KV4Cache

    gen = torch.Generator(device="cuda").manual_seed(8)
    n, T = 100, TYPES[dtype]
    for case in range(4):
        cache = KV4Cache(1, 1, 64, n)
        k = torch.randn(n, 1, 64, generator=gen, device="cuda")
        v = torch.randn(n, 1, 64, generator=gen, device="cuda")
        q = torch.randn(1, 2, 64, generator=gen, device="cuda")
        if case == 0:
            v *= 10.0 ** (9 * torch.rand(n, 1, 1, generator=gen, device="cuda") - 5)
        elif case == 1:   # the first token takes nearly all the weight, its values are a thousandth of the others'
            k[0] = q[0, :1] * 3
            v[0] *= 1e-3
        elif case == 2:
            v[:] = torch.randn(n, 1, 1, generator=gen, device="cuda")
            k[::2] = 0.25
        else:
            q *= 1e-4
            k *= 300
        q = q.to(T)
        at, starts = rows_of(1, [0], [n])
        cache.append(k, v, at, starts)
        check_attention(cache, q, torch.tensor([n - 1], device="cuda"), None, T)


def test_a_dominant_token_does_not_hide_a_large_value() -> None:
    """Values 2^20 apart under the wrong weights: the small rows must keep their bits although a large one is masked by its score."""
    from ivonar_inference_b200 import KV4Cache

    gen = torch.Generator(device="cuda").manual_seed(8)
    cache = KV4Cache(1, 1, 64, 40)
    q = torch.randn(1, 1, 64, generator=gen, device="cuda")
    k = 0.1 * torch.randn(40, 1, 64, generator=gen, device="cuda")
    k[7] = -40 * q[0]                # a weight of e^-300
    v = 1e-3 * torch.randn(40, 1, 64, generator=gen, device="cuda")
    v[7] = 1e4
    v[7, 0, :32] = -1e4
    at, starts = rows_of(1, [0], [40])
    cache.append(k, v, at, starts)
    got = cache.attention(q, torch.tensor([39], device="cuda"))
    kk, vv, _ = contents(cache.data, 64)
    want = attended(q, kk[0], vv[0], [39], 0.125, 0, 0)
    # the scores here are below 1 but for the hidden one, and the values below 4e-3
    assert float((got.double().cpu() - want).abs().max()) < 2 * 4e-3 * (16 * 2.0**-18 + 2.0**-17)


def test_scale_and_strides_and_alignment() -> None:
    from ivonar_inference_b200 import KV4Cache

    for dtype in TYPES.values():
        for dim in (32, 64, 128):
            cache = KV4Cache(3, 2, dim, 40)
            gen = torch.Generator(device="cuda").manual_seed(3)
            # one buffer of queries, keys and values per token; an odd row length leaves no row aligned
            fused = torch.randn(41 * 3, 8 * dim + 1, generator=gen, device="cuda").to(dtype)
            n = [40, 3, 25]
            at, starts = rows_of(3, [0, 0, 0], n)
            part = fused[: sum(n)]
            k = part[:, 1 + 4 * dim:1 + 6 * dim].unflatten(1, (2, dim))
            v = part[:, 1 + 6 * dim:].unflatten(1, (2, dim))
            cache.append(k, v, at, starts)
            kr, vr = cache.read(at, starts, rows=sum(n))
            assert torch.equal(kr.cpu(), held(k).float()) and torch.equal(vr.cpu(), held(v).float())
            # heads before rows
            q = part[:, 1:1 + 4 * dim].unflatten(1, (4, dim))
            turned = torch.empty(4, sum(n), dim, dtype=dtype, device="cuda").transpose(0, 1)
            check_attention(cache, q, at, starts, dtype, scale=0.31, out=turned)
            check_attention(cache, q.transpose(0, 1).contiguous().transpose(0, 1), at, starts, dtype, scale=-0.2)
            check_attention(cache, q, at, starts, dtype, scale=0.0)
            odd = torch.empty(sum(n), 4 * dim + 1, dtype=dtype, device="cuda")[:, 1:].unflatten(1, (4, dim))
            assert torch.equal(cache.attention(q, at, starts, out=odd), cache.attention(q.contiguous(), at, starts))
            both = torch.empty(sum(n), 2, 2, dim + 1, dtype=dtype, device="cuda")[..., 1:]
            cache.read(at, starts, out=(both[:, 0], both[:, 1]))
            assert torch.equal(both[:, 0].cpu(), held(k).float().to(dtype))


def test_offsets_beyond_32_bits() -> None:
    from ivonar_inference_b200 import KV4Cache

    length = 1 << 24
    cache = KV4Cache(3, 1, 128, length)   # 2.3 GB a sequence
    assert cache.nbytes > 6 * 2**30
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(90, 1, 128, generator=gen, device="cuda")
    at, starts = rows_of(3, [length - 30, 11, length - 30], [30, 30, 30])
    cache.append(x, -x, at, starts)
    k, v = cache.read(at, starts, rows=90)
    assert torch.equal(k.cpu(), held(x).float()) and torch.equal(v.cpu(), held(-x).float())
    q = torch.randn(3, 2, 128, generator=gen, device="cuda")
    got = cache.attention(q, at + 29, window=30)
    prompt = cache.attention(x.expand(90, 2, 128).contiguous(), at, starts, window=9)
    for b in range(3):
        mine = x[30 * b:30 * b + 30]
        kk, vv = held(mine).transpose(0, 1), held(-mine).transpose(0, 1)
        want = attended(q[b:b + 1], kk, vv, [29], 128**-0.5, 0, 0)
        tol = tolerance(q[b], reach(mine), reach(-mine), 128**-0.5, want, torch.float32)
        assert bool(((got[b].double().cpu() - want[0]).abs() <= tol[0]).all())
        # rows from the ninth on see written positions only
        want = attended(mine.expand(30, 2, 128), kk, vv, range(30), 128**-0.5, 9, 0)[8:]
        tol = tolerance(mine, reach(mine), reach(-mine), 128**-0.5, want, torch.float32)
        assert bool(((prompt[30 * b + 8:30 * b + 30].double().cpu() - want).abs() <= tol).all())
    cache.check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,batch,first,counts,group,window,sinks", [
    (64, 1, 600, [700], 2, 0, 0),          # one sequence, few tiles: clusters of four
    (128, 1, 0, [530], 1, 0, 0),
    (32, 1, 1000, [290], 4, 300, 70),
    (64, 4, 3, [513, 16, 17, 129], 1, 0, 0),
    (128, 3, 290, [257, 49, 1], 1, 100, 5),
    (64, 24, 0, [130, 3] * 12, 2, 33, 0),  # many tiles: one CTA each
])
def test_long_prompts(dim, batch, first, counts, group, window, sinks, dtype) -> None:
    """Prompts over more than one tile of rows and many of positions, with accumulators that are folded, against 64 bits."""
    from ivonar_inference_b200 import KV4Cache

    T, Hkv = TYPES[dtype], 2
    cache = KV4Cache(batch, Hkv, dim, first + max(counts) + 3)
    total = [first + n for n in counts]
    filled(cache, total, seed=dim + batch)
    gen = torch.Generator(device="cuda").manual_seed(9)
    q = (torch.randn(sum(counts), Hkv * group, dim, generator=gen, device="cuda") * 1.5).to(T)
    at, starts = rows_of(batch, [first] * batch, counts)
    got = cache.attention(q, at, starts, window=window, sinks=sinks)
    cache.check()
    k, v, par = contents(cache.data, dim)
    bounds = starts.tolist()
    for b in sorted({0, batch // 2, batch - 1}):
        n, L = counts[b], total[b]
        where, mine = torch.arange(L), torch.arange(first, L)[:, None]
        hidden = where > mine
        if window:
            hidden |= (where <= mine - window) & (where >= sinks)
        x = q[bounds[b]:bounds[b + 1]].double().cpu().unflatten(1, (Hkv, group))
        score = torch.einsum("nhgd,hjd->hgnj", x, k[b, :, :L]) * dim**-0.5
        weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
        want = torch.einsum("hgnj,hjd->nhgd", weight, v[b, :, :L]).flatten(1, 2)
        most = float((par[b, :, :L, 1].abs() + 15 * par[b, :, :L, 0]).max())
        tol = tolerance(q[bounds[b]:bounds[b + 1]], most, float(v[b, :, :L].abs().max()), dim**-0.5, want, T)
        diff = (got[bounds[b]:bounds[b + 1]].double().cpu() - want).abs()
        assert bool((diff <= tol).all()), (b, float(diff.max()))
        if T == torch.float32:
            # what folding is for: without it the error of the whole grows with the history, with it it stays near that of
            # 32-bit products (2^-24 a rounding, a chain of 2^5 products before each fold, cut towards zero: 2^-20)
            assert float(diff.norm() / want.norm()) < 2.0**-18


def test_long_histories_keep_fp32() -> None:
    """Many sequences, so that one warp walks many groups and folds its accumulators: the error stays that of 32-bit sums."""
    from ivonar_inference_b200 import KV4Cache

    for batch, heads, dim, length in ((600, 4, 64, 1500), (300, 8, 32, 1700), (300, 8, 128, 1300)):
        cache = KV4Cache(batch, heads, dim, length)
        filled(cache, [length] * batch, seed=dim)
        gen = torch.Generator(device="cuda").manual_seed(9)
        for group in (1, 6):
            q = torch.randn(batch, heads * group, dim, generator=gen, device="cuda")
            got = cache.attention(q, torch.full((batch,), length - 1, device="cuda"))
            for b in (0, batch - 1):
                k, v, _ = contents(cache.data[b:b + 1], dim)
                x = q[b].double().cpu().unflatten(0, (heads, group))
                weight = torch.softmax(torch.einsum("hgd,hjd->hgj", x, k[0, :, :length]) * dim**-0.5, -1)
                want = torch.einsum("hgj,hjd->hgd", weight, v[0, :, :length]).flatten(0, 1)
                assert float((got[b].double().cpu() - want).norm() / want.norm()) < 2.0**-18


def test_a_visible_nan_reaches_its_rows_only_in_prompts() -> None:
    from ivonar_inference_b200 import KV4Cache

    for dtype in TYPES.values():
        cache = KV4Cache(2, 2, 64, 400)
        filled(cache, [400, 400])
        x = torch.randn(2, 2, 64, device="cuda")
        x[0, 1, 5] = math.nan                       # the key of sequence 0, head 1, and the value of sequence 1, head 0
        y = torch.randn(2, 2, 64, device="cuda")
        y[1, 0, 7] = math.inf
        cache.append(x, y, torch.tensor([200, 200], device="cuda"))
        q = torch.randn(400, 4, 64, device="cuda").to(dtype)
        q[350, 3, 0] = math.inf
        at, starts = rows_of(2, [100, 100], [200, 200])
        got = cache.attention(q, at, starts)
        bad = torch.zeros(400, 4, dtype=torch.bool)
        bad[100:200, 2:] = True                     # rows at positions 200 .. 299 of sequence 0
        bad[300:400, :2] = True
        bad[350, 3] = True
        assert torch.equal(got.isnan().all(-1).cpu(), bad) and torch.equal(got.isnan().any(-1).cpu(), bad)
        got = cache.attention(q, at, starts, window=50)
        assert bool(torch.isfinite(got[160:200]).all()) and bool(got[100:150, 2:].isnan().all()) and bool(torch.isfinite(got[100:150, :2]).all())


def test_large_and_small_queries() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(1, 1, 64, 300)
    filled(cache, [300])
    q = torch.randn(40, 1, 64, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    at, starts = rows_of(1, [260], [40])
    want = cache.attention(q, at, starts, scale=0.125)
    for size in (2.0**120, 2.0**-60):
        # the queries' power of two comes off exactly, and the scale's product with log2 e is rounded alike
        assert torch.equal(cache.attention(q * size, at, starts, scale=0.125 / size), want)
        one = cache.attention(q[39:], at + 39, scale=0.125)
        assert torch.equal(cache.attention(q[39:] * size, at + 39, scale=0.125 / size), one)


def test_expanded_inputs() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(3, 2, 64, 40)
    x = torch.randn(1, 1, 64, device="cuda").expand(3, 2, 64)
    at = torch.tensor([3, 3, 3], device="cuda")
    cache.append(x, x, at)
    k, v = cache.read(at)
    assert torch.equal(k.cpu(), held(x).float()) and torch.equal(v, k)
    q = torch.randn(1, 4, 64, device="cuda")
    assert torch.equal(cache.attention(q.expand(3, 4, 64), at), cache.attention(q.repeat(3, 1, 1), at))


# ---- as they are used ---------------------------------------------------------------------------
def test_a_prompt_and_steps_together() -> None:
    """Prompts of several sequences written and attended to in one call, then single tokens: every output against 64 bits over
    what the cache holds, and the history never changed by later calls."""
    from ivonar_inference_b200 import KV4Cache

    gen = torch.Generator(device="cuda").manual_seed(6)
    n, steps, H, Hkv, D = [19, 64, 1, 33], 20, 4, 2, 64
    cache = KV4Cache(4, Hkv, D, 100)
    at, starts = rows_of(4, [0] * 4, n)
    written_k, written_v = [[] for _ in range(4)], [[] for _ in range(4)]

    def add(k, v, bounds):
        for b in range(4):
            written_k[b].append(held(k[bounds[b]:bounds[b + 1]]))
            written_v[b].append(held(v[bounds[b]:bounds[b + 1]]))

    def qkv(rows):
        f = torch.randn(rows, (H + 2 * Hkv) * D, generator=gen, device="cuda")
        return f[:, :H * D].unflatten(1, (H, D)), f[:, H * D:(H + Hkv) * D].unflatten(1, (Hkv, D)), f[:, (H + Hkv) * D:].unflatten(1, (Hkv, D))

    q, k, v = qkv(sum(n))
    cache.append(k, v, at, starts)
    outs = [(q, cache.attention(q, at, starts, window=24, sinks=2), at.clone(), starts.tolist())]
    add(k, v, starts.tolist())
    at = at + torch.tensor(n, device="cuda")
    for _ in range(steps):
        q, k, v = qkv(4)
        cache.append(k, v, at)
        outs.append((q, cache.attention(q, at, window=24, sinks=2), at.clone(), [0, 1, 2, 3, 4]))
        add(k, v, [0, 1, 2, 3, 4])
        at = at + 1
    cache.check()
    for b in range(4):
        kk, vv = torch.cat(written_k[b]).transpose(0, 1), torch.cat(written_v[b]).transpose(0, 1)
        for q, got, where, bounds in outs:
            rows = range(int(where[b]), int(where[b]) + bounds[b + 1] - bounds[b])
            want = attended(q[bounds[b]:bounds[b + 1]], kk, vv, list(rows), D**-0.5, 24, 2)
            tol = tolerance(q, 10.0, 5.0, D**-0.5, want, torch.float32)  # rows here reach less than 5 sigma either way
            assert bool(((got[bounds[b]:bounds[b + 1]].double().cpu() - want).abs() <= tol).all())


def test_results_are_the_same_every_time_on_any_stream_and_in_graphs() -> None:
    from ivonar_inference_b200 import KV4Cache

    gen = torch.Generator(device="cuda").manual_seed(6)
    caches, expected, inputs = [], [], []
    for i in range(2):
        cache = KV4Cache(3, 2, 64, 600)
        filled(cache, [500, 77, 300], seed=i)
        q = torch.randn(3, 4, 64, generator=gen, device="cuda")
        k, v = torch.randn(2, 3, 2, 64, generator=gen, device="cuda")
        at = torch.tensor([500, 77, 300], device="cuda")
        cache.append(k, v, at)
        expected.append(cache.attention(q, at))
        caches.append(cache)
        inputs.append((q, k, v, at))
    torch.cuda.synchronize()
    outs, graphs = [], []
    for cache, (q, k, v, at) in zip(caches, inputs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.append(k, v, at)
            out = cache.attention(q, at)
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    other = []
    for cache, (q, k, v, at), stream in zip(caches, inputs, reversed(streams)):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            other.append(cache.attention(q, at))
    torch.cuda.synchronize()
    for a, b, c in zip(expected, outs, other):
        assert torch.equal(a, b) and torch.equal(a, c)
    # a replay reads the positions of its time
    q, k, v, at = inputs[0]
    at.add_(1)
    graphs[0].replay()
    moved = outs[0].clone()
    assert torch.equal(moved, caches[0].attention(q, at)) and not torch.equal(moved, expected[0])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts", [[65], [64, 65], [33, 32, 64, 65, 1, 31, 66]])
def test_between_few_rows_and_prompts(counts, dtype) -> None:
    """Sequences on either side of where the kernels change, with few sequences in a call and with many."""

    from ivonar_inference_b200 import KV4Cache

    lengths = [90 - 11 * i for i in range(len(counts))]
    cache = KV4Cache(len(counts), 6, 64, 300)
    filled(cache, [n + c for n, c in zip(lengths, counts)], seed=3)
    at, starts = rows_of(len(counts), lengths, counts)
    gen = torch.Generator(device="cuda").manual_seed(12)
    q = torch.randn(sum(counts), 6, 64, generator=gen, device="cuda").to(TYPES[dtype])
    check_attention(cache, q, at, starts, TYPES[dtype])


@pytest.mark.parametrize("captured", [False, True])
def test_calls_that_follow_one_another_need_no_wait_between_them(captured) -> None:
    """Each call's inputs are the last one's outputs, prompts and few rows in one call: as with a wait after every call."""

    from ivonar_inference_b200 import KV4Cache

    counts, lengths = [1, 100, 3, 40, 1, 70, 2], [400, 0, 250, 130, 7, 300, 511]
    at, starts = rows_of(7, lengths, counts)
    rows = sum(counts)
    gen = torch.Generator(device="cuda").manual_seed(13)
    start = torch.randn(rows, 8, 64, generator=gen, device="cuda")
    results = []
    for wait in (True, False):
        cache = KV4Cache(7, 4, 64, 1100)
        filled(cache, lengths, seed=4)
        x, where, history = start.clone(), at.clone(), []
        moves = torch.tensor(counts, device="cuda")

        def step():
            cache.append(x[:, :4], x[:, 4:], where, starts)
            y = cache.attention(x, where, starts)
            if wait:
                torch.cuda.synchronize()
            cache.attention(y, where, starts, out=x)
            where.add_(moves)
            k, v = cache.read(where - moves, starts, rows)
            if wait:
                torch.cuda.synchronize()
            return y, k, v

        if captured and not wait:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            for _ in range(5):
                graph.replay()
                history.append([t.clone() for t in (*out, x)])
        else:
            for _ in range(5):
                history.append([t.clone() for t in (*step(), x)])
        torch.cuda.synchronize()
        results.append(history)
    for waited, free in zip(*results):
        for a, b in zip(waited, free):
            assert torch.isfinite(a).all() and torch.equal(a, b)


def test_a_graph_that_joins_streams_before_each_call() -> None:
    from ivonar_inference_b200 import KV4Cache

    counts, lengths = [1, 90, 2], [300, 10, 77]
    at, starts = rows_of(3, lengths, counts)
    gen = torch.Generator(device="cuda").manual_seed(14)
    base = torch.randn(sum(counts), 4, 64, generator=gen, device="cuda")
    side = torch.cuda.Stream()

    def step(cache, x):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        k = x[:, :2] * 2
        with torch.cuda.stream(side):
            v = x[:, 2:] + 1
            q = torch.zeros_like(x)
        main.wait_stream(side)
        cache.append(k, v, at, starts)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            q.add_(x)
            held = cache.read(at, starts, sum(counts))
        q2 = x * 0.5
        main.wait_stream(side)
        out = cache.attention(q, at, starts) + cache.attention(q2, at, starts)
        return out, *held

    caches = [KV4Cache(3, 2, 64, 400) for _ in range(2)]
    for cache in caches:
        filled(cache, lengths, seed=5)
    x = base.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], x)
    for i in range(3):
        x.copy_(base * (i + 1))
        graph.replay()
        want = step(caches[1], x)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_one_sequence_of_a_cache() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(3, 2, 32, 64)
    filled(cache, [20, 20, 20])
    one = cache.sequence(1)
    x = torch.randn(2, 2, 32, device="cuda")
    at, starts = rows_of(1, [20], [2])
    before = cache.data.clone()
    one.append(x, x, at, starts)
    assert torch.equal(cache.data[0], before[0]) and torch.equal(cache.data[2], before[2])
    q = torch.randn(3, 2, 32, device="cuda")
    whole = cache.attention(q, torch.tensor([19, 21, 19], device="cuda"))
    assert torch.equal(one.attention(q[1:2], torch.tensor([21], device="cuda")), whole[1:2])


def test_calls_that_are_refused() -> None:
    from ivonar_inference_b200 import KV4Cache

    with pytest.raises(ValueError, match="head_dim"):
        KV4Cache(1, 1, 48, 16)
    with pytest.raises(ValueError, match="positive"):
        KV4Cache(1, 0, 64, 16)
    with pytest.raises(ValueError, match="data must be"):
        KV4Cache(1, 1, 64, 16, data=torch.zeros(1, 1, 2, 100, dtype=torch.uint8, device="cuda"))
    cache = KV4Cache(2, 2, 64, 16)
    at = torch.zeros(2, dtype=torch.int64, device="cuda")
    x = torch.zeros(2, 2, 64, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for wrong in (x[:, :1], x[..., :32], x[0], x.double(), x.cpu(), x.transpose(1, 2).contiguous().transpose(1, 2), x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            cache.append(wrong, x, at)
        with pytest.raises(ValueError):
            cache.append(x, wrong, at)
        if wrong.ndim != 3 or wrong.shape[1] != 1:
            with pytest.raises(ValueError):
                cache.attention(wrong, at)
        with pytest.raises(ValueError):
            cache.read(at, out=(x, wrong))
    with pytest.raises(ValueError, match="type"):
        cache.append(x, x.half(), at)
    with pytest.raises(ValueError, match="positions"):
        cache.append(x, x, at.int())
    with pytest.raises(ValueError, match="positions"):
        cache.append(x, x, at[:1])
    with pytest.raises(ValueError, match="starts"):
        cache.append(x, x, at, starts.long())
    with pytest.raises(ValueError, match="starts"):
        cache.append(x, x, at, starts[:2])
    with pytest.raises(ValueError, match="need starts"):
        cache.attention(torch.zeros(3, 2, 64, device="cuda"), at)
    with pytest.raises(ValueError, match="multiple"):
        cache.attention(torch.zeros(2, 3, 64, device="cuda"), at)
    with pytest.raises(ValueError, match="negative"):
        cache.attention(x, at, window=-1)
    with pytest.raises(ValueError, match="overlap"):
        cache.attention(x, at, out=torch.zeros(1, 2, 64, device="cuda").expand(2, 2, 64))
    with pytest.raises(ValueError, match="disagree"):
        cache.attention(x, at, starts, out=torch.zeros(3, 2, 64, device="cuda"))
    with pytest.raises(ValueError, match="rows has to be given"):
        cache.read(at, starts)
    with pytest.raises(ValueError, match="dtype"):
        cache.read(at, dtype=torch.float64)
    with pytest.raises(IndexError):
        cache.sequence(2)
    with pytest.raises(RuntimeError, match="error word"):
        KV4Cache(2, 2, 64, 16, data=cache.data).check()
    empty = torch.zeros(0, 2, 64, device="cuda")
    cache.append(empty, empty, at, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert cache.attention(empty, at, torch.zeros(3, dtype=torch.int32, device="cuda")).shape == (0, 2, 64)
    assert bool((cache.data == 0).all())
