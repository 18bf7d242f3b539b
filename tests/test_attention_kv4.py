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
