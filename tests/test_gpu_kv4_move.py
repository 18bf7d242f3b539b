"""Sequences of the 4-bit key/value cache forked and compacted on a B200: every byte against a form on the host."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_kv4 import contents, filled, rows_of

pytestmark = pytest.mark.gpu


def places(dim: int) -> np.ndarray:
    """The position that each word of a tile belongs to (keys, values, scales and offsets in include/ivonar_b200.h's order)."""
    place, n = np.full(4 * (dim + 8), -1), dim // 32
    for p in range(16):
        for i in range(dim // 8):
            lane, half = (2 * (p // 4) + p % 2) * 4 + i // n, p // 2 % 2
            place[{32: 2 * lane + half, 64: 4 * lane + 2 * half + i % n, 128: 128 * half + 4 * lane + i % n}[dim]] = p
            place[2 * dim + 128 * (i // 8) + (4 * (i % 8) + p // 4) * 4 + p % 4] = p
        place[4 * dim + 2 * p], place[4 * dim + 2 * p + 1] = p, p
    assert (place >= 0).all()
    return place


def words(cache) -> np.ndarray:
    return cache.data.cpu().numpy().view("<u4").copy()


def random_cache(batch, heads, dim, max_len, seed):
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(batch, heads, dim, max_len)
    cache.data.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(seed))
    return cache


def device(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def forked(to, source, sources, lengths, dim, most):
    out, place = to.copy(), places(dim)
    for b, (s, n) in enumerate(zip(sources, lengths)):
        if 0 <= s < source.shape[0] and 0 < n <= most:
            at = 16 * np.arange(to.shape[2])[:, None] + place
            tiles = min(to.shape[2], source.shape[2])
            taken = at[:tiles] < n
            out[b, :, :tiles] = np.where(taken, source[s, :, :tiles], out[b, :, :tiles])
    return out


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("batch,heads,max_len", [(1, 1, 5), (4, 3, 100), (9, 2, 500), (300, 1, 40), (2, 5, 3001)])
def test_within_a_cache(batch, heads, max_len, dim) -> None:
    gen = np.random.default_rng(batch + dim)
    for kind in ("turned", "random", "one", "kept"):
        cache = random_cache(batch, heads, dim, max_len, batch)
        sources = {"turned": (np.arange(batch) + 1) % batch, "random": gen.integers(0, batch, batch), "one": np.zeros(batch, int),
                   "kept": np.where(gen.random(batch) < 0.5, -1, np.arange(batch)[::-1])}[kind]
        lengths = gen.integers(0, max_len + 1, batch)
        lengths[: min(batch, 7)] = np.minimum([max_len, 1, 16, 15, 17, 0, 32][: min(batch, 7)], max_len)
        before = words(cache)
        cache.fork(device(sources.tolist()), device(lengths.tolist()))
        cache.check()
        want = forked(before, before, [-1 if s == b else s for b, s in enumerate(sources)], lengths, dim, max_len)
        assert np.array_equal(words(cache), want), kind


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("batch,others,max_len,other_len", [(5, 3, 200, 70), (5, 3, 70, 200), (130, 1, 33, 33), (1, 40, 300, 300)])
def test_from_another_cache(batch, others, max_len, other_len, dim) -> None:
    gen = np.random.default_rng(dim)
    cache, other = random_cache(batch, 3, dim, max_len, 1), random_cache(others, 3, dim, other_len, 2)
    most = min(max_len, other_len)
    sources, lengths = gen.integers(0, others, batch), gen.integers(0, most + 1, batch)
    before, source = words(cache), words(other)
    cache.fork(device(sources.tolist()), device(lengths.tolist()), source=other)
    cache.check()
    assert np.array_equal(words(cache), forked(before, source, sources, lengths, dim, most))
    assert np.array_equal(words(other), source)


def test_what_a_fork_gives_is_what_was_written() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(3, 2, 64, 90)
    filled(cache, [90, 70, 50])
    k, v, _ = contents(cache.data, 64)
    cache.fork(device([1, 2, 0]), device([33, 50, 90]))
    got_k, got_v, _ = contents(cache.data, 64)
    for b, (s, n) in enumerate(((1, 33), (2, 50), (0, 90))):
        assert torch.equal(got_k[b][:, :n], k[s][:, :n]) and torch.equal(got_v[b][:, :n], v[s][:, :n])
        assert torch.equal(got_k[b][:, n:], k[b][:, n:]) and torch.equal(got_v[b][:, n:], v[b][:, n:])


def test_sources_and_lengths_that_are_not_there() -> None:
    cache = random_cache(6, 2, 64, 50, 3)
    before = words(cache)
    sources, lengths = [1, -(2**62), 0, 2**40, 3, 2], [51, 50, -5, 10, 50, 2**62]
    cache.fork(device(sources), device(lengths))
    with pytest.raises(ValueError):
        cache.check()
    cache.check()
    want = forked(before, before, [-1, -1, -1, -1, 3, -1], [0, 0, 0, 0, 50, 0], 64, 50)
    assert np.array_equal(words(cache), want)
    cache.fork(device([1, 1, 2, 3, 4, 6]), device([0, 0, 0, 0, 0, 3]))
    with pytest.raises(ValueError, match="cannot take"):
        cache.check()
    cache.fork(device([1, 1, 2, 3, 4, 5]), device([51] * 6))
    with pytest.raises(ValueError, match="capacity"):
        cache.check()
    small = random_cache(2, 2, 64, 20, 3)
    cache.fork(device([0] * 6), device([21] * 6), source=small)
    with pytest.raises(ValueError, match="capacity"):
        cache.check()
    assert np.array_equal(words(cache), want)


def test_many_sequences_in_one_cache() -> None:
    from ivonar_inference_b200 import KernelError

    cache = random_cache(4096, 1, 32, 20, 3)
    before = words(cache)
    turned = (np.arange(4096) + 5) % 4096
    cache.fork(device(turned.tolist()), device([19] * 4096))
    assert np.array_equal(words(cache), forked(before, before, turned, [19] * 4096, 32, 20))
    more, other = random_cache(5000, 1, 32, 20, 3), random_cache(2, 1, 32, 20, 3)
    with pytest.raises(KernelError, match="within one cache"):
        more.fork(device([0] * 5000), device([1] * 5000))
    before, source = words(more), words(other)
    more.fork(device([1] * 5000), device([20] * 5000), source=other)
    assert np.array_equal(words(more), forked(before, source, [1] * 5000, [20] * 5000, 32, 20))


def compacted(before, index, first, bounds, dim, max_len):
    out, place = before.copy(), places(dim)
    for b in range(before.shape[0]):
        for i in range(bounds[b + 1] - bounds[b]):
            r, p = bounds[b] + i, first[b] + i
            if r < 0 or r >= len(index):
                continue
            s = index[r]
            if 0 <= p < max_len and p <= s < max_len:
                to, by = np.flatnonzero(place == p % 16), np.flatnonzero(place == s % 16)
                out[b, :, p // 16, to] = before[b, :, s // 16, by]
    return out


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_words_of_a_position_are_in_one_order(dim) -> None:
    """What `compacted` relies on: a position's words come in the same order in every position of a tile."""
    cache = random_cache(1, 1, dim, 32, 1)
    k, v, par = contents(cache.data, dim)
    raw, place = words(cache), places(dim)
    moved = raw.copy()
    for p in range(16):
        moved[0, 0, 1, np.flatnonzero(place == p)] = raw[0, 0, 0, np.flatnonzero(place == 15 - p)]
    k2, v2, _ = contents(torch.from_numpy(moved.view(np.uint8)), dim)
    for got, want in ((k2, k), (v2, v)):
        assert torch.equal(got[0, 0, 16:].nan_to_num(7.0), want[0, 0, :16].flip(0).nan_to_num(7.0))


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("counts,first,max_len", [([1], [0], 1), ([3, 0, 1, 16], [2, 5, 30, 7], 64), ([40, 33, 17], [0, 1, 100], 200),
                                                  ([2500], [5], 5003), ([700, 1, 650], [3, 900, 16], 1500), ([5] * 200, list(range(200)), 256)])
def test_rows_move_up(counts, first, max_len, dim) -> None:
    gen = np.random.default_rng(dim + len(counts))
    for kind in ("kept", "behind", "any", "same"):
        cache = random_cache(len(counts), 2, dim, max_len, 5)
        index = []
        for n, a in zip(counts, first):
            p = a + np.arange(n)
            if kind == "kept":     # a part of what lies from the first row on, in order
                index += sorted(gen.choice(np.arange(a, max_len), n, replace=False).tolist())
            elif kind == "behind":  # moved as one
                index += np.minimum(p + 7, max_len - 1).tolist()
            elif kind == "any":
                index += [int(gen.integers(q, max_len)) if gen.random() < 0.9 else -1 for q in p]
            else:
                index += p.tolist()
        at, starts = rows_of(len(counts), first, counts)
        before = words(cache)
        cache.compact(device(index), at, starts)
        cache.check()
        want = compacted(before, index, first, [0] + np.cumsum(counts).tolist(), dim, max_len)
        assert np.array_equal(words(cache), want), kind


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("batch,rows", [(1, 30_000), (3, 9000), (300, 200), (700, 40)])
def test_sources_that_are_written_in_the_same_turn(batch, rows, dim) -> None:
    """Rows that move up by less than what is moved at a time: what one warp, or another CTA of the cluster, reads is written by its neighbour
    in the same turn. Many times over, as an order that is missing shows now and then."""
    cache = random_cache(batch, 2, dim, rows + 2200, 5)
    words_of = [np.flatnonzero(places(dim) == p) for p in range(16)]
    word = torch.from_numpy(np.stack(words_of)).cuda()   # [16 positions, words]
    at, starts = rows_of(batch, [0] * batch, [rows] * batch)

    def positions(data):   # [batch, heads, positions, words of one]
        return data.view(torch.int32)[..., word].flatten(2, 3)

    for by in (1, 15, 16, 17, 33, 250, 256, 2047, 2048):
        before = positions(cache.data)
        index = torch.arange(by, rows + by, device="cuda").repeat(batch)
        for _ in range(5):
            before[:, :, :rows] = before[:, :, by:rows + by].clone()
            cache.compact(index, at, starts)
        cache.check()
        assert torch.equal(positions(cache.data), before), by


def test_one_row_a_sequence() -> None:
    cache = random_cache(5, 3, 64, 40, 2)
    before = words(cache)
    index, first = [9, 39, -1, 3, 20], [0, 16, 5, 3, -1]
    cache.compact(device(index), device(first))
    cache.check()
    assert np.array_equal(words(cache), compacted(before, index, first, list(range(6)), 64, 40))


def test_rows_that_are_not_there() -> None:
    cache = random_cache(4, 2, 64, 50, 3)
    before = words(cache)
    first, bounds = [-2, 47, 2**62, -(2**63)], [-3, 4, 9, 11, 40]   # rows before and behind the call's
    index = [20, 7, -1, 30, 47, 48, 60, 2**40, 49, 5, 6, 1, 2, 3]
    cache.compact(device(index), device(first), torch.tensor(bounds, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        cache.check()
    want = compacted(before, index, first, bounds, 64, 50)
    assert np.array_equal(words(cache), want)
    for index, first, match in (([5], 6, "cannot take"), ([50], 6, "capacity"), ([60], 50, "capacity"), ([2**62], 2**62, "capacity")):
        one = random_cache(1, 2, 64, 50, 3)
        before = words(one)
        one.compact(device(index), device([first]))
        with pytest.raises(ValueError, match=match):
            one.check()
        one.check()
        assert np.array_equal(words(one), before)
    one.compact(device([-1]), device([60]))
    one.check()


def test_offsets_beyond_32_bits() -> None:
    from ivonar_inference_b200 import KV4Cache

    length = 1 << 24
    cache = KV4Cache(3, 1, 128, length)   # 2.3 GB a sequence
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(40, 1, 128, generator=gen, device="cuda")
    at, starts = rows_of(3, [0, 0, length - 40], [0, 0, 40])
    cache.append(x, -x, at, starts)
    cache.fork(device([2, -1, -1]), device([length, 0, 0]))
    cache.check()
    here, rows = rows_of(3, [length - 40, 0, 0], [40, 0, 0])
    want = cache.read(at, starts, rows=40)
    got = cache.read(here, rows, rows=40)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # 20 rows from the end to 30 places before it
    to, few = rows_of(3, [0, 0, length - 70], [0, 0, 20])
    cache.compact(torch.arange(length - 20, length, device="cuda"), to, few)
    cache.check()
    got = cache.read(to, few, rows=20)
    assert torch.equal(got[0], want[0][20:]) and torch.equal(got[1], want[1][20:])


def test_captured_and_on_another_stream() -> None:
    cache = random_cache(6, 2, 64, 80, 3)
    start = cache.data.clone()
    sources, lengths = device([1, 2, 3, 4, 5, 0]), device([80, 70, 33, 1, 64, 80])
    index, (at, starts) = device(list(range(20, 50))), rows_of(6, [0] * 6, [5] * 6)

    def both():
        cache.fork(sources, lengths)
        cache.compact(index, at, starts)

    both()
    want = cache.data.clone()
    cache.data.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(2):
        cache.data.copy_(start)
        graph.replay()
        assert torch.equal(cache.data, want)
    # the numbers are read when the graph runs
    cache.data.copy_(start)
    lengths.zero_()
    index.fill_(-1)
    graph.replay()
    assert torch.equal(cache.data, start)
    lengths.copy_(device([80, 70, 33, 1, 64, 80]))
    index.copy_(torch.arange(20, 50, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    side.synchronize()
    assert torch.equal(cache.data, want)


def test_refusals() -> None:
    from ivonar_inference_b200 import KV4Cache

    cache = KV4Cache(3, 2, 64, 40)
    n = device([0, 0, 0])
    for bad in (n.int(), n[:2], n.cpu(), torch.zeros(6, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(ValueError, match="sources must be"):
            cache.fork(bad, n)
        with pytest.raises(ValueError, match="lengths must be"):
            cache.fork(n, bad)
    for other in (KV4Cache(3, 1, 64, 40), KV4Cache(3, 2, 32, 40)):
        with pytest.raises(ValueError, match="source must be"):
            cache.fork(n, n, source=other)
    with pytest.raises(ValueError, match="shares memory"):
        cache.fork(n, n, source=cache.sequence(1))
    with pytest.raises(ValueError, match="shares memory"):
        cache.sequence(1).fork(n[:1], n[:1], source=cache)
    one = cache.sequence(0)
    one.fork(n[:1], device([40]), source=cache.sequence(2))
    assert torch.equal(cache.data[0], cache.data[2])
    cache.fork(n, n, source=KV4Cache(3, 2, 64, 40, data=cache.data))
    for bad in (n.int(), n[:, None], n.cpu(), torch.zeros(6, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(ValueError, match="index must be"):
            cache.compact(bad, n)
    with pytest.raises(ValueError, match="starts"):
        cache.compact(device([1, 2]), n)
    with pytest.raises(ValueError, match="positions"):
        cache.compact(n, n.int())
    with pytest.raises(ValueError, match="starts must be"):
        cache.compact(n, n, torch.zeros(4, device="cuda"))
    cache.compact(n[:0], n, torch.zeros(4, dtype=torch.int32, device="cuda"))
