"""Log probabilities on a B200 against 64 bits.

Tolerances, with V the vocabulary and n = V / 4096 + 1 turns of a thread (16 values each). A term e^d of S: d is off by 2^-22 of
itself (the difference, the reciprocal temperature, its product with log2 e and the product are rounded), so S by
2^-22 sum p |d| <= 2^-22 ln V of itself, and by 2^-22 for each exp2; a thread's sum has 16 n additions and n rescalings of two roundings
and an exp2 (2^-21), lanes, warps, CTAs and slices join it 5 + 3 + 3 + 1 times with as much:
    S is off by   s = 2^-22 (ln V + 1) + 16 n 2^-24 + (n + 12) 2^-21   of itself
    ln p by       s + 2^-22 |ln p| + 2^-22 (|ln p| is at least the difference over the temperature; ln S, the sum)
The entropy is ln S - sum p d: the second sum's terms are off by as much as S's and 2^-24 more, twice (of it and of S), and it is at most ln V:
    the entropy by   s + 2 (s + 2^-22) ln V + 2^-22 ln V
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def logits_of(rows, vocab, seed=0, dtype=torch.float32, size=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = size * torch.randn(rows, vocab, generator=gen, device="cuda")
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 4), generator=gen, device="cuda"), 9 * torch.rand(rows, 4, generator=gen, device="cuda"))
    return x.to(dtype), torch.randint(0, vocab, (rows,), generator=gen, device="cuda")


def expected(x, tokens, top, temperature):
    x = x.double()
    order = x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    ids = torch.argsort(-order, dim=1, stable=True)[:, :top]
    lp = torch.log_softmax(x / temperature, 1)
    p = lp.exp()
    entropy = -torch.where(p == 0, 0.0, p * lp).sum(1)
    two = tokens if tokens.ndim == 2 else tokens[:, None]
    inside = (two >= 0) & (two < x.shape[1])
    given = torch.where(inside, lp.gather(1, two.clamp(0, x.shape[1] - 1)), math.nan).view(tokens.shape)
    return given, entropy, lp.gather(1, ids), ids


def close(got, want, tol):
    got, want = got.double(), want.double()
    finite = torch.isfinite(want)
    assert torch.equal(got[~finite].nan_to_num(nan=7.0), want[~finite].nan_to_num(nan=7.0))
    assert bool(((got - want).abs() <= tol)[finite].all()), float(((got - want).abs() - tol)[finite].max())


def check(found, x, tokens, top=0, temperature=1.0):
    given, entropy, best, ids = expected(x, tokens, top, temperature)
    V = x.shape[1]
    n = V // 4096 + 1
    s = 2.0**-22 * (math.log(V) + 1) + 16 * n * 2.0**-24 + (n + 12) * 2.0**-21
    for got, want in ((found.tokens, given), (found.top, best)):
        assert got.dtype == torch.float32 and got.shape == want.shape
        close(got, want, s + 2.0**-22 * (want.abs() + 1))
    close(found.entropy, entropy, s + 2 * (s + 2.0**-22) * math.log(V) + 2.0**-22 * math.log(V))
    assert torch.equal(found.ids, ids)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (1, 31, 31), (5, 257, 0), (2, 300, 256), (70, 1000, 5), (1, 4096, 20), (3, 4097, 64),
                                            (700, 8195, 3), (1, 32768, 5), (2, 32768, 256), (33, 32768, 20), (9, 100003, 1), (1, 200001, 64)])
def test_against_64_bits(rows, vocab, top, dtype) -> None:
    from ivonar_inference_b200 import log_probs

    x, tokens = logits_of(rows, vocab, vocab + top, TYPES[dtype])
    for temperature in (1.0, 0.7):
        check(log_probs(x, tokens, top=top, temperature=temperature), x, tokens, top, temperature)


@pytest.mark.parametrize("top", [1, 7, 256])
@pytest.mark.parametrize("kind", ["equal", "levels", "ascending", "descending", "zeros", "last", "mostly banned"])
def test_orders_that_a_bound_does_not_help(kind, top) -> None:
    """Ties go to the lowest token, and rows whose every turn has larger values than the last are ranked all the same."""
    from ivonar_inference_b200 import log_probs

    for rows, vocab in ((2, 40007), (1, 9001), (600, 5000), (300, 33001), (1, 300001)):   # up to ten turns a CTA
        gen = torch.Generator(device="cuda").manual_seed(top)
        ramp = torch.arange(vocab, device="cuda") / vocab * 4
        x = {"equal": torch.full((rows, vocab), 1.25, device="cuda"),
             "levels": torch.randint(0, 3, (rows, vocab), generator=gen, device="cuda").float(),
             "ascending": ramp.expand(rows, vocab).contiguous(),
             "descending": -ramp.expand(rows, vocab).contiguous(),
             "zeros": torch.randint(0, 2, (rows, vocab), generator=gen, device="cuda").float() * -0.0,
             "last": torch.zeros(rows, vocab, device="cuda"),
             "mostly banned": torch.full((rows, vocab), -math.inf, device="cuda")}[kind]
        if kind == "zeros":
            x = torch.where(torch.rand(rows, vocab, generator=gen, device="cuda") < 0.5, 0.0, -0.0)
        if kind == "last":
            x[:, -300:] = torch.rand(rows, 300, generator=gen, device="cuda")
        if kind == "mostly banned":
            x[:, 17::vocab // 5] = torch.rand(x[:, 17::vocab // 5].shape, generator=gen, device="cuda")
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        check(log_probs(x, tokens, top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_with_special_values(dtype) -> None:
    from ivonar_inference_b200 import log_probs

    T = TYPES[dtype]
    x, _ = logits_of(12, 5003, 4, T)
    least, most = torch.finfo(T).min, torch.finfo(T).max
    x[0] = -math.inf                     # nothing is left
    x[1] = -math.inf
    x[1, 4001] = 3.0                     # one token is left
    x[2] = least                         # the type's lowest value throughout: any token
    x[3, ::2] = least
    x[4, 77] = math.nan
    x[5, 78] = math.inf
    x[6] = most
    x[7, 9] = most
    x[8, :4999] = -math.inf
    x[9, 100:] = least
    x[9, :100] = -math.inf
    x[10, 5] = -math.nan
    tokens = torch.tensor([4001, 4001, 5, 6, 7, 78, 5002, 9, 5000, 3, 5, 0], device="cuda")
    for temperature in (1.0, 1.5):
        check(log_probs(x, tokens, top=9, temperature=temperature), x, tokens, 9, temperature)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("temperature", [4.0, 1e30])
def test_logits_further_apart_than_fp32_reaches(temperature, dtype) -> None:
    """The lowest and the largest value of the type in one row: their difference is no fp32 number, that over the temperature is one."""
    from ivonar_inference_b200 import log_probs
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    x, tokens = logits_of(4, 5000, 6, TYPES[dtype])
    x[:, ::3] = torch.finfo(TYPES[dtype]).min
    x[:2, 70] = torch.finfo(TYPES[dtype]).max
    x[1, 9] = -math.inf
    given = torch.tensor([0, 9, 70, 71], device="cuda").expand(4, 4).contiguous()
    check(log_probs(x, given, 5, temperature), x, given, 5, temperature)
    parts = torch.stack([log_probs_slice(x[:, a:b], given, a, 5, temperature) for a, b in ((0, 60), (60, 5000))])
    check(log_probs_merge(parts, given, 5, temperature), x, given, 5, temperature)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 32768), (300, 9001), (3, 500)])
def test_tokens_that_are_nearly_certain(rows, vocab, dtype) -> None:
    """ln p of a token with nearly all of the probability, and the entropy then, to their own last bits: the others' sum r is off by s (above)
    of itself, ln(1 + r) by that and a rounding, and so is r's part of the entropy, whose terms d e^d have |d| of under 40 here (2^-22 each
    of d, twice, and of r)."""
    from ivonar_inference_b200 import log_probs
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    x, _ = logits_of(rows, vocab, 5, TYPES[dtype], size=1.0)
    x = x.clamp(-6, 6)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x[torch.arange(rows, device="cuda"), tokens] = torch.linspace(17, 30, rows, device="cuda").to(x.dtype)
    given, entropy, _, _ = expected(x, tokens, 0, 1.0)
    assert float(given.min()) > -32768 * math.exp(0.5 - 17) - 1e-3  # of normal logits e^x is e^0.5 on average
    n = vocab // 4096 + 1
    s = 2.0**-22 * (math.log(vocab) + 40) + 16 * n * 2.0**-24 + (n + 13) * 2.0**-21
    parts = torch.stack([log_probs_slice(x[:, a:b], tokens, a) for a, b in ((0, 100), (100, vocab))])
    for found in (log_probs(x, tokens), log_probs_merge(parts, tokens)):
        assert bool(((found.tokens.double() - given).abs() <= s * given.abs()).all())
        assert bool(((found.entropy.double() - entropy).abs() <= 2 * s * entropy.abs()).all())


@pytest.mark.parametrize("top", [0, 3])
def test_sums_at_the_border_of_what_counts_as_certain(top) -> None:
    """Warps whose sums lie within a few steps of 1.125 on both sides, where a lane's sum may be below it and its neighbour's not: a warp holds
    every eighth run of 128 values of a row of 4096, and each has one large value here."""
    from ivonar_inference_b200 import log_probs

    rows, vocab = 3000, 4096
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, 4, 8, 128, generator=gen, device="cuda", dtype=torch.float64)
    sure = torch.randint(0, 512, (rows, 8, 1), generator=gen, device="cuda")
    x = x.transpose(1, 2).reshape(rows, 8, 512)
    x.scatter_(2, sure, -math.inf)
    steps = torch.randint(-3, 4, (rows, 8, 1), generator=gen, device="cuda") * 2.0**-23
    x += torch.log(0.125 + steps) - torch.logsumexp(x, 2, keepdim=True)
    x.scatter_(2, sure, 0.0)
    x = x.view(rows, 8, 4, 128).transpose(1, 2).reshape(rows, vocab).float()
    # rounded to fp32 the logits move their sum by 2^-24 |x| of each term at most, |x| < 16 here: 0.125 * 16 * 2^-24 = 2^-23
    sums = x.double().view(rows, 4, 8, 128).exp().sum((1, 3))
    assert float((sums - 1.125).abs().max()) <= 5 * 2.0**-23 and bool((sums < 1.125).any()) and bool((sums > 1.125).any())
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    tokens[::2] = x[::2].argmax(1)
    check(log_probs(x, tokens, top=top), x, tokens, top)


@pytest.mark.parametrize("top", [1, 20, 64, 65, 256])
@pytest.mark.parametrize("rows,vocab", [(1, 32768), (2, 32768), (256, 32768), (3, 300)])
def test_rows_of_which_a_mask_leaves_little(rows, vocab, top) -> None:
    """Runs and single tokens allowed, fewer than `top` or more, at the beginning, the end, and where the warps' and the CTAs' parts meet."""
    from ivonar_inference_b200 import log_probs
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    for step, (begin, end, every) in enumerate(((0, 7, 1), (0, 100, 1), (vocab - 30, vocab, 1), (vocab // 8 - 3, vocab // 8 + 300, 1), (5, vocab, 1024),
                                                (vocab // 2, vocab, 2), (0, 1, 1))):
        for dtype, fill in ((torch.float32, -math.inf), (torch.bfloat16, -math.inf), (torch.float32, math.nan)):
            x, tokens = logits_of(rows, vocab, 40 + step, dtype, 2)
            masked = torch.ones(vocab, dtype=torch.bool, device="cuda")
            masked[begin:end:every] = False
            if fill == fill:
                x[:, masked] = fill
            else:  # these rows have no distribution, and NaN ranks with -inf
                x[:, masked] = -math.inf
                x[:, vocab // 3] = fill
            found = log_probs(x, tokens, top=top)
            check(found, x, tokens, top, 1.0)
            cut = vocab // 3 + 1
            parts = torch.stack([log_probs_slice(x[:, a:b], tokens, a, top) for a, b in ((0, cut), (cut, vocab)) if b > a])
            assert torch.equal(log_probs_merge(parts, tokens, top).ids, found.ids)


def test_tokens_of_every_kind() -> None:
    from ivonar_inference_b200 import log_probs

    x, _ = logits_of(5, 777, 1)
    tokens = torch.tensor([[-1, 0, 776], [777, 5, 5], [2**40, -(2**62), 1], [3, 2, 1], [776, 776, 776]], device="cuda")
    check(log_probs(x, tokens, top=2), x, tokens, 2)
    none = torch.empty(5, 0, dtype=torch.int64, device="cuda")
    found = log_probs(x, none, top=4)
    check(found, x, none, 4)
    many = torch.randint(0, 777, (5, 1000), device="cuda")
    check(log_probs(x, many), x, many)
    empty = log_probs(x[:0], tokens[:0], top=2)
    assert [tuple(t.shape) for t in empty] == [(0, 3), (0,), (0, 2), (0, 2)]


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_and_alignment(dtype) -> None:
    from ivonar_inference_b200 import log_probs

    wide, tokens = logits_of(40, 4500, 3, TYPES[dtype])
    for cut in (wide[:, 1:4001], wide[::3, 3:1000], wide[:, 7:12], wide[5:6, 4:4404], wide[:1].expand(40, 4500), wide[:, 2:3]):
        t = (tokens[: cut.shape[0]] % cut.shape[1]).contiguous()
        check(log_probs(cut, t, top=min(4, cut.shape[1])), cut, t, min(4, cut.shape[1]))
    odd, t = logits_of(9, 4501, 3, TYPES[dtype])   # every row begins elsewhere in its 16 bytes
    check(log_probs(odd, t, top=6), odd, t, 6)


def test_offsets_beyond_32_bits() -> None:
    from ivonar_inference_b200 import log_probs

    x = torch.empty(3, 1_500_000_001, dtype=torch.bfloat16, device="cuda")[:, :5000]
    part, tokens = logits_of(3, 5000, 3, torch.bfloat16)
    x.copy_(part)
    check(log_probs(x, tokens, top=3), x, tokens, 3)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab,cuts", [(5000, [0, 2500, 5000]), (300, [0, 7, 8, 200, 300]), (40001, [0, 128, 30000, 40001])])
def test_slices_of_a_vocabulary(vocab, cuts, dtype) -> None:
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    x, _ = logits_of(6, vocab, vocab, TYPES[dtype])
    x[1, : vocab // 2] = x[1, 0]
    x[2] = -math.inf
    x[3, cuts[1]:cuts[2]] = -math.inf
    tokens = torch.randint(-2, vocab + 2, (6, 3), device="cuda")
    for top in (0, 1, 256):
        parts = torch.stack([log_probs_slice(x[:, a:b], tokens, a, top, 0.9) for a, b in zip(cuts, cuts[1:])])
        check(log_probs_merge(parts, tokens, top, 0.9), x, tokens, top, 0.9)
        check(log_probs_merge(parts.flip(0).contiguous(), tokens, top, 0.9), x, tokens, top, 0.9)


def test_many_slices() -> None:
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    x, tokens = logits_of(2, 64 * 300, 1)
    parts = torch.stack([log_probs_slice(x[:, a:a + 300], tokens, a, 256) for a in range(0, 64 * 300, 300)])
    check(log_probs_merge(parts, tokens, 256), x, tokens, 256)


def test_slices_of_fewer_tokens_than_alternatives() -> None:
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    x, tokens = logits_of(5, 30, 1)
    x[1, :20] = -math.inf
    for top in (31, 64, 256):
        for cuts in ([0, 30], [0, 1, 17, 30], list(range(31))):
            parts = torch.stack([log_probs_slice(x[:, a:b], tokens, a, top) for a, b in zip(cuts, cuts[1:])])
            found = log_probs_merge(parts, tokens, top)
            check(found._replace(top=found.top[:, :30], ids=found.ids[:, :30]), x, tokens, 30)
            assert bool((found.ids[:, 30:] == -1).all()) and bool(found.top[:, 30:].isnan().all())


def test_slices_that_are_handed_in_more_than_once() -> None:
    """A part that comes `times` times: each alternative stands there as often, and each token counts as often in the sums."""
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    for vocab, top, times in ((5000, 256, 2), (5000, 256, 13), (5000, 20, 3), (5000, 200, 2), (300, 1, 9), (5000, 255, 8), (40, 256, 20)):
        x, tokens = logits_of(4, vocab, 2)
        x[1] = 0.0
        part = log_probs_slice(x, tokens, 0, top)
        found = log_probs_merge(part.expand(times, *part.shape).contiguous(), tokens, top)
        many = min(vocab, -(-top // times))
        given, _, best, ids = expected(x, tokens, many, 1.0)
        have = min(top, times * many)
        assert torch.equal(found.ids[:, :have], ids.repeat_interleave(times, 1)[:, :have]), (vocab, top, times)
        assert bool((found.ids[:, have:] == -1).all())
        # s of `check` is 1.1e-5 here, up to 20 joins of slices add 2^-21 each, and |ln p| < 30 adds 2^-22 of itself: 2.8e-5
        tol = 2.0**-15
        close(found.tokens, given - math.log(times), tol)
        close(found.top[:, :have], (best - math.log(times)).repeat_interleave(times, 1)[:, :have], tol)


def test_streams_graphs_and_repeated_calls() -> None:
    from ivonar_inference_b200 import log_probs

    x, tokens = logits_of(64, 32768, 2)
    want = log_probs(x, tokens, top=20)
    check(want, x, tokens, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = log_probs(x, tokens, top=20)
    side.synchronize()
    # two calls at once, and the same bits each time
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    graph, still = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        found = log_probs(still, tokens, top=20)
    for seed in (5, 6):
        fresh, _ = logits_of(64, 32768, seed)
        still.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        check(found, fresh, tokens, 20)
    reserved = torch.cuda.memory_allocated()
    log_probs(x, tokens)
    assert torch.cuda.memory_allocated() == reserved


def test_refusals() -> None:
    from ivonar_inference_b200 import KernelError, log_probs
    from ivonar_inference_b200.logprobs import log_probs_merge, log_probs_slice

    x, tokens = logits_of(4, 100)

    def refused(match, *args, **kwargs):
        with pytest.raises(ValueError, match=match):
            log_probs(*args, **kwargs)

    refused("contiguous", x.t(), tokens.new_zeros(100))
    refused("contiguous", x, tokens.repeat(2).view(4, 2).t().contiguous().t())
    refused("tokens must be", x, tokens.int())
    refused("tokens must be", x, tokens[:3])
    refused("tokens must be", x, tokens.cpu())
    refused("tokens must be", x, tokens[:, None, None])
    refused("top", x, tokens, top=-1)
    refused("top", x, tokens, top=257)
    refused("vocabulary of 100", x, tokens, top=101)
    for t in (0.0, -1.0, math.nan, math.inf):
        refused("temperature", x, tokens, temperature=t)
    refused("gradient", x.clone().requires_grad_(), tokens)
    with torch.no_grad():
        log_probs(x.clone().requires_grad_(), tokens)
    with torch.autograd.forward_ad.dual_level():
        refused("tangent", torch.autograd.forward_ad.make_dual(x, x), tokens)
    with pytest.raises(ValueError, match="from -1"):
        log_probs_slice(x, tokens, -1)
    parts = log_probs_slice(x, tokens, 0, 3)
    for bad in (parts, parts[None].long(), parts[None, :3], parts[None, :, :5]):
        with pytest.raises(ValueError, match="parts must be"):
            log_probs_merge(bad, tokens, 3)
    with pytest.raises((KernelError, ValueError)):
        log_probs_merge(parts[None], tokens, 3, 0.0)
