"""One prompt answered many times, on a B200: a beginning that the sequences share, beams that are forked, log probabilities of what
they say (`B200TensorParallel(cache="kv4", prefix_len=)`, one rank)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv4 import attended, contents, tolerance
from test_gpu_kv4_decode import HEAD_DIM, HEADS, VOCAB, model_of
from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


def decoder(layers=2, batch=4, max_len=40, **kwargs):
    from ivonar_inference_b200.tp import B200TensorParallel

    return B200TensorParallel(model_of(layers, 3), 0, 1, batch=batch, max_len=max_len, device="cuda:0", cache="kv4", **kwargs)


def tokens(*shape, seed=0):
    return torch.randint(0, VOCAB, shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("window,sinks", [(0, 0), (12, 3)])
def test_a_block_attends_to_the_beginning_and_to_its_own(window, sinks) -> None:
    """What one block's attention gives at each step, against 64 bits over what both caches hold."""
    tp = decoder(layers=1, batch=3, window=window, sinks=sinks, prefix_len=30)
    tp.start(tokens(3, 1, seed=1), [1, 2, 3], 1.0, 1, prefix=tokens(21))
    assert tp.prefix_length.tolist() == [21] and tp.positions.tolist() == [1, 1, 1]
    for t in range(1, 25):
        tp.step(tokens(3, seed=t), sample=False)
        torch.cuda.synchronize()
        assert tp.places.tolist() == [21 + t] * 3
        pk, pv, pp = contents(tp.layers[0]["prefix"].data, HEAD_DIM)
        k, v, par = contents(tp.layers[0]["cache"].data, HEAD_DIM)
        for b in range(3):
            kk, vv, par_b = (torch.cat([x[0][:, :21], y[b][:, : t + 1]], 1) for x, y in ((pk, k), (pv, v), (pp, par)))
            want = attended(tp.q[b:b + 1], kk, vv, [21 + t], HEAD_DIM**-0.5, window, sinks)
            most = float((par_b[..., 1].abs() + 15 * par_b[..., 0]).max())
            tol = tolerance(tp.q[b], most, float(vv.abs().max()), HEAD_DIM**-0.5, want, torch.float32) + 2 * float(vv.abs().max()) * 2.0**-17
            assert bool(((tp.y[b].view(1, HEADS, HEAD_DIM).double().cpu() - want).abs() <= tol).all()), (t, b)
    assert int(tp.error.item()) == 0


def test_the_beginning_rotates_as_if_each_had_held_it() -> None:
    """Keys behind a beginning are those of the same tokens in a prompt of its own: one block's, from the same latents and positions."""
    whole, shared = decoder(layers=1, batch=2), decoder(layers=1, batch=2, prefix_len=16)
    text, own = tokens(16, seed=4), tokens(2, 5, seed=5)
    whole.start(torch.cat([text.expand(2, 16), own], 1), [1, 2], 1.0, 1)
    shared.start(own, [1, 2], 1.0, 1, prefix=text)
    a, b = whole.layers[0]["cache"], shared.layers[0]["cache"]
    # the embeddings and the projections of a token do not depend on the others: the first block's rows are the same to the last bit
    for x, y, z in zip(contents(a.data, HEAD_DIM), contents(b.data, HEAD_DIM), contents(shared.layers[0]["prefix"].data, HEAD_DIM)):
        assert torch.equal(x[:, :, 16:21], y[:, :, :5])
        assert torch.equal(x[0][:, :16], z[0][:, :16])


def beams(tp, width, steps, prefix=None):
    """Beam search: the `width` likeliest continuations, by the sum of log probabilities; every beam's tokens, sums and the sources taken."""
    tp.start(tokens(width, 3, seed=9)[:1].expand(width, 3), range(width), 1.0, 1, prefix=prefix)
    said = torch.zeros(width, 0, dtype=torch.int64, device="cuda")
    total = torch.full((width,), -1e30, device="cuda")
    total[0] = 0.0   # the beams are alike at first
    taken = []
    for _ in range(steps):
        found = tp.log_probs(torch.zeros(width, dtype=torch.int64, device="cuda"), top=width)
        check(found, tp.logits, torch.zeros(width, dtype=torch.int64, device="cuda"), width)
        total, best = (total[:, None] + found.top).flatten().topk(width)
        sources, chosen = best // width, found.ids.flatten()[best]
        tp.fork(sources)
        taken.append(sources)
        said = torch.cat([said[sources], chosen[:, None]], 1)
        tp.step(chosen, sample=False)
    return said, total, taken


@pytest.mark.parametrize("prefix_len", [0, 12])
def test_a_beam_search_ends_where_its_answers_read_anew_do(prefix_len) -> None:
    """Forks, the shared beginning and the log probabilities together: each beam, read from the start in a decoder of its own
    without a fork, has the same logits to the last bit, and its sum of log probabilities is that of its tokens one by one."""
    width, steps = 4, 9
    text = tokens(12, seed=2) if prefix_len else None
    tp = decoder(batch=width, prefix_len=prefix_len)
    said, total, taken = beams(tp, width, steps, text)
    assert len({tuple(row) for row in said.tolist()}) == width
    assert any(s.tolist() != list(range(width)) for s in taken[1:])   # beams did change places
    anew = decoder(batch=width, prefix_len=prefix_len)
    anew.start(tokens(width, 3, seed=9)[:1].expand(width, 3), range(width), 1.0, 1, prefix=text)
    sums = torch.zeros(width, device="cuda")
    for t in range(steps):
        sums += anew.log_probs(said[:, t].contiguous()).tokens
        anew.step(said[:, t], sample=False)
    assert torch.equal(anew.logits, tp.logits) and torch.equal(anew.positions, tp.positions)
    assert torch.allclose(sums, total, rtol=0, atol=steps * 2.0**-18 * float(total.abs().max()))


def test_sampled_streams_behind_a_beginning_with_and_without_graphs() -> None:
    streams = []
    for graphs in (True, False):
        tp = decoder(batch=3, max_len=64, prefix_len=20, graphs=graphs)
        tp.start(tokens(3, 4, seed=1), [1, 2, 3], 0.8, 20, 1.1, prefix=tokens(20, seed=6))
        first = tp.decode(10).clone()
        tp.fork(torch.tensor([1, -1, 1]))
        assert torch.equal(tp.history[0, :10], first[1])
        streams.append([first.tolist(), tp.decode(15).tolist()])
    assert streams[0] == streams[1]
    after = streams[0][1]
    assert after[0] != after[1] or after[1] != after[2]   # each has its own random numbers


def test_a_fork_of_the_latent_cache() -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    tp, anew = (B200TensorParallel(model_of(2, 3), 0, 1, batch=2, max_len=16, device="cuda:0") for _ in range(2))
    own = tokens(2, 5, seed=3)
    tp.start(own, [1, 2], 1.0, 1)
    anew.start(own[:1].expand(2, 5), [1, 2], 1.0, 1)
    tp.fork(torch.tensor([0, 0]))
    assert torch.equal(tp.logits, anew.logits)
    for t in range(4):
        both = tokens(2, seed=t)
        tp.step(both, sample=False)
        anew.step(both, sample=False)
        assert torch.equal(tp.logits, anew.logits)


@pytest.mark.parametrize("rank", [0, 1])
def test_log_probs_of_a_head_on_two_ranks(rank, monkeypatch) -> None:
    """Two ranks' slices of the head, the gather between them done here."""
    from ivonar_inference_b200.logprobs import log_probs_slice
    from ivonar_inference_b200.tp import B200TensorParallel

    ranks = [B200TensorParallel(model_of(1, 3), r, 2, batch=3, max_len=8, device="cuda:0") for r in range(2)]
    logits = 3 * torch.randn(3, VOCAB, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    for tp in ranks:
        tp.logits.copy_(logits[:, tp.v_range[0]:tp.v_range[1]])
    given = torch.randint(0, VOCAB, (3, 5), generator=torch.Generator("cuda").manual_seed(2), device="cuda")

    def gather(out, mine, group=None):
        for r, tp in enumerate(ranks):
            out[r].copy_(mine if r == rank else log_probs_slice(tp.logits, given, tp.v_range[0], 7, 0.7))

    monkeypatch.setattr(torch.distributed, "all_gather_into_tensor", gather)
    check(ranks[rank].log_probs(given, 7, 0.7), logits, given, 7, 0.7)


def test_refusals() -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    model = model_of(1, 0)
    with pytest.raises(ValueError, match="shared beginning"):
        B200TensorParallel(model, 0, 1, device="cuda:0", prefix_len=8)
    with pytest.raises(ValueError, match="shared beginning"):
        B200TensorParallel(model, 0, 1, device="cuda:0", cache="kv4", prefix_len=-1)
    tp = decoder(layers=1, batch=2, prefix_len=8)
    with pytest.raises(ValueError, match="capacity"):
        tp.start(tokens(2, 2), [1, 2], 1.0, 1, prefix=tokens(9))
    with pytest.raises(ValueError, match="capacity"):
        decoder(layers=1, batch=2).start(tokens(2, 2), [1, 2], 1.0, 1, prefix=tokens(1))
    for bad in (torch.tensor([0, 1], dtype=torch.int32), torch.tensor([0]), torch.tensor([0, 2])):
        with pytest.raises(ValueError, match="sources"):
            tp.fork(bad)


def test_a_fork_of_more_sequences_than_a_cache_takes_is_refused_before_anything_moves() -> None:
    many = decoder(layers=1, batch=4097, max_len=2, history_len=4)
    many.step(torch.arange(4097) % VOCAB, sample=False)
    before = [t.clone() for t in (many.tokens, many.positions, many.logits, many.layers[0]["cache"].data)]
    with pytest.raises(ValueError, match="4097 sequences"):
        many.fork(torch.zeros(4097, dtype=torch.int64))
    for was, now in zip(before, (many.tokens, many.positions, many.logits, many.layers[0]["cache"].data)):
        assert torch.equal(was, now)


@pytest.mark.parametrize("cache,prefix_len", [("kv4", 9), ("kv4", 0), ("latent", 0)])
def test_a_fork_takes_recurrent_states_too(cache, prefix_len) -> None:
    """Sequences that change places between recurrent and attention blocks go on as if each had read its tokens itself."""
    from ivonar_inference_b200.tp import B200TensorParallel
    from test_attention_kv4_decode import hybrid

    model, text = hybrid(["mamba", "mla", "mamba"], 4), tokens(prefix_len, seed=9) if prefix_len else None
    tp, anew = (B200TensorParallel(model, 0, 1, batch=4, max_len=24, device="cuda:0", cache=cache, prefix_len=prefix_len) for _ in range(2))
    read = tokens(4, 11, seed=1)
    tp.start(read[:, :6], [1, 2, 3, 4], 1.0, 1, prefix=text)
    for t in range(6, 11):
        tp.step(read[:, t], sample=False)
    sources = torch.tensor([2, 0, -1, 1])
    tp.fork(sources)
    mine = read[torch.tensor([2, 0, 2, 1])]
    anew.start(mine[:, :6], [1, 2, 3, 4], 1.0, 1, prefix=text)
    for t in range(6, 11):
        anew.step(mine[:, t], sample=False)
    assert torch.equal(tp.logits, anew.logits) and tp.positions.tolist() == anew.positions.tolist()
    for t in range(5):
        both = tokens(4, seed=20 + t)
        tp.step(both, sample=False)
        anew.step(both, sample=False)
        assert torch.equal(tp.logits, anew.logits), t
    assert int(tp.error.item()) == 0
