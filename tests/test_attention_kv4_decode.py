"""The batched decode over the 4-bit cache with recurrent blocks beside the attention's, and with its heads split over two ranks."""

from __future__ import annotations

import threading
from types import SimpleNamespace

import pytest
import torch

from test_gpu_kv4 import attended, contents, held, tolerance
from test_gpu_kv4_decode import HEAD_DIM, HEADS, HIDDEN, VOCAB, model_of

pytestmark = pytest.mark.gpu

STATE, TAPS = 16, 4


def hybrid(kinds: list[str], seed: int):
    """`model_of` with recurrent blocks where `kinds` says "mamba"."""
    model, gen = model_of(len(kinds), seed), torch.Generator().manual_seed(seed + 1)

    def linear(rows):
        codes = torch.randint(0, 3, (rows, HIDDEN // 4, 4), generator=gen, dtype=torch.uint8)
        return SimpleNamespace(packed_weight=codes[..., 0] | codes[..., 1] << 2 | codes[..., 2] << 4 | codes[..., 3] << 6, group_size=128, eps=1e-5,
                               weight_scales=(torch.rand(rows, 1, generator=gen) * 0.1 + 0.05).half(), in_features=HIDDEN, out_features=rows,
                               bias=torch.randn(rows, generator=gen) * 0.1)

    for block, kind in zip(model.blocks, kinds):
        if kind == "mamba":
            block.mixer_type = "mamba"
            block.mixer = SimpleNamespace(
                state_dim=STATE, conv_kernel_size=TAPS, dt_min=0.001, dt_max=0.1, in_proj=linear(2 * HIDDEN), bc_dt_proj=linear(3 * HEADS * STATE),
                out_proj=linear(HIDDEN), log_decay=torch.rand(HEADS, STATE, generator=gen) * 0.5 - 1, theta=torch.rand(HEADS, STATE, generator=gen) * 3,
                skip=1 + 0.1 * torch.randn(HEADS, HEAD_DIM, generator=gen), conv_weight=0.3 * torch.randn(HIDDEN, 1, TAPS, generator=gen),
                conv_bias=0.01 * torch.randn(HIDDEN, generator=gen))
    return model


def attention_of_the_last_step(tp, layer: int, t: int, window: int, sinks: int) -> None:
    """What the last attention block wrote and gave for position t, against 64 bits."""
    heads = tp.heads_local
    cache = tp.layers[layer]["cache"]
    k, v, par = contents(cache.data, HEAD_DIM)
    assert torch.equal(k[:, :, t], held(tp.k)) and torch.equal(v[:, :, t], held(tp.v))
    for b in range(tp.batch):
        want = attended(tp.q[b:b + 1], k[b], v[b], [t], HEAD_DIM**-0.5, window, sinks)
        most = float((par[b, :, : t + 1, 1].abs() + 15 * par[b, :, : t + 1, 0]).max())
        tol = tolerance(tp.q[b], most, float(v[b, :, : t + 1].abs().max()), HEAD_DIM**-0.5, want, torch.float32)
        assert bool(((tp.attended[b].view(1, heads, HEAD_DIM).double().cpu() - want).abs() <= tol).all()), (t, b)


def keeping(base):
    """`base` that keeps what its last attention block gave (the next mixer writes to the same place)."""

    class Keeping(base):
        def _attend_kv4(self, desc, layer, ld):
            super()._attend_kv4(desc, layer, ld)
            self.attended = self.y.clone()

    return Keeping


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2)])
def test_attention_between_recurrent_blocks(window, sinks) -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    model, batch, steps = hybrid(["mamba", "mla", "mamba"], 4), 3, 30
    feed = torch.randint(0, VOCAB, (steps, batch), generator=torch.Generator().manual_seed(2))
    kv4 = keeping(B200TensorParallel)(model, 0, 1, batch=batch, max_len=steps, device="cuda:0", cache="kv4", window=window, sinks=sinks)
    latent = B200TensorParallel(model, 0, 1, batch=batch, max_len=steps, device="cuda:0")
    for t in range(steps):
        kv4.step(feed[t], sample=False)
        latent.step(feed[t], sample=False)
        attention_of_the_last_step(kv4, 1, t, window, sinks)
        # the block before the attention does not know of its cache, the one after does
        for name, state in kv4.layers[0]["state"].items():
            assert torch.equal(state, latent.layers[0]["state"][name]), (t, name)
        assert all(bool(torch.isfinite(s).all()) for s in kv4.layers[2]["state"].values()) and bool(torch.isfinite(kv4.logits).all())
    assert not torch.equal(kv4.layers[2]["state"]["ssm_state"], latent.layers[2]["state"]["ssm_state"])
    assert int(kv4.error.item()) == 0


def test_streams_of_a_hybrid_with_and_without_graphs() -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    model = hybrid(["mamba", "mla", "mla", "mamba"], 5)
    prompts = torch.randint(0, VOCAB, (3, 9), generator=torch.Generator().manual_seed(5))
    streams = []
    for graphs in (True, False, True):
        tp = B200TensorParallel(model, 0, 1, batch=3, max_len=48, device="cuda:0", graphs=graphs, cache="kv4", window=12, sinks=1)
        for _ in range(2):  # the second start finds the first one's cache
            tp.start(prompts, [1, 2, 3], 0.8, 20, 1.1)
            streams.append([tp.tokens.tolist()] + tp.decode(10).tolist() + tp.decode(20).tolist())
    assert all(s == streams[0] for s in streams)


def test_two_ranks_split_the_heads() -> None:
    """Both ranks of one process, a thread each, with the sums over ranks made on the host between launches. The first block's keys and
    values are those of one rank to the last bit, its outputs within the attention's tolerance; the logits differ by the order of sums, after
    which a code of the activations (8 bits, root mean square over 16 of 127 steps) is another one at the most: 2^-4 of their norm."""
    from ivonar_inference_b200.tp import B200TensorParallel

    model, batch, steps = hybrid(["mla", "mamba", "mla"], 6), 2, 24
    feed = torch.randint(0, VOCAB, (steps, batch), generator=torch.Generator().manual_seed(2))
    meet, parts, failed = threading.Barrier(2, timeout=120), [None, None], []

    class Rank(keeping(B200TensorParallel)):
        def _all_reduce(self, t, op):
            parts[self.rank] = t.clone()
            torch.cuda.synchronize()
            meet.wait()
            t.copy_(torch.maximum(*parts) if op == torch.distributed.ReduceOp.MAX else parts[0] + parts[1])
            torch.cuda.synchronize()
            meet.wait()

    one = keeping(B200TensorParallel)(model, 0, 1, batch=batch, max_len=steps, device="cuda:0", cache="kv4", window=10, sinks=2)
    ranks = [Rank(model, r, 2, batch=batch, max_len=steps, device="cuda:0", cache="kv4", window=10, sinks=2) for r in range(2)]

    def run(tp, t):
        try:
            with torch.cuda.device(0):
                tp.step(feed[t], sample=False)
                torch.cuda.synchronize()
        except BaseException as error:  # a thread's failure ends the other's wait and the test
            failed.append(error)
            meet.abort()

    half = HEADS // 2
    for t in range(steps):
        one.step(feed[t], sample=False)
        threads = [threading.Thread(target=run, args=(tp, t)) for tp in ranks]
        for thread in threads:
            thread.start()
        for thread in threads:
            thread.join()
        assert not failed, failed
        for r, tp in enumerate(ranks):
            assert torch.equal(tp.layers[0]["cache"].data, one.layers[0]["cache"].data[:, r * half:(r + 1) * half])
            attention_of_the_last_step(tp, 2, t, 10, 2)
        logits = torch.cat([tp.logits for tp in ranks], 1)
        assert float((logits - one.logits).norm()) <= 2.0**-4 * float(one.logits.norm()), t
