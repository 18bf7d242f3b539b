"""The batched decode with its attention blocks over the 4-bit key/value cache (`B200TensorParallel(cache="kv4")`, one rank)."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from test_gpu_kv4 import attended, contents, held, tolerance

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, LATENT, DENSE, VOCAB = 128, 4, 64, 256, 512
HEAD_DIM = HIDDEN // HEADS
ROPE = HEAD_DIM // 2
NOPE = HEAD_DIM - ROPE


class Rotary:
    head_dim = ROPE

    def rotate(self, x, offset=0):
        angle = (torch.arange(x.shape[1]) + offset)[:, None] * 10000.0 ** (-torch.arange(0, ROPE, 2) / ROPE)
        cos, sin = angle.cos()[None, :, None], angle.sin()[None, :, None]
        y = torch.empty_like(x)
        y[..., 0::2], y[..., 1::2] = x[..., 0::2] * cos - x[..., 1::2] * sin, x[..., 0::2] * sin + x[..., 1::2] * cos
        return y


def model_of(layers: int, seed: int):
    """A model with the attributes that the decoder reads, of attention blocks only."""
    gen = torch.Generator().manual_seed(seed)

    def linear(rows, cols, bias=True):
        codes = torch.randint(0, 3, (rows, cols // 4, 4), generator=gen, dtype=torch.uint8)
        packed = codes[..., 0] | codes[..., 1] << 2 | codes[..., 2] << 4 | codes[..., 3] << 6
        scales = (torch.rand(rows, math.ceil(cols / 128), generator=gen) * 0.1 + 0.05).half()
        return SimpleNamespace(packed_weight=packed, weight_scales=scales, in_features=cols, out_features=rows, group_size=128, eps=1e-5,
                               bias=torch.randn(rows, generator=gen) * 0.1 if bias else None)

    def norm():
        return SimpleNamespace(weight=1 + 0.1 * torch.randn(HIDDEN, generator=gen), eps=1e-6, clip=8.0)

    def block():
        mixer = SimpleNamespace(q_proj=linear(HIDDEN, HIDDEN), kv_down_proj=linear(LATENT, HIDDEN), k_rope_proj=linear(HEADS * ROPE, HIDDEN),
                                k_nope_up_proj=linear(HEADS * NOPE, LATENT), v_up_proj=linear(HIDDEN, LATENT), out_proj=linear(HIDDEN, HIDDEN),
                                rope_dim=ROPE, nope_dim=NOPE, latent_dim=LATENT, head_dim=HEAD_DIM, num_heads=HEADS, rope=Rotary())
        ffn = SimpleNamespace(gate_proj=linear(DENSE, HIDDEN), up_proj=linear(DENSE, HIDDEN), down_proj=linear(HIDDEN, DENSE))
        return SimpleNamespace(mixer=mixer, mixer_type="mla", mixer_norm=norm(), ffn_norm=norm(), ffn=ffn)

    return SimpleNamespace(config=SimpleNamespace(hidden_dim=HIDDEN, num_heads=HEADS), blocks=[block() for _ in range(layers)],
                           token_io=SimpleNamespace(projection=linear(VOCAB, HIDDEN, bias=False)), final_norm=norm())


@pytest.mark.parametrize("window,sinks", [(0, 0), (7, 2)])
def test_a_block_attends_to_what_its_cache_holds(window, sinks) -> None:
    """Every step of one block: queries and keys from the entry rows, what is written, and the attention's output, in 64 bits."""
    from ivonar_inference_b200.tp import B200TensorParallel

    batch, steps = 3, 40
    tp = B200TensorParallel(model_of(1, 0), 0, 1, batch=batch, max_len=steps, device="cuda:0", cache="kv4", window=window, sinks=sinks)
    gen = torch.Generator().manual_seed(1)
    for t in range(steps):
        tp.step(torch.randint(0, VOCAB, (batch,), generator=gen), sample=False)
        torch.cuda.synchronize()
        ld = tp.layers[0]["entry"].rows
        ent = tp.ent.view(-1)[: batch * ld].view(batch, ld).double().cpu()
        q = ent[:, :HIDDEN].view(batch, HEADS, HEAD_DIM)
        k_rope = ent[:, HIDDEN + LATENT:HIDDEN + LATENT + HEADS * ROPE].view(batch, HEADS, ROPE)
        angle = t * 10000.0 ** (-torch.arange(0, ROPE, 2).float() / ROPE)
        cos, sin = angle.cos().double(), angle.sin().double()

        def turned(x):
            return torch.stack([x[..., 0::2] * cos - x[..., 1::2] * sin, x[..., 0::2] * sin + x[..., 1::2] * cos], -1).flatten(-2)

        want_q = torch.cat([q[..., :NOPE], turned(q[..., NOPE:])], -1)
        want_k = torch.cat([tp.k_nope.double().cpu().view(batch, HEADS, NOPE), turned(k_rope)], -1)
        # two products and a sum in 32 bits, of sines that are within 2^-22 of these
        for got, want in ((tp.q, want_q), (tp.k, want_k)):
            assert float((got.double().cpu() - want).abs().max()) <= 2.0**-20 * float(want.abs().max()) * 2
        cache = tp.layers[0]["cache"]
        k, v, par = contents(cache.data, HEAD_DIM)
        assert torch.equal(k[:, :, t], held(tp.k)) and torch.equal(v[:, :, t], held(tp.v))
        for b in range(batch):
            want = attended(tp.q[b:b + 1], k[b], v[b], [t], HEAD_DIM**-0.5, window, sinks)
            most = float((par[b, :, : t + 1, 1].abs() + 15 * par[b, :, : t + 1, 0]).max())
            tol = tolerance(tp.q[b], most, float(v[b, :, : t + 1].abs().max()), HEAD_DIM**-0.5, want, torch.float32)
            assert bool(((tp.y[b].view(1, HEADS, HEAD_DIM).double().cpu() - want).abs() <= tol).all()), (t, b)
    assert int(tp.error.item()) == 0
    with pytest.raises(ValueError, match="capacity"):
        tp.step(torch.zeros(batch, dtype=torch.int64), sample=False)


@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 3)])
def test_streams_are_the_same_with_and_without_graphs(window, sinks) -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    model, batch = model_of(2, 3), 2
    prompts = torch.randint(0, VOCAB, (batch, 11), generator=torch.Generator().manual_seed(5))
    streams = []
    for graphs in (True, False):
        tp = B200TensorParallel(model, 0, 1, batch=batch, max_len=64, device="cuda:0", graphs=graphs, cache="kv4", window=window, sinks=sinks)
        tp.start(prompts, [1, 2], 0.8, 20, 1.1)
        first = tp.tokens.tolist()
        streams.append([first] + tp.decode(12).tolist() + tp.decode(20).tolist())
    assert streams[0] == streams[1]
    assert all(0 <= t < VOCAB for row in streams[0] for t in row)


def test_a_whole_window_is_the_unlimited_attention() -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    model, logits = model_of(2, 3), []
    feed = torch.randint(0, VOCAB, (9, 1), generator=torch.Generator().manual_seed(5))
    for window in (0, 9):
        tp = B200TensorParallel(model, 0, 1, max_len=16, device="cuda:0", cache="kv4", window=window)
        for t in range(9):
            tp.step(feed[t], sample=False)
        logits.append(tp.logits.clone())
    assert torch.equal(*logits)


def test_caches_that_are_refused() -> None:
    from ivonar_inference_b200.tp import B200TensorParallel

    model = model_of(1, 0)
    with pytest.raises(ValueError, match="cache"):
        B200TensorParallel(model, 0, 1, device="cuda:0", cache="int4")
    with pytest.raises(ValueError, match="window"):
        B200TensorParallel(model, 0, 1, device="cuda:0", window=8)
    with pytest.raises(ValueError, match="negative"):
        B200TensorParallel(model, 0, 1, device="cuda:0", cache="kv4", window=-1)
