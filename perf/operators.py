"""What is measured of the 4-bit key/value cache: writing rows into it and reading them back, and causal attention over it
with a sliding window and visible first tokens ("sinks").

The cache of one call is one uint8 tensor ``data`` [batch, kv_heads, tiles, 16 * (D + 8)]: a tile holds 16 positions of one
key/value head as 8 D bytes of key codes, 8 D bytes of value codes and 16 x 4 fp16 (key scale, key offset, value scale,
value offset). A row x of D values is kept as x = offset + scale * code with codes 0..15:

    offset = fp16(min x),  scale = fp16((max x - offset) / 15),  code = round((x - offset) / scale), clipped to 0..15

Codes are packed in 32-bit words of 8 channels, channel 2 j in nibble j and channel 2 j + 1 in nibble j + 4 (j = 0..3). Word i
of position p (0..15) of a tile, in words from the start of the tile's codes, with n = D / 32:

    keys:   lane = (2 (p / 4) + p % 2) * 4 + i / n, half = p / 2 % 2, w = i % n
            D = 32: 2 lane + half      D = 64: 4 lane + 2 half + w      D = 128: 128 half + 4 lane + w
    values: 128 (i / 8) + (4 (i % 8) + p / 4) * 4 + p % 4

Rows of a call: rows starts[b] .. starts[b + 1] - 1 belong to sequence b and hold its positions positions[b], positions[b] + 1, ...
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------------------------------------------
# kind: "store" (write rows, read them back), "read", "attend", or "step" (write the rows' keys and values, then attend: what a
# decoder does per layer). Sequence b starts at a position spread evenly over [first, last] and has a number of rows spread
# evenly over [few, many].
def _case(name, kind, dtype, batch, heads, kv_heads, dim, max_len, first, last, few, many, window=0, sinks=0):
    c = dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, max_len=max_len, first=first, last=last,
             few=few, many=many, window=window, sinks=sinks)
    return {"name": name, **c} if name else c


def listed():
    return [
        # one layer of a 256-sequence decode step writes its tokens' keys and values (fp32, as the projections give them)
        _case("store_batch_256", "store", "fp32", 256, 16, 16, 64, 1024, 128, 640, 1, 1),
        # one layer of a 7B-shaped model writes a prompt of 2048 tokens
        _case("store_prompt_2048", "store", "bf16", 1, 32, 32, 128, 2048, 0, 0, 2048, 2048),
        # a long history is read back, for another kind of attention or to move it to another holder
        _case("read_history_8192", "read", "fp32", 1, 16, 16, 64, 8192, 0, 0, 8192, 8192),
        # the unequal histories of a few small sequences
        _case("read_ragged_fp16", "read", "fp16", 7, 4, 4, 32, 1500, 3, 40, 1, 1301),
        # the first tokens of one chat: nothing but latency
        _case("attend_one_short", "attend", "fp32", 1, 16, 16, 64, 512, 17, 17, 1, 1),
        # the attention of one layer of a 256-sequence decode step
        _case("attend_batch_256", "attend", "fp32", 256, 16, 16, 64, 1024, 128, 640, 1, 1),
        # a few long documents, query heads sharing key/value heads
        _case("attend_long_shared", "attend", "bf16", 4, 32, 8, 128, 32768, 29001, 32766, 1, 1),
        # long chats held to a window with the first tokens kept visible
        _case("attend_window_sinks", "attend", "bf16", 32, 32, 8, 128, 16384, 4099, 16001, 1, 1, 1024, 4),
        # a prompt in one call, fp32 as the projections give it
        _case("attend_prompt_2048", "attend", "fp32", 1, 16, 16, 64, 2048, 0, 0, 2048, 2048),
        # the last chunk of an 8192-token prompt of a 7B-shaped model under a window
        _case("attend_chunk_window", "attend", "bf16", 1, 32, 32, 128, 8192, 6144, 6144, 2048, 2048, 4096, 4),
        # one layer of a decode step: write the token, then attend
        _case("step_batch_64", "step", "fp32", 64, 16, 16, 64, 2048, 300, 1900, 1, 1),
        # drafted tokens being verified beside prompts that are still coming in
        _case("step_mixed_fp16", "step", "fp16", 12, 24, 6, 64, 2048, 5, 1333, 1, 437, 700, 3),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["store", "read", "attend", "attend", "step"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    dim = rng.choice([32, 64, 128])
    kv_heads = _spread(rng, 1, 16)
    group = rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * kv_heads <= 32])
    prompt = rng.random() < 0.4 or kind == "read"
    batch = _spread(rng, 1, 6) if prompt else _spread(rng, 1, 192)
    if prompt:
        many = _spread(rng, 2, 1500)
        few = max(1, many - _spread(rng, 1, many))
        last = _spread(rng, 1, max(1, min(3000, 300_000_000 // (batch * many * kv_heads * group))))
    else:
        few = many = 1
        last = _spread(rng, 2, max(64, min(30000, 4_000_000 // (batch * kv_heads))))
    first = rng.randint(0, last)
    window, sinks = (_spread(rng, 1, last + 1), rng.randint(0, 8)) if rng.random() < 0.4 and kind in ("attend", "step") else (0, 0)
    return _case(None, kind, dtype, batch, kv_heads * group, kv_heads, dim, last + many + rng.randint(0, 100), first, last, few, many,
                 window, sinks)


def _rows(case):
    """The first position and the number of rows of each sequence."""
    n = case["batch"]
    at = [case["first"] + (case["last"] - case["first"]) * i // max(1, n - 1) for i in range(n)]
    # the longest in the middle, so that the order of lengths is not that of positions
    rows = [case["few"] + (case["many"] - case["few"]) * (n - 1 - abs(2 * i - (n - 1))) // max(1, n - 1) if n > 1 else case["many"]
            for i in range(n)]
    return at, rows


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _keys_values(gen, shape, dtype):
    """Keys with channels of their own level and size, values around zero; tokens of different size."""
    dim = shape[-1]
    level = torch.randn(shape[-2:], generator=gen, device="cuda")
    size = torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device="cuda"))
    token = torch.exp(0.3 * torch.randn(shape[:-2] + (1, 1), generator=gen, device="cuda"))
    k = torch.randn(shape, generator=gen, device="cuda").mul_(size).add_(level).mul_(1.0 / math.sqrt(math.sqrt(dim)))
    v = torch.randn(shape, generator=gen, device="cuda").mul_(token).mul_(0.7)
    return k.to(dtype), v.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    B, H, Hkv, D, dtype = case["batch"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    at, rows = _rows(case)
    total = sum(rows)
    tiles = 2 * ((case["max_len"] + 31) // 32)
    data = torch.zeros(B, Hkv, tiles, 16 * (D + 8), dtype=torch.uint8, device="cuda")
    state = {"case": dict(case), "data": data}
    # the history that the cache holds, a part of the batch at a time
    if case["kind"] != "store":
        length = max(a + n for a, n in zip(at, rows))
        step = max(1, 64_000_000 // (length * Hkv * D))
        for b0 in range(0, B, step):
            n = min(step, B - b0)
            k, v = _keys_values(gen, (n * length, Hkv, D), torch.float32)
            seq = torch.arange(b0, b0 + n, device="cuda").repeat_interleave(length)
            _store(data, k, v, seq, torch.arange(length, device="cuda").repeat(n))
    # starts is None where every sequence has one row
    if case["many"] > 1:
        state["starts"] = torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    else:
        state["starts"] = None
    state["positions"] = torch.tensor(at, dtype=torch.int64, device="cuda")
    state["rows"], state["longest"], state["length"] = total, max(rows), max(a + n for a, n in zip(at, rows))
    if case["kind"] in ("store", "step"):
        k, v = _keys_values(gen, (total, Hkv, D), dtype)
        # keys and values side by side in one row, as a fused projection leaves them
        both = torch.cat([k.reshape(total, -1), v.reshape(total, -1)], dim=1)
        state["k"] = both[:, : Hkv * D].view(total, Hkv, D)
        state["v"] = both[:, Hkv * D:].view(total, Hkv, D)
    if case["kind"] in ("attend", "step"):
        state["q"] = torch.randn(total, H, D, generator=gen, device="cuda").mul_(1.5 * math.sqrt(math.sqrt(D))).to(dtype)
        state["scale"] = 1.0 / math.sqrt(D)
    return state


# ---- the plain form -----------------------------------------------------------------------------------------------------
def _word_offsets(dim, position):
    """Word numbers in a tile of the key and value words [..., dim / 8] of positions 0..15 of the tile."""
    n, i, p = dim // 32, torch.arange(dim // 8, device=position.device), position.unsqueeze(-1)
    lane, half, w = (2 * (p // 4) + p % 2) * 4 + i // n, p // 2 % 2, i % n
    keys = 2 * lane + half if dim == 32 else 4 * lane + 2 * half + w if dim == 64 else 128 * half + 4 * lane + w
    values = 128 * (i // 8) + (4 * (i % 8) + p // 4) * 4 + p % 4
    return keys, 2 * dim + values


def _quantise(x):
    """Scale and offset (fp16) and codes of the rows of x, the quotients in 64 bits: their roundings lie next to borders."""
    x = x.double()
    offset = x.amin(-1, keepdim=True).clamp(-65504.0, 65504.0).half()
    scale = ((x.amax(-1, keepdim=True) - offset.double()) / 15.0).clamp(0.0, 65504.0).half()
    s = scale.double()
    code = torch.where(s > 0, torch.round((x - offset.double()) / torch.where(s > 0, s, 1.0)), 0.0).clamp_(0.0, 15.0)
    return scale, offset, code.int()


def _shifts(device):
    """Where in its word the code of channel 2 j + e stands [4, 2]."""
    bits = torch.arange(0, 16, 4, dtype=torch.int32, device=device)
    return torch.stack([bits, bits + 16], -1)


def _pack(code):
    """Words [..., dim / 8] of codes [..., dim]."""
    c = code.unflatten(-1, (-1, 4, 2))
    shift = _shifts(code.device)
    return (c << shift).sum((-1, -2)).to(torch.int32)


def _unpack(word):
    """Codes [..., dim] of words [..., dim / 8]."""
    shift = _shifts(word.device)
    return ((word[..., None, None] >> shift) & 15).flatten(-3)


def _places(data, sequence, position):
    """Flat word numbers of each row's tiles [rows, heads, 1], and the positions in them."""
    heads, tiles, words = data.shape[1], data.shape[2], data.shape[3] // 4
    tile = (sequence[:, None] * heads + torch.arange(heads, device=data.device)) * tiles + (position // 16)[:, None]
    return (tile * words).unsqueeze(-1), (position % 16)[:, None]


def _store(data, k, v, sequence, position):
    dim, flat = k.shape[-1], data.view(torch.int32).view(-1)
    base, p = _places(data, sequence, position)
    at = _word_offsets(dim, p)
    parameters = []
    for x, offset in ((k, at[0]), (v, at[1])):
        scale, zero, code = _quantise(x)
        flat[base + offset] = _pack(code)
        parameters += [scale, zero]
    flat[base + 4 * dim + 2 * p.unsqueeze(-1) + torch.arange(2, device=data.device)] = torch.cat(parameters, -1).view(torch.int32)


def _load(data, dim, sequence, position):
    flat = data.view(torch.int32).view(-1)
    base, p = _places(data, sequence, position)
    at = _word_offsets(dim, p)
    par = flat[base + 4 * dim + 2 * p.unsqueeze(-1) + torch.arange(2, device=data.device)].view(torch.float16).float()
    k, v = (par[..., j + 1:j + 2] + par[..., j:j + 1] * _unpack(flat[base + at[j // 2]]).float() for j in (0, 2))
    return k, v


def _row_places(s):
    """Sequence, position and number within the sequence of each row."""
    n = torch.arange(s["rows"], device="cuda")
    if s["starts"] is None:
        return n, s["positions"], torch.zeros_like(n)
    sequence = (n[:, None] >= s["starts"][None, 1:]).sum(1)
    within = n - s["starts"][sequence]
    return sequence, s["positions"][sequence] + within, within


def _attend(s):
    c, q = s["case"], s["q"].float()
    B, H, Hkv, D = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    sequence, position, within = _row_places(s)
    L = s["length"]
    every = torch.arange(B, device="cuda").repeat_interleave(L), torch.arange(L, device="cuda").repeat(B)
    k, v = (x.view(B, L, Hkv, 1, D).permute(0, 2, 3, 1, 4) for x in _load(s["data"], D, *every))  # [B, Hkv, 1, L, D]
    padded = torch.zeros(B, s["longest"], H, D, device="cuda")
    padded[sequence, within] = q
    at = torch.full((B, s["longest"]), -1, dtype=torch.int64, device="cuda")
    at[sequence, within] = position
    j = torch.arange(L, device="cuda")
    seen = j <= at[..., None]
    if c["window"]:
        seen &= (j > at[..., None] - c["window"]) | (j < c["sinks"])
    seen = seen[:, None, None]                                                      # [B, 1, 1, T, L]
    x = padded.view(B, s["longest"], Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4) @ k.transpose(-1, -2)
    x = x.mul_(s["scale"]).masked_fill_(~seen, -math.inf)                           # [B, Hkv, G, T, L]
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, s["longest"], H, D)
    return out[sequence, within].to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        from ivonar_inference_b200 import KV4Cache

        cache = KV4Cache(c["batch"], c["kv_heads"], c["dim"], c["max_len"], data=s["data"])
        if c["kind"] in ("store", "step"):
            cache.append(s["k"], s["v"], s["positions"], s["starts"])
        if c["kind"] in ("store", "read"):
            return cache.read(s["positions"], s["starts"], rows=s["rows"], dtype=DTYPES[c["dtype"]])
        return cache.attention(s["q"], s["positions"], s["starts"], scale=s["scale"], window=c["window"], sinks=c["sinks"])
    sequence, position, _ = _row_places(s)
    if c["kind"] in ("store", "step"):
        _store(s["data"], s["k"], s["v"], sequence, position)
    if c["kind"] in ("store", "read"):
        return tuple(x.to(DTYPES[c["dtype"]]) for x in _load(s["data"], c["dim"], sequence, position))
    return _attend(s)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    at, rows = _rows(case)
    H, Hkv, D, size = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]].itemsize
    total, moved, operations = sum(rows), 0, 0
    if case["kind"] in ("store", "step"):
        moved += total * Hkv * (2 * D * size + D + 8)
        operations += total * Hkv * D * 2 * 4
    if case["kind"] in ("store", "read"):
        moved += total * Hkv * 2 * D * size + (total * Hkv * (D + 8) if case["kind"] == "read" else 0)
        operations += total * Hkv * D * 2 * 2
    else:
        moved += 2 * total * H * D * size
        window, sinks = case["window"], case["sinks"]
        for a, n in zip(at, rows):
            if not window:
                union, pairs = a + n, n * (a + 1) + n * (n - 1) // 2
            else:
                low = max(0, a - window + 1)
                union = a + n - low + min(low, sinks)
                pairs = sum(p - max(0, p - window + 1) + 1 + min(max(0, p - window + 1), sinks) for p in range(a, a + n))
            moved += union * Hkv * (D + 8)
            operations += 4 * D * H * pairs
    return {"bytes": moved, "flops": operations}


# ---- in 64 bits ---------------------------------------------------------------------------------------------------------
def _exact_rows(x):
    """What the cache holds of the rows of x, in 64 bits."""
    x = x.to(torch.float64)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    zero = low.to(torch.float16).to(torch.float64)
    unit = torch.relu((high - zero) / 15).to(torch.float16).to(torch.float64)
    return zero + unit * torch.nan_to_num((x - zero) / unit, nan=0.0, posinf=15.0, neginf=0.0).round().clip(0, 15)


def _exact_history(data, b, dim, count):
    """Keys and values [kv_heads, count, dim] of one sequence, looked up nibble by nibble in the tiles' bytes."""
    tile = data[b, :, : (count + 15) // 16]
    nibble = torch.stack([tile[..., : 16 * dim] & 15, tile[..., : 16 * dim] >> 4], -1).flatten(-2)  # 32 dim nibbles a tile
    p, d = torch.meshgrid(torch.arange(16, device="cuda"), torch.arange(dim, device="cuda"), indexing="ij")
    word, place, each = d // 8, (d % 8) // 2 + 4 * (d % 2), dim // 32
    lane, half = (2 * (p // 4) + p % 2) * 4 + word // each, p // 2 % 2
    key = {32: 2 * lane + half, 64: 4 * lane + 2 * half + word % each, 128: 128 * half + 4 * lane + word % each}[dim]
    value = 2 * dim + 128 * (word // 8) + (4 * (word % 8) + p // 4) * 4 + p % 4
    par = tile[..., 16 * dim:].contiguous().view(torch.float16).unflatten(-1, (16, 4)).to(torch.float64)
    found = []
    for at, j in ((key, 0), (value, 2)):
        code = nibble.index_select(-1, (8 * at + place).flatten()).unflatten(-1, (16, dim)).to(torch.float64)
        found.append((par[..., j + 1:j + 2] + par[..., j:j + 1] * code).flatten(1, 2)[:, :count])
    return found


def exact(case, seed):
    s = prepare(case, seed)
    at, rows = _rows(case)
    B, H, Hkv, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    new = [_exact_rows(s[x]) for x in ("k", "v")] if case["kind"] in ("store", "step") else None
    if case["kind"] == "store":
        return tuple(new)
    if case["kind"] == "read":
        k, v = (torch.zeros(s["rows"], Hkv, D, dtype=torch.float64, device="cuda") for _ in range(2))
    else:
        out = torch.zeros(s["rows"], Hkv, H // Hkv, D, dtype=torch.float64, device="cuda")
        queries = s["q"].double().unflatten(1, (Hkv, H // Hkv))
    r0 = 0
    for b in range(B):
        a, n = at[b], rows[b]
        r1, count = r0 + n, at[b] + n
        kb, vb = _exact_history(s["data"], b, D, count)
        if case["kind"] == "read":
            k[r0:r1], v[r0:r1] = kb[:, a:].transpose(0, 1), vb[:, a:].transpose(0, 1)
        else:
            if new is not None:
                kb[:, a:], vb[:, a:] = new[0][r0:r1].transpose(0, 1), new[1][r0:r1].transpose(0, 1)
            where = torch.arange(count, device="cuda")
            hidden = where > where[a:, None]
            if case["window"]:
                hidden |= (where <= where[a:, None] - case["window"]) & (where >= case["sinks"])
            step = max(1, 300_000_000 // (n * count * (H // Hkv)))
            for h in range(0, Hkv, step):  # so many heads at a time
                score = torch.einsum("nhgd,hjd->hgnj", queries[r0:r1, h:h + step], kb[h:h + step]) * s["scale"]
                weight = torch.softmax(score.masked_fill_(hidden, -math.inf), -1)
                out[r0:r1, h:h + step] = torch.einsum("hgnj,hjd->nhgd", weight, vb[h:h + step])
        r0 = r1
    return (k, v) if case["kind"] == "read" else out.flatten(1, 2)
