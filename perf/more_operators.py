"""What is measured of answering one prompt many times: sequences of the 4-bit key/value cache forked and compacted, attention
of a batch whose sequences begin with the same tokens, held and read once for all, and log probabilities of given tokens
with the entropy and the likeliest alternatives.

A cache is one uint8 tensor [batch, kv_heads, tiles, 16 * (D + 8)]: a tile holds 16 positions of one key/value head as 8 D bytes
of key codes, 8 D bytes of value codes and 16 x 4 fp16 (key scale, key offset, value scale, value offset); a row x of D values
is kept as x = offset + scale * code with

    offset = fp16(min x),  scale = fp16((max x - offset) / 15),  code = round((x - offset) / scale), clipped to 0..15

Codes are packed in 32-bit words of 8 channels, channel 2 j in nibble j and channel 2 j + 1 in nibble j + 4 (j = 0..3). Word i
of position p (0..15) of a tile, in words from the start of the tile, with n = D / 32:

    keys:   lane = (2 (p / 4) + p % 2) * 4 + i / n, half = p / 2 % 2, w = i % n
            D = 32: 2 lane + half      D = 64: 4 lane + 2 half + w      D = 128: 128 half + 4 lane + w
    values: 2 D + 128 (i / 8) + (4 (i % 8) + p / 4) * 4 + p % 4
    scales and offsets: 4 D + 2 p and 4 D + 2 p + 1

fork      sequence b takes the first lengths[b] positions of sequence sources[b], of the same cache as it was or of another
compact   position positions[b] + i of sequence b takes the row at index[starts[b] + i] of the same sequence, which lies there
          or behind
attend    causal attention, rows starts[b] .. starts[b + 1] - 1 at the positions positions[b], positions[b] + 1, ... of sequence
          b, before which come the first prefix_lengths[g] positions of sequence g of another cache, where
          prefix_groups[g] <= b < prefix_groups[g + 1]; windows and first tokens ("sinks") count from the beginning
logprobs  log p of given tokens, the entropy -sum p log p and the `top` likeliest tokens, with p = softmax(logits / temperature);
          among equal logits the lowest token comes first
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------------------------------------------
def _fork(name, batch, kv_heads, dim, max_len, short, long, every, outside):
    """`batch` sequences take beginnings of between `short` and `long` positions, every `every`-th one staying as it is (and
    giving its own to those behind it), or all of them from another cache of every `every`-th's."""
    c = dict(kind="fork", batch=batch, kv_heads=kv_heads, dim=dim, max_len=max_len, short=short, long=long, every=every, outside=outside)
    return {"name": name, **c} if name else c


def _compact(name, batch, kv_heads, dim, max_len, first, last, few, many, spread):
    """Each of `batch` sequences keeps between `few` and `many` rows from its position first..last on, out of those that begin
    as many places behind, one of `spread` on the average."""
    c = dict(kind="compact", batch=batch, kv_heads=kv_heads, dim=dim, max_len=max_len, first=first, last=last, few=few, many=many, spread=spread)
    return {"name": name, **c} if name else c


def _attend(name, dtype, groups, batch, heads, kv_heads, dim, short, long, first, last, few, many, window=0, sinks=0):
    """`batch` sequences in `groups` groups that begin with short..long positions of their own, then first..last tokens of each
    sequence's own, then few..many rows that attend."""
    c = dict(kind="attend", dtype=dtype, groups=groups, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, short=short, long=long,
             first=first, last=last, few=few, many=many, window=window, sinks=sinks)
    return {"name": name, **c} if name else c


def _logprobs(name, dtype, rows, vocab, given, top, temperature, banned):
    """`given` tokens a row; of the vocabulary one of `banned` is ruled out (0: none)."""
    c = dict(kind="logprobs", dtype=dtype, rows=rows, vocab=vocab, given=given, top=top, temperature=temperature, banned=banned)
    return {"name": name, **c} if name else c


def listed():
    return [
        # the beams of a short answer take the places of those that fell out, in one layer: nothing but latency
        _fork("fork_beams_8", 8, 16, 64, 512, 150, 150, 4, False),
        # the beams of 16 requests
        _fork("fork_beams_128", 128, 16, 64, 1024, 300, 700, 4, False),
        # 64 answers to one prompt of 2048 tokens, which another cache holds, one layer of a model with shared heads
        _fork("fork_prompt_64", 64, 8, 128, 4096, 2048, 2048, 64, True),
        # what is accepted of 64 sequences' trees of drafted tokens moves up behind what they have
        _compact("compact_drafts_64", 64, 16, 64, 2048, 300, 1900, 1, 6, 3),
        # four long chats drop what is least looked at of the older half
        _compact("compact_history", 4, 8, 128, 32768, 4, 4, 13001, 14400, 1.1),
        # the first tokens of four answers to one question
        _attend("attend_answers_4", "fp32", 1, 4, 16, 16, 64, 300, 300, 5, 40, 1, 1),
        # 64 answers to one long document
        _attend("attend_document_64", "fp32", 1, 64, 16, 16, 64, 8192, 8192, 10, 500, 1, 1),
        # three tools' instructions and their 96 chats, query heads sharing key/value heads
        _attend("attend_groups_96", "bf16", 3, 96, 32, 8, 128, 16001, 29990, 17, 900, 1, 1),
        # eight questions of some 200 tokens each about one text
        _attend("attend_questions_8", "bf16", 1, 8, 32, 8, 128, 4100, 4100, 0, 0, 150, 260),
        # the answer token of one request, with five alternatives
        _logprobs("logprobs_one", "fp32", 1, 32768, 1, 5, 1.0, 0),
        # a decode step of 256 sequences, as the head gives it, some tokens ruled out
        _logprobs("logprobs_batch_256", "fp32", 256, 32768, 1, 20, 0.8, 50),
        # the tokens of a text under a large vocabulary of an odd size
        _logprobs("logprobs_text_1500", "bf16", 1500, 100003, 1, 2, 1.0, 0),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["fork", "compact", "attend", "attend", "logprobs"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    dim = rng.choice([32, 64, 128])
    kv_heads = _spread(rng, 1, 16)
    if kind == "logprobs":
        rows = _spread(rng, 1, 2000)
        vocab = _spread(rng, 300, min(200_000, 150_000_000 // rows))
        return _logprobs(None, dtype, rows, vocab, rng.choice([1, 1, 1, 4]), rng.choice([0, 1, 5, 20, 64]), rng.choice([1.0, 0.7, 1.3]),
                         rng.choice([0, 0, 7, 100]))
    if kind == "fork":
        batch = _spread(rng, 2, 192)
        long = _spread(rng, 2, min(20_000, 110_000_000 // (batch * kv_heads * (dim + 8))))
        return _fork(None, batch, kv_heads, dim, long + rng.randint(0, 500), rng.randint(1, long), long, rng.randint(2, max(2, min(batch, 16))),
                     rng.random() < 0.4)
    if kind == "compact":
        batch = _spread(rng, 1, 96)
        many = _spread(rng, 1, min(8000, 40_000_000 // (batch * kv_heads * (dim + 8))))
        last = _spread(rng, 1, 1000)
        spread = rng.choice([1, 1.5, 3])
        return _compact(None, batch, kv_heads, dim, last + many + int(many * spread) + 1 + rng.randint(0, 100), rng.randint(0, last), last,
                        rng.randint(1, many), many, spread)
    group = rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * kv_heads <= 32])
    prompt = rng.random() < 0.35
    batch = _spread(rng, 1, 8) if prompt else _spread(rng, 2, 160)
    groups = rng.choice([1, 1, 1, min(batch, rng.randint(1, 5))])
    if prompt:
        many = _spread(rng, 2, 500)
        few = rng.randint(1, many)
        long = _spread(rng, 1, max(2, min(5000, 250_000_000 // (batch * many * kv_heads * group))))
        last = rng.randint(0, 300)
    else:
        few = many = 1 if rng.random() < 0.7 else rng.randint(2, 6)
        long = _spread(rng, 1, max(64, min(30_000, 30_000_000 // (batch * many * kv_heads * group))))
        last = rng.randint(0, 400)
    window, sinks = (_spread(rng, 1, long + last + 1), rng.randint(0, 8)) if rng.random() < 0.3 else (0, 0)
    return _attend(None, dtype, groups, batch, kv_heads * group, kv_heads, dim, rng.randint(1, long), long, rng.randint(0, last), last, few, many,
                   window, sinks)


def _evenly(low, high, n):
    return [low + (high - low) * i // max(1, n - 1) for i in range(n)]


def _humped(few, many, n):
    """The largest in the middle, so that the order of sizes is not that of the sequences."""
    return [few + (many - few) * (n - 1 - abs(2 * i - (n - 1))) // max(1, n - 1) if n > 1 else many for i in range(n)]


def _bounds(counts):
    return [sum(counts[:b]) for b in range(len(counts) + 1)]


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _values_of(gen, n, heads, dim):
    """Keys with channels of their own level and size, values around zero; tokens of different size."""
    shape = (n, heads, dim)
    level = torch.randn(shape[1:], generator=gen, device="cuda")
    size = torch.exp(0.5 * torch.randn(shape[1:], generator=gen, device="cuda"))
    token = torch.exp(0.3 * torch.randn((n, 1, 1), generator=gen, device="cuda"))
    k = torch.randn(shape, generator=gen, device="cuda").mul_(size).add_(level).mul_(1.0 / math.sqrt(math.sqrt(dim)))
    v = torch.randn(shape, generator=gen, device="cuda").mul_(token).mul_(0.7)
    return k, v


def _cache(gen, batch, heads, dim, max_len, length):
    """The storage of a cache whose sequences hold `length` positions each."""
    data = torch.zeros(batch, heads, 2 * ((max_len + 31) // 32), 16 * (dim + 8), dtype=torch.uint8, device="cuda")
    step = max(1, 64_000_000 // max(1, length * heads * dim))
    for b0 in range(0, batch if length else 0, step):
        n = min(step, batch - b0)
        k, v = _values_of(gen, n * length, heads, dim)
        seq = torch.arange(b0, b0 + n, device="cuda").repeat_interleave(length)
        _store(data, k, v, seq, torch.arange(length, device="cuda").repeat(n))
    return data


def _device(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s, c = {"case": dict(case)}, case
    if c["kind"] == "logprobs":
        rows, vocab = c["rows"], c["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device="cuda").mul_(2.0)
        # a few tokens stand out, by other amounts in each row
        favoured = torch.randint(0, vocab, (rows, 8), generator=gen, device="cuda")
        x.scatter_add_(1, favoured, 8.0 * torch.rand(rows, 8, generator=gen, device="cuda"))
        if c["banned"]:
            out = torch.rand(vocab, generator=gen, device="cuda") < 1.0 / c["banned"]
            out[0] = False
            x.masked_fill_(out, -math.inf)
        tokens = torch.randint(0, vocab, (rows, c["given"]), generator=gen, device="cuda")
        tokens[::2, 0] = favoured[::2, 0]
        s["logits"], s["tokens"] = x.to(DTYPES[c["dtype"]]), tokens
        return s
    B, H, D = c["batch"], c["kv_heads"], c["dim"]
    if c["kind"] == "fork":
        lengths = _humped(c["short"], c["long"], B)
        s["data"] = _cache(gen, B, H, D, c["max_len"], c["long"])
        if c["outside"]:
            s["source"] = _cache(gen, (B + c["every"] - 1) // c["every"], H, D, c["long"], c["long"])
            sources = [b // c["every"] for b in range(B)]
        else:
            sources = [b // c["every"] * c["every"] for b in range(B)]
        s["sources"], s["lengths"], s["tiles"] = _device(sources), _device(lengths), (c["long"] + 15) // 16
    elif c["kind"] == "compact":
        at, kept = _evenly(c["first"], c["last"], B), _humped(c["few"], c["many"], B)
        s["data"] = _cache(gen, B, H, D, c["max_len"], min(c["max_len"], c["last"] + c["many"] + int(c["many"] * c["spread"]) + 1))
        index = []
        for a, n in zip(at, kept):
            order = torch.rand(max(n, int(n * c["spread"])), generator=gen, device="cuda").argsort()[:n].sort().values
            index.append(a + n + order)
        s["index"], s["positions"], s["starts"] = torch.cat(index), _device(at), _device(_bounds(kept), torch.int32)
    else:
        dtype, G = DTYPES[c["dtype"]], c["groups"]
        at, rows, long = _evenly(c["first"], c["last"], B), _humped(c["few"], c["many"], B), _evenly(c["short"], c["long"], G)
        total, length = sum(rows), max(a + n for a, n in zip(at, rows))
        s["data"] = _cache(gen, B, H, D, length, length)
        s["prefix"] = _cache(gen, G, H, D, c["long"], c["long"])
        s["positions"], s["prefix_lengths"] = _device(at), _device(long)
        s["prefix_groups"] = None if G == 1 else _device([g * B // G for g in range(G + 1)], torch.int32)
        s["starts"] = None if c["many"] == 1 else _device(_bounds(rows), torch.int32)
        s["plan"] = [(g * B // G, (g + 1) * B // G, long[g]) for g in range(G)], _bounds(rows), length, max(rows)
        s["q"] = torch.randn(total, c["heads"], D, generator=gen, device="cuda").mul_(1.5 * math.sqrt(math.sqrt(D))).to(dtype)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def _word_offsets(dim, position):
    """Word numbers in a tile of the key and value words [..., dim / 8] of positions 0..15 of the tile."""
    n, i, p = dim // 32, torch.arange(dim // 8, device=position.device), position.unsqueeze(-1)
    lane, half, w = (2 * (p // 4) + p % 2) * 4 + i // n, p // 2 % 2, i % n
    keys = 2 * lane + half if dim == 32 else 4 * lane + 2 * half + w if dim == 64 else 128 * half + 4 * lane + w
    return keys, 2 * dim + 128 * (i // 8) + (4 * (i % 8) + p // 4) * 4 + p % 4


def _row_words(dim, position):
    """All of a position's words in its tile [..., dim / 4 + 2]."""
    par = 4 * dim + 2 * position.unsqueeze(-1) + torch.arange(2, device=position.device)
    return torch.cat([*_word_offsets(dim, position), par], -1)


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
        flat[base + offset] = (code.unflatten(-1, (-1, 4, 2)) << _shifts(data.device)).sum((-1, -2)).to(torch.int32)
        parameters += [scale, zero]
    flat[base + 4 * dim + 2 * p.unsqueeze(-1) + torch.arange(2, device=data.device)] = torch.cat(parameters, -1).view(torch.int32)


def _load(data, dim, sequence, position):
    flat = data.view(torch.int32).view(-1)
    base, p = _places(data, sequence, position)
    at = _word_offsets(dim, p)
    par = flat[base + 4 * dim + 2 * p.unsqueeze(-1) + torch.arange(2, device=data.device)].view(torch.float16).float()
    code = [((flat[base + a][..., None, None] >> _shifts(data.device)) & 15).flatten(-3).float() for a in at]
    k, v = (par[..., 2 * j + 1:2 * j + 2] + par[..., 2 * j:2 * j + 1] * code[j] for j in (0, 1))
    return k, v


def _plain_fork(s):
    c, tiles = s["case"], s["tiles"]
    D, data = c["dim"], s["data"].view(torch.int32)
    source = s.get("source", s["data"]).view(torch.int32)
    place = torch.empty(16 * (D + 8) // 4, dtype=torch.int64, device="cuda")  # position in the tile of each of its words
    p = torch.arange(16, device="cuda")
    place[_row_words(D, p)] = p[:, None].expand(-1, D // 4 + 2)
    at = 16 * torch.arange(tiles, device="cuda")[:, None] + place
    taken = at < s["lengths"][:, None, None, None]
    data[:, :, :tiles] = torch.where(taken, source[s["sources"], :, :tiles], data[:, :, :tiles])
    return s["data"]


def _rows_of(starts, positions, total):
    """Sequence and position of each row, and its number within the sequence."""
    n = torch.arange(total, device="cuda")
    if starts is None:
        return n, positions, torch.zeros_like(n)
    sequence = (n[:, None] >= starts[None, 1:]).sum(1)
    within = n - starts[sequence]
    return sequence, positions[sequence] + within, within


def _plain_compact(s):
    D, flat = s["case"]["dim"], s["data"].view(torch.int32).view(-1)
    sequence, position, _ = _rows_of(s["starts"], s["positions"], s["index"].numel())
    (base, p), (source, f) = _places(s["data"], sequence, position), _places(s["data"], sequence, s["index"])
    flat[base + _row_words(D, p)] = flat[source + _row_words(D, f)]
    return s["data"]


def _plain_attend(s):
    c, q = s["case"], s["q"].float()
    H, Hkv, D, window, sinks = c["heads"], c["kv_heads"], c["dim"], c["window"], c["sinks"]
    groups, bounds, length, longest = s["plan"]
    sequence, position, within = _rows_of(s["starts"], s["positions"], q.shape[0])
    out = torch.empty_like(q)
    for g, (b0, b1, L) in enumerate(groups):
        n, rows = b1 - b0, slice(bounds[b0], bounds[b1])
        if n == 0:
            continue
        cell = (sequence[rows] - b0, within[rows])
        padded = torch.zeros(n, longest, H, D, device="cuda")
        padded[cell] = q[rows]
        at = torch.full((n, longest), -1, dtype=torch.int64, device="cuda")  # from the beginning of the group
        at[cell] = position[rows] + L
        x = padded.view(n, longest, Hkv, H // Hkv, D).permute(2, 0, 3, 1, 4)  # [Hkv, n, G, T, D]
        k0, v0 = (y.transpose(0, 1) for y in _load(s["prefix"], D, torch.full((L,), g, device="cuda"), torch.arange(L, device="cuda")))
        every = torch.arange(b0, b1, device="cuda").repeat_interleave(length), torch.arange(length, device="cuda").repeat(n)
        k1, v1 = (y.view(n, length, Hkv, 1, D).permute(2, 0, 3, 1, 4) for y in _load(s["data"], D, *every))
        score = (x.reshape(Hkv, -1, D) @ k0.transpose(1, 2)).view(*x.shape[:-1], L), x @ k1.transpose(-1, -2)
        score = torch.cat(score, -1).mul_(D**-0.5)
        j = torch.cat([torch.arange(L, device="cuda"), L + torch.arange(length, device="cuda")])
        seen = j <= at[..., None]
        if window:
            seen &= (j > at[..., None] - window) | (j < sinks)
        score.masked_fill_(~seen[:, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = p.sum(-1, keepdim=True)
        y = (p[..., :L].reshape(Hkv, -1, L) @ v0).view(x.shape) + p[..., L:] @ v1
        y = y / torch.where(total > 0, total, 1.0)
        out[rows] = y.permute(1, 3, 0, 2, 4).reshape(n, longest, H, D)[cell]
    return out.to(s["q"].dtype)


def _plain_logprobs(s):
    c, x = s["case"], s["logits"].float()
    if c["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : c["top"]]
    else:
        ids = torch.empty(c["rows"], 0, dtype=torch.int64, device="cuda")
    x = x / c["temperature"]
    below = x - x.amax(1, keepdim=True)
    e = torch.exp(below)
    total = e.sum(1, keepdim=True)
    log_p = below - torch.log(total)
    entropy = -torch.where(e > 0, (e / total) * log_p, 0.0).sum(1)
    return log_p.gather(1, s["tokens"]), entropy, log_p.gather(1, ids), ids


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"fork": _plain_fork, "compact": _plain_compact, "attend": _plain_attend, "logprobs": _plain_logprobs}[c["kind"]](s)
    from ivonar_inference_b200 import KV4Cache, log_probs

    if c["kind"] == "logprobs":
        found = log_probs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"])
        return found.tokens, found.entropy, found.top, found.ids
    if "cache" not in s:  # a user's program keeps these
        def cache(data, max_len):
            return KV4Cache(data.shape[0], c["kv_heads"], c["dim"], max_len, data=data)

        s["cache"] = cache(s["data"], c["max_len"] if c["kind"] != "attend" else s["plan"][2])
        s["other"] = cache(s["source"], c["long"]) if "source" in s else cache(s["prefix"], c["long"]) if "prefix" in s else None
    if c["kind"] == "fork":
        s["cache"].fork(s["sources"], s["lengths"], source=s["other"])
        return s["data"]
    if c["kind"] == "compact":
        s["cache"].compact(s["index"], s["positions"], s["starts"])
        return s["data"]
    return s["cache"].attention(s["q"], s["positions"], s["starts"], window=c["window"], sinks=c["sinks"], prefix=s["other"],
                                prefix_lengths=s["prefix_lengths"], prefix_groups=s["prefix_groups"])


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "logprobs":
        moved = c["rows"] * (c["vocab"] * DTYPES[c["dtype"]].itemsize + c["given"] * 12 + 4 + c["top"] * 12)
        return {"bytes": moved, "flops": 7 * c["rows"] * c["vocab"]}  # less, scaled, exp, two sums and a maximum
    row = c["kv_heads"] * (c["dim"] + 8)
    if c["kind"] == "fork":
        lengths, longest, written = _humped(c["short"], c["long"], c["batch"]), {}, 0
        for b, n in enumerate(lengths):
            if c["outside"] or b % c["every"]:
                longest[b // c["every"]] = max(n, longest.get(b // c["every"], 0))
                written += n
        return {"bytes": row * (written + sum(longest.values())) + 16 * c["batch"], "flops": 0}
    if c["kind"] == "compact":
        kept = sum(_humped(c["few"], c["many"], c["batch"]))
        return {"bytes": kept * (2 * row + 8), "flops": 0}
    B, G, window, sinks = c["batch"], c["groups"], c["window"], c["sinks"]
    at, rows, long = _evenly(c["first"], c["last"], B), _humped(c["few"], c["many"], B), _evenly(c["short"], c["long"], G)
    moved, pairs = 2 * sum(rows) * c["heads"] * c["dim"] * DTYPES[c["dtype"]].itemsize, 0
    for g in range(G):
        shared = 0  # positions of the beginning that some row of the group sees
        for b in range(g * B // G, (g + 1) * B // G):
            start = long[g] + at[b]
            low = max(0, start - window + 1) if window else 0
            shared = max(shared, long[g] - min(low, long[g]) + min(min(low, long[g]), sinks))
            mine = max(low, long[g])
            moved += (start + rows[b] - mine + max(0, min(sinks, mine) - long[g])) * row
            for p in range(start, start + rows[b]):
                left = max(0, p - window + 1) if window else 0
                pairs += p + 1 - left + min(left, sinks)
        moved += shared * row
    return {"bytes": moved, "flops": 4 * c["dim"] * c["heads"] * pairs}


# ---- in 64 bits ---------------------------------------------------------------------------------------------------------
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
    c = case
    if c["kind"] in ("fork", "compact"):
        return None  # bytes that are moved, not computed
    s = prepare(case, seed)
    if c["kind"] == "logprobs":
        parts = [[], [], [], []]
        for r0 in range(0, c["rows"], 64):
            x = s["logits"][r0:r0 + 64].to(torch.float64)
            # by value, then by token: of equal ones the order of a stable sort of the negated values
            ids = torch.argsort(-x, dim=1, stable=True)[:, : c["top"]]
            log_p = torch.log_softmax(x / c["temperature"], 1)
            parts[0].append(torch.take_along_dim(log_p, s["tokens"][r0:r0 + 64], 1))
            parts[1].append(-torch.special.xlogy(log_p.exp(), log_p.exp()).sum(1))
            parts[2].append(torch.take_along_dim(log_p, ids, 1))
            parts[3].append(ids)
        return tuple(torch.cat(p) for p in parts)
    (groups, bounds, _, _), H, Hkv, D = s["plan"], c["heads"], c["kv_heads"], c["dim"]
    at = _evenly(c["first"], c["last"], c["batch"])
    out = torch.zeros(bounds[-1], Hkv, H // Hkv, D, dtype=torch.float64, device="cuda")
    q = s["q"].to(torch.float64).unflatten(1, (Hkv, H // Hkv))
    for g, (b0, b1, L) in enumerate(groups):
        shared = _exact_history(s["prefix"], g, D, L)
        for b in range(b0, b1):
            n = bounds[b + 1] - bounds[b]
            k, v = (torch.cat([a, o], 1) for a, o in zip(shared, _exact_history(s["data"], b, D, at[b] + n)))
            where = torch.arange(L + at[b] + n, device="cuda")
            mine = where[L + at[b]:, None]
            hidden = where > mine
            if c["window"]:
                hidden |= (where <= mine - c["window"]) & (where >= c["sinks"])
            step = max(1, 300_000_000 // (n * where.numel() * (H // Hkv)))
            for h in range(0, Hkv, step):  # so many heads at a time
                score = torch.einsum("nhgd,hjd->hgnj", q[bounds[b]:bounds[b + 1], h:h + step], k[h:h + step]) / math.sqrt(D)
                weight = torch.softmax(score.masked_fill_(hidden, -math.inf), -1)
                out[bounds[b]:bounds[b + 1], h:h + step] = torch.einsum("hgnj,hjd->nhgd", weight, v[h:h + step])
    return out.flatten(1, 2)
