"""The measured operators of a serving loop over the paged KV cache, each in its plain form and through the op adapter (`ops`).

  append  the q and k heads of new tokens are rotated by their positions' angles, k and v rows go into the cache
  chunk   attention of several new tokens of each sequence, which the cache holds already, over all that it holds
  window  the same where a token sees the last `window` tokens up to itself and the first `sinks` of its sequence;
          with `single`, one new token for each sequence (a decode step)

What each sequence holds is drawn from the case's own `mix`, so that all seeds of a case do the same work; everything else
that a state holds comes from the seed. `index` is the type of slot tables, lengths, positions and destinations.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INDEX = {"int32": torch.int32, "int64": torch.int64}

# query heads, K/V heads, head size
SMALL = (8, 8, 64)
BASE = (32, 32, 128)
GROUPED = (32, 8, 128)
WIDE = (40, 40, 128)
LARGE = (64, 8, 128)

MOST_SCORES = 2 * 32 * 2048 * 8192   # scores of a drawn case's plain form: those of the largest listed one


def _case(kind, size, dtype, index="int32", mix=0, **more):
    heads, kv_heads, d = size
    return dict(kind=kind, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, index=index, mix=mix, **more)


def _append(size, tokens, dtype, index="int32", stacked=False, interleaved=False, by_position=True, mix=0, **more):
    return _case("append", size, dtype, index, mix, tokens=tokens, stacked=stacked, interleaved=interleaved, by_position=by_position, **more)


def _batch(kind, size, batch, new, cached, dtype, index="int32", mix=0, ones=0, window=0, sinks=0, single=False, **more):
    """`ones` of the sequences have one new token, the others from new[0] to new[1]; behind cached[0] to cached[1] of them."""
    return _case(kind, size, dtype, index, mix, batch=batch, min_new=new[0], max_new=new[1], min_cached=cached[0], max_cached=cached[1], ones=ones, window=window,
                 sinks=sinks, single=single, **more)


def listed():
    return [
        # a decode step of 64 sequences: one row each, all launch latency
        _append(BASE, 64, "bf16", interleaved=True, name="append_64_bf16"),
        # a prompt on grouped K/V heads: slices of the stacked projection's rows, a table row for each token
        _append(GROUPED, 1777, "fp16", "int64", stacked=True, by_position=False, name="append_1777_stacked_fp16"),
        # the benchmark layer's full batch of prompts, 4 x 2048 tokens
        _append(BASE, 8192, "bf16", stacked=True, interleaved=True, name="append_8192_bf16"),
        # one user's five speculated tokens, checked at once: the latency of a small batch
        _batch("chunk", GROUPED, 1, (5, 5), (1777, 1777), "bf16", name="chunk_1x5_1777_bf16"),
        # short turns of very different lengths in the fp32 parity configuration's heads
        _batch("chunk", SMALL, 16, (1, 40), (0, 260), "fp32", "int64", mix=1, name="chunk_16_short_fp32"),
        # continuous batching: most sequences decode a token, a few bring a piece of their prompt
        _batch("chunk", GROUPED, 24, (200, 333), (100, 3000), "bf16", mix=2, ones=20, name="chunk_24_mixed_bf16"),
        # pieces of long prompts on grouped K/V heads
        _batch("chunk", GROUPED, 4, (512, 512), (1000, 7000), "fp16", mix=3, name="chunk_4x512_grouped_fp16"),
        # the same with a K/V head for each query head: the most work
        _batch("chunk", BASE, 2, (2048, 2048), (6000, 6000), "bf16", name="chunk_2x2048_bf16"),
        # one user waiting for a token of a windowed model
        _batch("window", GROUPED, 1, (1, 1), (6000, 6000), "bf16", window=1024, sinks=4, single=True, name="window_1x6001_bf16"),
        # the throughput end of decoding with a window, on grouped K/V heads
        _batch("window", GROUPED, 48, (1, 1), (100, 12000), "fp16", mix=4, window=2048, sinks=4, single=True, name="window_48_grouped_fp16"),
        # the same without first tokens and with a K/V head for each query head
        _batch("window", BASE, 64, (1, 1), (512, 6000), "bf16", "int64", mix=5, window=2048, single=True, name="window_64_bf16"),
        # the benchmark layer's batch of prompts in a windowed model
        _batch("window", BASE, 4, (2048, 2048), (0, 0), "bf16", window=512, sinks=4, name="window_4x2048_bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "chunk", "chunk", "chunk", "window", "window", "window"])
    heads, kv_heads, d = rng.choice([SMALL, BASE, GROUPED, WIDE, LARGE])
    size = heads, kv_heads, rng.choice([d, d, d, 64, 80, 96, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    index = rng.choice(["int32", "int32", "int64"])
    mix = rng.randrange(1 << 20)
    if kind == "append":
        most = min(16384, 8192 * 4096 // (size[0] * size[2]))
        return _append(size, _spread(rng, 1, most), dtype, index, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.7, mix)
    single = kind == "window" and rng.random() < 0.6
    batch = _spread(rng, 1, 64)
    work = MOST_SCORES * 96 // (size[2] * 4 if dtype == "fp32" else size[2])       # (query, key) pairs times heads, and tokens of a sequence:
    rows = 64 * 1600 * 4096 // (size[1] * size[2] * batch * (2 if dtype == "fp32" else 1))
    most = 1 if single else _spread(rng, 1, max(2, min(2048, rows // 2, int(math.sqrt(work / (heads * batch))))))
    new = rng.choice([most, rng.randint(1, most), 1]), most
    high = _spread(rng, 1, max(2, min(12000, rows - most, work // (heads * batch * most) - most)))
    cached = rng.choice([high, rng.randint(0, high), high // rng.randint(2, 16)]), high
    ones = rng.choice([0, 0, batch // 2, batch - 1])
    window, sinks = (_spread(rng, 1, 4096), rng.choice([0, 1, 4, 4, 16, 100])) if kind == "window" else (0, 0)
    return _batch(kind, size, batch, new, cached, dtype, index, mix, ones, window, sinks, single)


def _lens(case):
    """New tokens of each sequence, and all of its tokens with them."""
    rng = random.Random(case["mix"])
    new = [rng.randint(case["min_new"], case["max_new"]) for _ in range(case["batch"])]
    new = [1 if i < case["ones"] else n for i, n in enumerate(new)]
    return new, [n + rng.randint(case["min_cached"], case["max_cached"]) for n in new]


# ------------------------------------------------------------------ what a program holds before the call
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, it = DTYPES[case["dtype"]], INDEX[case["index"]]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    s = {"case": case}
    if case["kind"] == "append":
        tokens = case["tokens"]
        slots = tokens + tokens // 8 + 16
        rows = torch.randn(tokens, heads + 2 * kv_heads, d, generator=gen, device=dev).to(dt)
        s["q"], s["k_new"], s["v_new"] = rows.split([heads, kv_heads, kv_heads], 1)
        if not case["stacked"]:
            s["q"], s["k_new"], s["v_new"] = s["q"].contiguous(), s["k_new"].contiguous(), s["v_new"].contiguous()
        # the model's table of angles for 8192 positions, or the tokens' own rows of it
        freq = 10000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        at = torch.randint(0, 8192, (tokens,), generator=gen, device=dev)
        angle = torch.outer(torch.arange(8192, device=dev).double() if case["by_position"] else at.double(), freq)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = at.to(it) if case["by_position"] else None
        s["loc"] = torch.randperm(slots, generator=gen, device=dev)[:tokens].to(it)
        s["k"], s["v"] = [torch.zeros(slots, kv_heads, d, dtype=dt, device=dev) for _ in range(2)]
        return s
    # the paged pool: every sequence owns slots scattered over it for the tokens that are still seen, an eighth of it is free;
    # what a table holds of tokens that have left every window is stale
    new, lens = _lens(case)
    width = max(lens)
    seen = [_tokens_seen(case, n, length) for n, length in zip(new, lens)]
    total = sum(len(t) for t in seen)
    slots = total + total // 8 + 16
    mine = torch.randperm(slots, generator=gen, device=dev)[:total].to(it)
    s["b_loc"] = torch.randint(0, slots, (len(lens), width), generator=gen, device=dev).to(it)
    owner = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor([len(t) for t in seen]))
    column = torch.cat([torch.tensor(t, dtype=torch.int64) + (width - length) for t, length in zip(seen, lens)])  # the table is right-aligned
    s["b_loc"][owner.to(dev), column.to(dev)] = mine
    s["k"], s["v"] = [torch.randn(slots, kv_heads, d, generator=gen, device=dev).to(dt) for _ in range(2)]
    s["q"] = torch.randn(sum(new), heads, d, generator=gen, device=dev).to(dt)
    s["b_new_len"], s["b_seq_len"] = torch.tensor(new, dtype=it, device=dev), torch.tensor(lens, dtype=it, device=dev)
    s["b_start_loc"] = (torch.cumsum(s["b_new_len"], 0) - s["b_new_len"]).to(it)
    s["max_new"], s["max_len"] = max(new), width
    return s


def _tokens_seen(case, new, length):
    """The tokens of a sequence that one of its new ones sees."""
    first = max(0, length - new - case["window"] + 1) if case["window"] else 0
    return list(range(min(case["sinks"], first))) + list(range(first, length))


# ------------------------------------------------------------------ one pass
_ops = None


def _adapter():
    global _ops
    if _ops is None:
        from __graft_entry__ import load_package
        _ops = load_package().ops
    return _ops


def run(s):
    if own:
        return _run_own(s, _adapter())
    if s["case"]["kind"] == "append":
        return _append_plain(s)
    return _attention_plain(s).to(s["q"].dtype)


def _run_own(s, ops):
    case = s["case"]
    if case["kind"] == "append":
        q = ops.rotary_dest_index_copy_kv_pair(s["q"], s["k_new"], s["v_new"], s["cos"], s["sin"], s["loc"], s["k"], s["v"], positions=s["positions"],
                                               interleaved=case["interleaved"])
        return [q, s["k"], s["v"]]
    if case["single"]:
        return ops.token_decode_attention_window(s["q"], s["k"], s["v"], s["b_loc"], s["b_start_loc"], s["b_seq_len"], s["max_len"], case["window"], case["sinks"])
    return ops.paged_context_attention(s["q"], s["k"], s["v"], s["b_loc"], s["b_start_loc"], s["b_new_len"], s["b_seq_len"], s["max_new"], s["max_len"],
                                       window=case["window"], sinks=case["sinks"])


def _append_plain(s):
    loc = s["loc"].long()
    cos, sin = (s["cos"], s["sin"]) if s["positions"] is None else (s["cos"][s["positions"].long()], s["sin"][s["positions"].long()])
    s["k"][loc] = _rotated(s["k_new"], cos[:, None], sin[:, None], s["case"]["interleaved"])
    s["v"][loc] = s["v_new"]
    return [_rotated(s["q"], cos[:, None], sin[:, None], s["case"]["interleaved"]), s["k"], s["v"]]


def _rotated(x, cos, sin, interleaved):
    """Pairs (x[2 i], x[2 i + 1]), or (x[i], x[i + d / 2]), turned by angle i."""
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2].float(), x[..., 1::2].float()) if interleaved else (x[..., :half].float(), x[..., half:].float())
    a, b = a * cos - b * sin, a * sin + b * cos
    return (torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)).to(x.dtype)


def _attention_plain(s):
    """Scores, softmax and the sum over V of the tokens that each new token sees. Every sequence is as wide as the longest one;
    places outside it count for nothing."""
    case, q = s["case"], s["q"].float()
    heads, d = q.shape[1:]
    kv_heads, group = s["k"].shape[1], heads // s["k"].shape[1]
    new, lens, start = s["b_new_len"].long(), s["b_seq_len"].long(), s["b_start_loc"].long()
    batch, width = s["b_loc"].shape
    t = torch.arange(s["max_new"], device=q.device)
    row = torch.where(t < new[:, None], start[:, None] + t, -1)                            # batch, max_new: a new token's row of q
    place = lens[:, None] - new[:, None] + t                                               # and its position
    if case["single"]:     # the first tokens and the window alone
        j = torch.arange(case["sinks"] + case["window"], device=q.device)
        key = torch.where(j < case["sinks"], j, lens[:, None] - case["window"] + (j - case["sinks"]))
        key = torch.where((j < case["sinks"]) | (key >= case["sinks"]), key, -1)           # (a first token inside the window counts once)
    else:
        key = torch.arange(width, device=q.device).expand(batch, width)
    slot = torch.gather(s["b_loc"].long(), 1, (width - lens[:, None] + key).clamp(0, width - 1))
    key, place = key[:, None, :], place[:, :, None]
    sees = (key >= 0) & (key <= place)
    if case["window"]:
        sees = sees & ((key > place - case["window"]) | (key < case["sinks"]))
    k, v = [s[n][slot].float().permute(0, 2, 1, 3).repeat_interleave(group, 1) for n in "kv"]                 # batch, heads, keys, d
    scores = q[row.clamp(min=0)].transpose(1, 2) @ k.transpose(2, 3) / math.sqrt(d)                          # batch, heads, max_new, keys
    scores = scores.masked_fill_(~sees[:, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.transpose(1, 2)[row >= 0]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    size, index = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]], {"int32": 4, "int64": 8}[case["index"]]
    if case["kind"] == "append":
        t = case["tokens"]
        tables = 4 * d * (min(t, 8192) if case["by_position"] else t)                      # cos and sin, d / 2 fp32 each
        return {"bytes": 2 * t * (heads + 2 * kv_heads) * d * size + tables + t * index * (1 + case["by_position"]), "flops": 3 * t * (heads + kv_heads) * d}
    new, lens = _lens(case)
    rows = sum(len(_tokens_seen(case, n, length)) for n, length in zip(new, lens))
    pairs = sum(_pairs(case, n, length) for n, length in zip(new, lens))
    return {"bytes": rows * (2 * kv_heads * d * size + index) + 2 * sum(new) * heads * d * size, "flops": 4 * pairs * heads * d}


def _pairs(case, new, length):
    """(new token, token that it sees) pairs of a sequence."""
    seen = 0
    for place in range(length - new, length):
        n = place + 1
        if case["window"] and n > case["window"]:
            n = case["window"] + min(case["sinks"], n - case["window"])
        seen += n
    return seen


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        cos, sin = s["cos"].to(torch.float64), s["sin"].to(torch.float64)
        if case["by_position"]:
            cos, sin = cos.index_select(0, s["positions"].to(torch.int64)), sin.index_select(0, s["positions"].to(torch.int64))
        turn = torch.complex(cos, sin).unsqueeze(1)
        k, v, loc = s["k"].to(torch.float64), s["v"].to(torch.float64), s["loc"].to(torch.int64)
        return [_turned(s["q"], turn, case), k.index_copy(0, loc, _turned(s["k_new"], turn, case)), v.index_copy(0, loc, s["v_new"].to(torch.float64))]
    new, lens = _lens(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group, first = case["heads"] // case["kv_heads"], 0
    for b, (n, length) in enumerate(zip(new, lens)):
        at = torch.tensor(_tokens_seen(case, n, length), device=out.device)
        slots = s["b_loc"][b].to(torch.int64).index_select(0, at + (s["b_loc"].shape[1] - length))
        back = torch.arange(length - n, length, device=out.device).unsqueeze(1) - at       # how far behind a new token
        allowed = back >= 0
        if case["window"] > 0:
            allowed &= (back < case["window"]) | (at < case["sinks"])
        for g in range(case["kv_heads"]):
            k, v = s["k"][:, g].index_select(0, slots).double(), s["v"][:, g].index_select(0, slots).double()
            for h in range(g * group, (g + 1) * group):
                scores = torch.mm(s["q"][first:first + n, h].double(), k.t()) * case["d"] ** -0.5
                out[first:first + n, h] = torch.mm(torch.softmax(torch.where(allowed, scores, float("-inf")), -1), v)
        first += n
    return out


def _turned(x, turn, case):
    x, d = x.to(torch.float64), case["d"]
    pairs = x.unflatten(-1, (d // 2, 2)) if case["interleaved"] else x.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    return y.flatten(-2) if case["interleaved"] else y.transpose(-1, -2).flatten(-2)
