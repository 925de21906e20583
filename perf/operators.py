"""The measured operators around the paged KV cache, each in its plain form and through the op adapter (`ops`).

  turnover   new K and V rows are quantised to int8 as they are written into the cache (a scale for each token and head),
             and the rows written are read back in the activations' type, as the next piece of a long prompt reads them
  read       cached int8 rows are read back alone: a sequence that continues after others had the machine
  int8       decode attention over the int8 cache
  prefix     decode attention of a batch whose sequences all begin with the same long prefix, kept once in the cache

Sequence lengths are drawn from [min_len, max_len] by the case's own `mix`, so that all seeds of a case do the same work;
everything else that a state holds comes from the seed. `index` is the type of slot tables, lengths and destinations.
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


def _case(kind, size, dtype, index="int32", mix=0, **more):
    heads, kv_heads, d = size
    return dict(kind=kind, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, index=index, mix=mix, **more)


def _rows(kind, size, tokens, dtype, index="int32", stacked=False, **more):
    return _case(kind, size, dtype, index, tokens=tokens, stacked=stacked, **more)


def _batch(kind, size, batch, min_len, max_len, dtype, index="int32", mix=0, prefix=0, **more):
    return _case(kind, size, dtype, index, mix, batch=batch, min_len=min_len, max_len=max_len, prefix=prefix, **more)


def listed():
    return [
        # a decode step of 64 sequences: one row each, all launch latency
        _rows("turnover", BASE, 64, "bf16", name="turnover_64_bf16"),
        # a prompt on grouped K/V heads, its K and V slices of the stacked projection's rows
        _rows("turnover", GROUPED, 1777, "fp16", "int64", stacked=True, name="turnover_1777_stacked_fp16"),
        # the benchmark layer's full batch of prompts, 4 x 2048 tokens
        _rows("turnover", BASE, 8192, "bf16", name="turnover_8192_bf16"),
        # a chat turn that comes back: a few hundred cached tokens on grouped heads
        _rows("read", GROUPED, 301, "fp16", name="read_301_fp16"),
        # a long document's cache
        _rows("read", WIDE, 15001, "bf16", "int64", name="read_15001_bf16"),
        # one user waiting for a token: the latency of a small batch
        _batch("int8", GROUPED, 1, 1777, 1777, "bf16", name="int8_1x1777_bf16"),
        # the fp32 parity configuration's heads, short sequences of very different lengths
        _batch("int8", SMALL, 16, 1, 300, "fp32", "int64", mix=1, name="int8_16_short_fp32"),
        # the throughput end of decoding on grouped K/V heads
        _batch("int8", GROUPED, 48, 512, 4096, "fp16", mix=2, name="int8_48_grouped_fp16"),
        # the same with a K/V head for each query head: the largest cache
        _batch("int8", BASE, 64, 512, 4096, "bf16", mix=3, name="int8_64_bf16"),
        # a few short answers under one system prompt in the fp32 parity configuration's heads
        _batch("prefix", SMALL, 5, 1, 60, "fp32", mix=4, prefix=777, name="prefix_777_5_fp32"),
        # many users of one assistant: a system prompt and a conversation each
        _batch("prefix", BASE, 64, 64, 512, "bf16", mix=5, prefix=2048, name="prefix_2048_64_bf16"),
        # questions about one long document on grouped K/V heads
        _batch("prefix", GROUPED, 48, 16, 300, "fp16", "int64", mix=6, prefix=16001, name="prefix_16001_48_fp16"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["turnover", "read", "int8", "int8", "int8", "prefix", "prefix", "prefix"])
    heads, kv_heads, d = rng.choice([SMALL, BASE, GROUPED, WIDE, LARGE])
    size = heads, kv_heads, rng.choice([d, d, d, 64, 80, 96, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    index = rng.choice(["int32", "int32", "int64"])
    mix = rng.randrange(1 << 20)
    row = size[1] * size[2]
    if kind in ("turnover", "read"):
        most = min(16384, 8192 * 4096 // row)
        return _rows(kind, size, _spread(rng, 1, most), dtype, index, kind == "turnover" and rng.random() < 0.3, mix=mix)
    batch = _spread(rng, 1, 64)
    most = 64 * 2304 * 4096 // (row * batch)                     # tokens of a sequence: no more work than the largest listed case
    if dtype == "fp32":
        most //= 4
    if kind == "int8":
        high = _spread(rng, 1, max(2, min(16384, most)))
        low = rng.choice([high, rng.randint(0, high), high // rng.randint(2, 16)])
        return _batch(kind, size, batch, low, high, dtype, index, mix)
    high = _spread(rng, 1, max(2, min(2048, most // 4)))
    low = rng.choice([high, rng.randint(0, high), high // rng.randint(2, 16)])
    return _batch(kind, size, batch, low, high, dtype, index, mix, prefix=_spread(rng, 1, max(2, min(32768, most // 4))))


def _lens(case):
    """Tokens of each sequence (behind the prefix, where there is one)."""
    rng = random.Random(case["mix"])
    return [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]


# ------------------------------------------------------------------ what a program holds before the call
def _int8_pool(slots, case, gen, dev):
    """A filled int8 cache: values as rows of normal numbers leave them (the largest of a row at 127, a deviation of about
    45), scales so that what they stand for has a deviation of one, more or less by head."""
    shape = slots, case["kv_heads"], case["d"]
    pool = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16).mul_(45).round_().clamp_(-127, 127).to(torch.int8)
    scale = (0.5 + torch.rand(shape[:2], generator=gen, device=dev)) / 45
    return pool, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, it = DTYPES[case["dtype"]], INDEX[case["index"]]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    s = {"case": case}
    if case["kind"] in ("turnover", "read"):
        tokens = case["tokens"]
        slots = tokens + tokens // 8 + 16
        s["loc"] = torch.randperm(slots, generator=gen, device=dev)[:tokens].to(it)
        if case["kind"] == "read":
            (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = [_int8_pool(slots, case, gen, dev) for _ in range(2)]
            return s
        # heads differ in size, and a few places of a head stand out, as in the keys of trained models
        spread = (0.25 + torch.rand(kv_heads, 1, generator=gen, device=dev) * 2) * (1 + 7 * (torch.rand(kv_heads, d, generator=gen, device=dev) < 0.03))
        make = lambda: (torch.randn(tokens, kv_heads, d, generator=gen, device=dev) * spread).to(dt)
        if case["stacked"]:
            rows = torch.cat([torch.randn(tokens, heads, d, generator=gen, device=dev).to(dt), make(), make()], dim=1)
            s["k_new"], s["v_new"] = rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
        else:
            s["k_new"], s["v_new"] = make(), make()
        for n in "kv":
            s[n] = torch.zeros(slots, kv_heads, d, dtype=torch.int8, device=dev)
            s[n + "_scale"] = torch.zeros(slots, kv_heads, device=dev)
        return s
    # the paged pool: every sequence owns slots scattered over it, an eighth of it is free
    lens = _lens(case)
    total, width = sum(lens) + case["prefix"], max(max(lens), 1)
    slots = total + total // 8 + 16
    perm = torch.randperm(slots, generator=gen, device=dev).to(it)
    s["q"] = torch.randn(len(lens), heads, d, generator=gen, device=dev).to(dt)
    s["prefix_loc"], mine = perm[:case["prefix"]], perm[case["prefix"]:total]
    s["b_seq_len"] = torch.tensor(lens, dtype=it, device=dev)
    s["b_start_loc"] = (torch.cumsum(s["b_seq_len"], 0) - s["b_seq_len"]).to(it)
    s["max_len"] = max(lens)
    owner = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    column = torch.cat([torch.arange(width - n, width) for n in lens])                   # the table is right-aligned
    s["b_loc"] = torch.zeros(len(lens), width, dtype=it, device=dev)
    s["b_loc"][owner.to(dev), column.to(dev)] = mine
    if case["kind"] == "int8":
        (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = [_int8_pool(slots, case, gen, dev) for _ in range(2)]
    else:
        for n in "kv":
            s[n] = torch.randn(slots, kv_heads, d, generator=gen, device=dev).to(dt)
    return s


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
    kind = s["case"]["kind"]
    if kind == "turnover":
        for n in "kv":
            _write_plain(s[n + "_new"], s["loc"].long(), s[n], s[n + "_scale"])
    if kind in ("turnover", "read"):
        return [_read_plain(s[n], s[n + "_scale"], s["loc"].long()).to(DTYPES[s["case"]["dtype"]]) for n in "kv"]
    return _attention_plain(s).to(s["q"].dtype)


def _run_own(s, ops):
    kind = s["case"]["kind"]
    if kind == "turnover":
        ops.dest_index_copy_kv_pair_int8(s["k_new"], s["v_new"], s["loc"], s["k"], s["k_scale"], s["v"], s["v_scale"])
    if kind in ("turnover", "read"):
        return ops.index_select_kv_pair_int8(s["k"], s["k_scale"], s["v"], s["v_scale"], s["loc"], dtype=DTYPES[s["case"]["dtype"]])
    if kind == "int8":
        return ops.token_decode_attention_int8(s["q"], s["k"], s["k_scale"], s["v"], s["v_scale"], s["b_loc"], s["b_start_loc"],
                                               s["b_seq_len"], s["max_len"])
    return ops.token_decode_attention_shared_prefix(s["q"], s["k"], s["v"], s["prefix_loc"], s["b_loc"], s["b_start_loc"],
                                                    s["b_seq_len"], s["max_len"])


def _write_plain(x, loc, pool, scale):
    """scale = the largest magnitude of a row / 127 as fp32; int8 = the whole number nearest to x / scale, ties to the even
    one (quotients in 64 bits: in 32, one that lies next to a half would be taken for it)."""
    x = x.double()
    s = (x.abs().amax(-1) / 127).float()
    q = torch.where(s[..., None] > 0, x / s.double()[..., None], 0).round()
    pool[loc], scale[loc] = q.to(torch.int8), s


def _read_plain(pool, scale, loc):
    return pool[loc].float() * scale[loc][..., None]


def _attention_plain(s):
    """Scores, softmax and the sum over V of all tokens that a sequence sees: those of its row of the table, at the right
    end, and the prefix. Every sequence is as wide as the table; places outside it count for nothing."""
    q, loc, lens = s["q"].float(), s["b_loc"].long(), s["b_seq_len"].long()
    batch, heads, d = q.shape
    kv_heads = s["k"].shape[1]
    rows = (lambda n, i: _read_plain(s[n], s[n + "_scale"], i)) if "k_scale" in s else (lambda n, i: s[n][i].float())
    q = q.view(batch, kv_heads, heads // kv_heads, d) / math.sqrt(d)
    counts = (torch.arange(loc.shape[1], device=q.device) >= loc.shape[1] - lens[:, None])[:, None, None]   # batch, 1, 1, width
    scores = q @ rows("k", loc).permute(0, 2, 3, 1)                                          # batch, kv_heads, group, width
    scores = scores.masked_fill_(~counts, -math.inf)
    prefix = s["prefix_loc"].long()
    by_head = lambda x: x.transpose(0, 1).reshape(kv_heads, batch * heads // kv_heads, x.shape[-1])  # the batch's rows of each K/V head
    back = lambda x: x.view(kv_heads, batch, heads // kv_heads, x.shape[-1]).transpose(0, 1)
    shared = back(by_head(q) @ rows("k", prefix).permute(1, 2, 0))
    top = torch.cat([scores, shared], -1).amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p, ps = torch.exp(scores - top), torch.exp(shared - top)
    total = p.sum(-1, keepdim=True) + ps.sum(-1, keepdim=True)
    out = p @ rows("v", loc).transpose(1, 2) + back(by_head(ps) @ rows("v", prefix).transpose(0, 1))
    return torch.where(total > 0, out / total, 0).reshape(batch, heads, d)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    size, index = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]], {"int32": 4, "int64": 8}[case["index"]]
    int8_row = 2 * kv_heads * (d + 4)
    if case["kind"] in ("turnover", "read"):
        t, rows = case["tokens"], 2 * kv_heads * d
        passes = 2 if case["kind"] == "turnover" else 1
        return {"bytes": t * (passes * rows * size + int8_row + index), "flops": t * rows * (4 * passes - 3)}
    lens = _lens(case)
    tokens = sum(lens) + case["prefix"]
    row = int8_row if case["kind"] == "int8" else 2 * kv_heads * d * size
    seen = sum(lens) + len(lens) * case["prefix"]
    return {"bytes": tokens * (row + index) + 2 * len(lens) * heads * d * size, "flops": 4 * seen * heads * d}


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "turnover":
        return [_stored(s["k_new"]), _stored(s["v_new"])]
    if case["kind"] == "read":
        return [s[n].double()[s["loc"].long()] * s[n + "_scale"].double()[s["loc"].long()].unsqueeze(-1) for n in "kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["heads"] // case["kv_heads"]

    def values(name, slots):
        x = s[name].index_select(0, slots).double()
        if case["kind"] == "int8":
            x *= s[name + "_scale"].index_select(0, slots).double()[:, :, None]
        return x.movedim(1, 0)                                       # kv_heads, tokens, d

    prefix = s["prefix_loc"].to(torch.int64)
    pk, pv = values("k", prefix), values("v", prefix)
    for b, n in enumerate(_lens(case)):
        if n + len(prefix) == 0:
            continue
        slots = s["b_loc"][b, s["b_loc"].shape[1] - n:].to(torch.int64)
        k, v = torch.cat([pk, values("k", slots)], 1), torch.cat([pv, values("v", slots)], 1)
        for j in range(group):
            w = torch.softmax((k * s["q"][b, j::group].double()[:, None]).sum(-1) * d_root(case), -1)
            out[b, j::group] = (w.unsqueeze(-1) * v).sum(1)
    return out


def d_root(case):
    return case["d"] ** -0.5


def _stored(x):
    x = x.to(torch.float64)
    most = x.abs().max(dim=-1, keepdim=True).values
    step = (most / 127).to(torch.float32).to(torch.float64)
    return torch.where(step > 0, torch.round(x / step) * step, torch.zeros_like(x))
