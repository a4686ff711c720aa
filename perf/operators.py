"""Performance cases of the paged key-value cache and the attention that reads it.

Three operators that a decoding program runs in every layer, each through
``fe2o3_amd.kernels`` on the program's own tensors:

  write   new tokens' K and V rows into their slots of a paged cache, copied
          (bf16) or quantised with a scale for each token and head (e4m3)
  read    cached rows of several sequences back into packed bf16 rows
  decode  attention of one new token a sequence over its pages, for shared and
          unshared heads, with its log-sum-exp

The cache holds pages of ``page_size`` tokens, either a token's heads next to
each other ("token" order) or a head's tokens ("head" order); the scales of an
e4m3 cache are [pages, kv_heads, page_size].  A block table names each
sequence's pages, which lie anywhere in the cache, as they do once sequences
have come and gone.

``own`` selects the framework's kernels; otherwise ``run`` computes the same
results with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
TINY = 1.17549435e-38   # the smallest normal float: the least amax a scale is made from
SCRATCH = 64 << 20      # bytes of device scratch that a serving program keeps


# ---- cases ------------------------------------------------------------------------------

def listed():
    return [
        # one user's chat turn, a short context: bound by launch and latency
        dict(name="decode_one_500", kind="decode", seqs=1, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, min_len=500, max_len=500, format="bf16", order="token", window=0),
        # one user with a very long context: only the cache's length can fill the device
        dict(name="decode_one_long", kind="decode", seqs=1, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, min_len=130001, max_len=130001, format="bf16", order="token",
             window=0),
        # an ordinary serving batch of mixed lengths, four query heads a KV head
        dict(name="decode_batch", kind="decode", seqs=32, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, min_len=1, max_len=4099, format="bf16", order="token", window=0),
        # the benchmark's attention shape with a head of K and V for every query head
        dict(name="decode_heads_4096", kind="decode", seqs=8, q_heads=32, kv_heads=32,
             head_dim=128, page_size=64, min_len=4096, max_len=4096, format="bf16",
             order="head", window=0),
        # the largest: many users on a quantised cache
        dict(name="decode_e4m3_batch", kind="decode", seqs=64, q_heads=32, kv_heads=8,
             head_dim=128, page_size=32, min_len=2, max_len=8190, format="e4m3", order="token",
             window=0),
        # one KV head for all query heads
        dict(name="decode_shared_head", kind="decode", seqs=48, q_heads=48, kv_heads=1,
             head_dim=128, page_size=32, min_len=100, max_len=6000, format="bf16",
             order="token", window=0),
        # short heads, pages of an odd size and a sliding window, some slots of the batch empty
        dict(name="decode_window_d64", kind="decode", seqs=40, q_heads=24, kv_heads=8,
             head_dim=64, page_size=24, min_len=0, max_len=5000, format="e4m3", order="head",
             window=1024),
        # a decoding step's new rows
        dict(name="write_step", kind="write", tokens=32, kv_heads=8, head_dim=128, page_size=16,
             pages=4096, format="bf16", order="token", padded=False),
        # a padded prompt batch quantised into pages of an odd size
        dict(name="write_e4m3_padded", kind="write", tokens=1000, kv_heads=8, head_dim=64,
             page_size=24, pages=100, format="e4m3", order="head", padded=True),
        # eight prompts of 4096 tokens, quantised
        dict(name="write_e4m3_prompts", kind="write", tokens=32768, kv_heads=8, head_dim=128,
             page_size=32, pages=1200, format="e4m3", order="token", padded=False),
        # one sequence's cached prefix, for a prompt that continues it
        dict(name="read_prefix", kind="read", seqs=1, kv_heads=8, head_dim=128, page_size=16,
             min_len=2001, max_len=2001, format="bf16", order="token"),
        # a batch's quantised prefixes, the last rows of the output padding
        dict(name="read_e4m3_batch", kind="read", seqs=16, kv_heads=8, head_dim=128,
             page_size=32, min_len=1, max_len=4097, format="e4m3", order="head"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "write", "read"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    head_dim = rng.choice([64, 128, 128])
    page_size = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    cache = dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size,
                 format=rng.choice(["bf16", "e4m3"]), order=rng.choice(["token", "head"]))
    row = kv_heads * head_dim
    if kind == "write":
        tokens = _log_int(rng, 1, max(1, min(32768, (1 << 25) // row)))
        pages = -(-tokens // page_size) + rng.randint(1, 64)
        return dict(cache, tokens=tokens, pages=pages, padded=rng.random() < 0.3)
    seqs = _log_int(rng, 1, 64)
    most = (1 << 25 if kind == "read" else 1 << 27) // (row * seqs)
    max_len = _log_int(rng, 1, max(1, min(131072, most)))
    min_len = rng.choice([max_len, max_len // 2, min(1, max_len), 0])
    cache.update(seqs=seqs, min_len=min_len, max_len=max_len)
    if kind == "read":
        return cache
    group = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    window = _log_int(rng, 1, max_len) if rng.random() < 0.2 else 0
    return dict(cache, q_heads=kv_heads * group, window=window)


# ---- inputs -----------------------------------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + part)


def _normal(shape, seed, part):
    return torch.randn(shape, generator=_generator(seed, part), device="cuda")


def _lengths(case):
    """A case's lengths, evenly spread; a seed only changes who has which."""
    n, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _cache(case, pages, seed):
    """A cache's arrays with rows in every slot, and views [pages, page_size, kv_heads, head_dim]."""
    h, d, n = case["kv_heads"], case["head_dim"], case["page_size"]
    token = case["order"] == "token"
    held = {}
    for part, name in enumerate("kv"):
        x = _normal((pages, n, h, d) if token else (pages, h, n, d), seed, 1 + part)
        if case["format"] == "bf16":
            x = x.to(torch.bfloat16)
        else:
            scale = (x.abs().amax(-1) / E4M3_MAX).clamp_min(TINY)
            x = (x / scale[..., None]).to(torch.float8_e4m3fn)
            held[name + "_scale"] = (scale.transpose(1, 2) if token else scale).contiguous()
        held[name] = x if token else x.transpose(1, 2)
    return held


def _table(case, lengths, pages, seed):
    """Block table of pages in random order; entries behind a sequence's pages are 0."""
    cols = max(1, -(-case["max_len"] // case["page_size"]))
    need = (lengths.long() + case["page_size"] - 1) // case["page_size"]
    order = torch.randperm(pages, generator=_generator(seed, 7), device="cuda")
    at = torch.cumsum(need, 0) - need
    col = torch.arange(cols, device="cuda")
    entry = (at[:, None] + col).clamp_max(pages - 1)
    return torch.where(col < need[:, None], order[entry], 0).to(torch.int32)


def prepare(case, seed):
    kind, h, d = case["kind"], case["kv_heads"], case["head_dim"]
    state = dict(case=case, kind=kind)
    if kind == "write":
        t = case["tokens"]
        state["cache"] = _cache(case, case["pages"], seed)
        # K and V are columns of one fused projection's output rows
        rows = _normal((t, 3, h, d), seed, 5).to(torch.bfloat16)
        state["k"], state["v"] = rows[:, 1], rows[:, 2]
        slots = torch.randperm(case["pages"] * case["page_size"], generator=_generator(seed, 6),
                               device="cuda")[:t].to(torch.int32)
        if case["padded"]:  # every fourth row is padding and has no slot
            slots[3::4] = -1
        state["slots"] = slots
        return state
    order = torch.randperm(case["seqs"], generator=_generator(seed, 8), device="cuda")
    lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order]
    pages = sum(-(-n // case["page_size"]) for n in _lengths(case)) + 3
    state["cache"] = _cache(case, pages, seed)
    state["table"] = _table(case, lengths, pages, seed)
    state["lengths"] = lengths
    if kind == "read":
        starts = torch.zeros(case["seqs"] + 1, device="cuda", dtype=torch.int32)
        starts[1:] = torch.cumsum(lengths, 0)
        state["starts"] = starts
        rows = sum(_lengths(case)) + 5  # a batch padded at its end
        for part, name in enumerate("kv"):
            state[name] = _normal((rows, h, d), seed, 9 + part).to(torch.bfloat16)
        return state
    state["q"] = _normal((case["seqs"], case["q_heads"], d), seed, 11).to(torch.bfloat16)
    state["out"] = torch.empty_like(state["q"])
    state["lse"] = torch.empty(case["seqs"], case["q_heads"], device="cuda")
    state["scratch"] = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    return state


# ---- one pass -----------------------------------------------------------------------------

def _widened(cache, name, page, offset):
    """Rows [..., kv_heads, head_dim] of a cache in 32 bits."""
    x = cache[name][page, offset].float()
    if name + "_scale" in cache:
        x = x * cache[name + "_scale"].transpose(1, 2)[page, offset][..., None]
    return x


def _plain_write(state):
    cache, n = state["cache"], state["case"]["page_size"]
    # a row without a slot repeats the first row, which has one
    slot = state["slots"].long()
    skip = slot < 0
    slot = torch.where(skip, slot[0], slot)
    for name in ("k", "v"):
        x = state[name].float()
        x = torch.where(skip[:, None, None], x[:1], x)
        if name + "_scale" in cache:
            scale = x.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
            x = (x / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
            cache[name + "_scale"].transpose(1, 2)[slot // n, slot % n] = scale
        cache[name][slot // n, slot % n] = x.to(cache[name].dtype)
    return cache


def _plain_read(state):
    starts, n = state["starts"].long(), state["case"]["page_size"]
    row = torch.arange(state["k"].shape[0], device="cuda")
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp_max(starts.numel() - 2)
    inside = row < starts[-1]
    at = torch.where(inside, row - starts[seq], 0)
    page = state["table"][seq, at // n].long()
    for name in ("k", "v"):
        x = _widened(state["cache"], name, page, at % n).to(torch.bfloat16)
        state[name].copy_(torch.where(inside[:, None, None], x, state[name]))
    return dict(k=state["k"], v=state["v"])


def _plain_decode(state):
    case, cache = state["case"], state["cache"]
    h, d, n = case["kv_heads"], case["head_dim"], case["page_size"]
    length = state["lengths"].long()[:, None]
    at = torch.arange(max(1, case["max_len"]), device="cuda")[None]
    page = state["table"][:, at[0] // n].long()
    keep = at < length
    if case["window"]:
        keep = keep & (at >= length - case["window"])
    keep = keep[:, None, None]
    q = state["q"].float().view(case["seqs"], h, -1, d)
    k = _widened(cache, "k", page, at % n).permute(0, 2, 3, 1)
    s = torch.matmul(q, k) * d ** -0.5
    del k
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    v = _widened(cache, "v", page, at % n).permute(0, 2, 1, 3)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    shape = (case["seqs"], case["q_heads"])
    state["out"].copy_(o.reshape(*shape, d))
    state["lse"].copy_(lse.reshape(shape))
    return dict(out=state["out"], lse=state["lse"])


def run(state):
    kind, case = state["kind"], state["case"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode}[kind](state)
    from fe2o3_amd import kernels
    held = state["cache"]
    cache = kernels.KvCache(held["k"], held["v"], held.get("k_scale"), held.get("v_scale"))
    if kind == "write":
        kernels.kv_cache_write(cache, state["k"], state["v"], state["slots"], sync=False)
        return held
    if kind == "read":
        kernels.kv_cache_read(cache, state["table"], state["starts"], state["k"], state["v"],
                              sync=False)
        return dict(k=state["k"], v=state["v"])
    kernels.paged_attention_decode(cache, state["q"], state["table"], state["lengths"],
                                   state["out"], state["lse"], state["scratch"],
                                   max_length=case["max_len"], window=case["window"],
                                   scale=case["head_dim"] ** -0.5, sync=False)
    return dict(out=state["out"], lse=state["lse"])


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    h, d = case["kv_heads"], case["head_dim"]
    # one token's K and V as the cache holds them, and as bf16
    cached = 2 * h * (2 * d if case["format"] == "bf16" else d + 4)
    plain = 2 * h * 2 * d
    if case["kind"] == "write":
        rows = case["tokens"] - (case["tokens"] // 4 if case["padded"] else 0)
        return dict(bytes=rows * (plain + cached) + 4 * case["tokens"], flops=2 * rows * 2 * h * d)
    lengths = _lengths(case)
    if case["kind"] == "read":
        return dict(bytes=sum(lengths) * (plain + cached) + 4 * sum(
            1 - (-n // case["page_size"]) for n in lengths), flops=sum(lengths) * 2 * h * d)
    keys = [min(n, case["window"]) if case["window"] else n for n in lengths]
    tables = 4 * sum(1 - (-n // case["page_size"]) for n in keys)
    heads = case["seqs"] * case["q_heads"]
    return dict(bytes=sum(keys) * cached + heads * (4 * d + 4) + tables,
                flops=4 * sum(keys) * case["q_heads"] * d)


# ---- the definitions in 64 bits ---------------------------------------------------------------

def _e4m3_nearest(x):
    """Nearest e4m3 value of 64-bit numbers within its range, ties to even."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -40))).clamp_min(-6.0)
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _row64(state, name, seq, count):
    """The first `count` rows of one sequence, [count, kv_heads, head_dim] in 64 bits."""
    cache, n = state["cache"], state["case"]["page_size"]
    pages = state["table"][seq, :-(-count // n)].long()
    x = cache[name][pages].double()
    if name + "_scale" in cache:
        x = x * cache[name + "_scale"][pages].double().permute(0, 2, 1)[..., None]
    return x.reshape(-1, *x.shape[2:])[:count]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "write":
        out = {name: x.double() for name, x in state["cache"].items()}
        kept = state["slots"] >= 0
        slots = state["slots"][kept].long()
        page, offset = slots // case["page_size"], slots % case["page_size"]
        for name in ("k", "v"):
            x = state[name][kept].double()
            if case["format"] == "e4m3":
                scale = x.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
                x = _e4m3_nearest(x / scale[..., None])
                out[name + "_scale"][page, :, offset] = scale
            out[name][page, offset] = x
        return out
    lengths = state["lengths"].tolist()
    if case["kind"] == "read":
        out = {}
        for name in ("k", "v"):
            out[name] = state[name].double()
            start = 0
            for seq, count in enumerate(lengths):
                if count:
                    out[name][start:start + count] = _row64(state, name, seq, count)
                start += count
        return out
    heads, group = case["q_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(case["seqs"], heads, case["head_dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((case["seqs"], heads), -math.inf, dtype=torch.float64, device="cuda")
    for seq, count in enumerate(lengths):
        if count == 0:
            continue
        first = max(0, count - case["window"]) if case["window"] else 0
        k = _row64(state, "k", seq, count)[first:]
        v = _row64(state, "v", seq, count)[first:]
        for head in range(case["kv_heads"]):
            mine = slice(head * group, (head + 1) * group)
            s = state["q"][seq, mine].double() @ k[:, head].T.contiguous() / math.sqrt(case["head_dim"])
            lse[seq, mine] = torch.logsumexp(s, -1)
            out[seq, mine] = torch.softmax(s, -1) @ v[:, head].contiguous()
    return dict(out=out, lse=lse)
