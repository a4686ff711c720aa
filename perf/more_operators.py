"""Performance cases of 4-bit inference: microscaled matrices and caches, and rotary positions.

Five operators around the microscaled 4-bit format (e2m1 elements, 32 of them on one
power-of-two scale), and the rotation that stands between a projection and the cache,
each through ``fe2o3_amd.kernels`` on the program's own tensors:

  quantize  a matrix into packed 4-bit codes and scales, and back into its own type
  product   C = A B^T of two packed matrices
  cache     new tokens' K and V rows quantised into their slots of a paged 4-bit cache,
            and the sequences' rows read back as packed bf16
  decode    attention of one new token a sequence over a 4-bit cache
  rotary    rotary positions of Q and K, and their gradient

A packed matrix of [rows, cols] holds panels of 256 columns: codes [rows, panels * 128]
(two to a byte, the even column in the low half) and scales [panels, rows rounded up to
16, 8], the eight blocks of a row's panel beside each other.  Columns past the last are
zeros.  A scale is the byte e of 2^(e - 127); 255 stands for NaN.  A 4-bit cache holds a
row's codes in head_dim / 2 bytes, and its scales as [pages, kv_heads, page_size,
head_dim / 32].

``own`` selects the framework's kernels; otherwise ``run`` computes the same results
with elementary torch operations in 32 bits (angles in 64).
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32      # elements on one scale
PANEL = 256     # columns of a panel
SCRATCH = 64 << 20      # bytes of device scratch that a serving program keeps
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases ------------------------------------------------------------------------------

def listed():
    return [
        # a decoding step's activations, quantised before a linear: bound by launches
        dict(name="quantize_step", kind="quantize", rows=33, cols=4096, dtype="bf16"),
        # a feed-forward weight, quantised from the optimizer's copy and checked against it
        dict(name="quantize_weight", kind="quantize", rows=14336, cols=4096, dtype="f32"),
        # a decoding step's linear: the weights' stream
        dict(name="product_step", kind="product", m=16, n=14336, k=4096),
        # odd sizes everywhere, a cut panel
        dict(name="product_ragged", kind="product", m=1000, n=1500, k=700),
        # a whole prompt batch through the widest linear
        dict(name="product_8192", kind="product", m=8192, n=8192, k=8192),
        # one prompt's next chunk into pages of an odd size, and its whole prefix back
        dict(name="cache_chunk", kind="cache", seqs=1, new=999, length=2001, kv_heads=8,
             head_dim=64, page_size=24, order="head"),
        # eight prompts of 4096 tokens
        dict(name="cache_prompts", kind="cache", seqs=8, new=4096, length=4096, kv_heads=8,
             head_dim=128, page_size=32, order="token"),
        # one user's chat turn, a short context: latency
        dict(name="decode_one_500", kind="decode", seqs=1, q_heads=32, kv_heads=8, head_dim=128,
             page_size=16, min_len=500, max_len=500, order="token", window=0),
        # many users of mixed lengths: the cache's stream
        dict(name="decode_batch", kind="decode", seqs=64, q_heads=32, kv_heads=8, head_dim=128,
             page_size=32, min_len=2, max_len=8190, order="token", window=0),
        # short heads, pages of an odd size and a sliding window, some slots of the batch empty
        dict(name="decode_window_d64", kind="decode", seqs=40, q_heads=24, kv_heads=8,
             head_dim=64, page_size=24, min_len=0, max_len=5000, order="head", window=1024),
        # a decoding step far into a stretched context: interleaved pairs, half of the head
        dict(name="rotary_step", kind="rotary", tokens=32, q_heads=32, kv_heads=8, head_dim=128,
             rotary_dim=64, first=130000, spread=50000, interleaved=True, inverse=False,
             factor=8.0, dtype="bf16"),
        # the gradient of a training step's four sequences of 4096 tokens
        dict(name="rotary_grad", kind="rotary", tokens=16384, q_heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, first=0, spread=4096, interleaved=False, inverse=True,
             factor=1.0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "cache", "decode", "decode", "rotary"])
    if kind == "quantize":
        cols = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, max(1, min(65536, (1 << 25) // cols)))
        return dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(["bf16", "f32"]))
    if kind == "product":
        n, k = _log_int(rng, 16, 16384), _log_int(rng, 32, 16384)
        m = _log_int(rng, 1, max(1, min(8192, (1 << 38) // (n * k))))
        return dict(kind=kind, m=m, n=n, k=k)
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    head_dim = rng.choice([64, 128, 128])
    row = kv_heads * head_dim
    if kind == "rotary":
        group = rng.choice([1, 2, 3, 4, 4, 7, 8])
        tokens = _log_int(rng, 1, max(1, min(16384, (1 << 25) // (row * (group + 1)))))
        return dict(kind=kind, tokens=tokens, q_heads=kv_heads * group, kv_heads=kv_heads,
                    head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2,
                                                              head_dim // 4 + 4]),
                    first=rng.choice([0, _log_int(rng, 1, 1 << 20)]),
                    spread=_log_int(rng, 1, 131072), interleaved=rng.random() < 0.5,
                    inverse=rng.random() < 0.4, factor=rng.choice([1.0, 1.0, 4.0, 32.0]),
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
    cache = dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim,
                 page_size=rng.choice([8, 16, 16, 24, 32, 64, 128, 256]),
                 order=rng.choice(["token", "head"]))
    if kind == "cache":
        seqs = _log_int(rng, 1, 32)
        length = _log_int(rng, 1, max(1, min(32768, (1 << 25) // (row * seqs))))
        return dict(cache, seqs=seqs, length=length, new=_log_int(rng, 1, length))
    seqs = _log_int(rng, 1, 64)
    max_len = _log_int(rng, 1, max(1, min(131072, (1 << 27) // (row * seqs))))
    min_len = rng.choice([max_len, max_len // 2, min(1, max_len), 0])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    window = _log_int(rng, 1, max_len) if rng.random() < 0.2 else 0
    return dict(cache, seqs=seqs, min_len=min_len, max_len=max_len, q_heads=kv_heads * group,
                window=window)


# ---- the 4-bit format --------------------------------------------------------------------

def _scale_of(code):
    """2^(e - 127) of scale bytes, NaN of 255, in 32 bits."""
    e = code.to(torch.int32)
    # 2^-127 lies below the normal range: half of 2^-126
    scale = (e.clamp_min(1) << 23).view(torch.float32)
    scale = torch.where(e == 0, scale * 0.5, scale)
    return torch.where(e == 255, math.nan, scale)


def _encode(x):
    """Codes (one a byte) and scale bytes of blocks [..., 32] in 32 bits."""
    top = x.abs().amax(-1)
    e = top.contiguous().view(torch.int32) >> 23
    # a NaN or an infinity in the block has the exponent 255
    scale = torch.where(e == 255, 255, (e - 2).clamp_min(0)).to(torch.uint8)
    y = (x / _scale_of(scale)[..., None]).abs()
    # the nearest of the magnitudes, ties to the even code
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5)
            + (y >= 3.5) + (y > 5.0))
    return code + 8 * torch.signbit(x).to(torch.uint8), scale


def _two_to_a_byte(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def _values(packed):
    """The values of packed codes [..., n] as [..., 2 n] in 32 bits."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=packed.device)
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return table[code.int()]


def _panels(cols):
    return -(-cols // PANEL)


def _pack_matrix(x):
    """(codes, scales) of a matrix, as the product takes them."""
    rows, cols = x.shape
    panels = _panels(cols)
    wide = torch.zeros(rows, panels * PANEL, device=x.device)
    wide[:, :cols] = x
    code, scale = _encode(wide.view(rows, panels, 8, BLOCK))
    scales = torch.zeros(panels, -(-rows // 16) * 16, 8, dtype=torch.uint8, device=x.device)
    scales[:, :rows] = scale.transpose(0, 1)
    return _two_to_a_byte(code).view(rows, panels * PANEL // 2), scales


def _unpack_matrix(codes, scales):
    """The matrix, padding columns among it, in 32 bits."""
    rows, panels = codes.shape[0], scales.shape[0]
    scale = _scale_of(scales[:, :rows]).transpose(0, 1)
    x = _values(codes).view(rows, panels, 8, BLOCK) * scale[..., None]
    return x.view(rows, panels * PANEL)


# ---- inputs -----------------------------------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + part)


def _normal(shape, seed, part):
    return torch.randn(shape, generator=_generator(seed, part), device="cuda")


def _channels(shape, seed, part):
    """Activations: a few of the last dimension's channels are many times the others."""
    x = _normal(shape, seed, part)
    gain = torch.exp(_normal(shape[-1:], seed, part + 100))
    return x * gain


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _lengths(case):
    """A decode's lengths, evenly spread; a seed only changes who has which."""
    n, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _cache(case, pages, seed):
    """A cache's arrays with rows in every slot, and views [pages, page_size, kv_heads,
    head_dim / 2]."""
    h, d, n = case["kv_heads"], case["head_dim"], case["page_size"]
    token = case["order"] == "token"
    held = {}
    for part, name in enumerate("kv"):
        x = _channels((pages, n, h, d) if token else (pages, h, n, d), seed, 1 + part)
        code, scale = _encode(x.to(torch.bfloat16).float().unflatten(-1, (d // BLOCK, BLOCK)))
        code = _two_to_a_byte(code).flatten(-2)
        held[name] = code if token else code.transpose(1, 2)
        held[name + "_scale"] = (scale.transpose(1, 2) if token else scale).contiguous()
    return held


def _table(case, lengths, cols, pages, seed):
    """Block table of pages in random order; entries behind a sequence's pages are 0."""
    need = (lengths.long() + case["page_size"] - 1) // case["page_size"]
    order = torch.randperm(pages, generator=_generator(seed, 7), device="cuda")
    at = torch.cumsum(need, 0) - need
    col = torch.arange(cols, device="cuda")
    entry = (at[:, None] + col).clamp_max(pages - 1)
    return torch.where(col < need[:, None], order[entry], 0).to(torch.int32)


def _prepare_quantize(case, seed):
    rows, cols = case["rows"], case["cols"]
    x = _channels((rows, cols), seed, 1).to(_dtype(case))
    panels = _panels(cols)
    return dict(
        x=x, out=torch.empty_like(x),
        codes=torch.empty(rows, panels * PANEL // 2, dtype=torch.uint8, device="cuda"),
        scales=torch.zeros(panels, -(-rows // 16) * 16, 8, dtype=torch.uint8, device="cuda"))


def _prepare_product(case, seed):
    a = _pack_matrix(_channels((case["m"], case["k"]), seed, 1).to(torch.bfloat16).float())
    b = _pack_matrix(_normal((case["n"], case["k"]), seed, 2) * case["k"] ** -0.5)
    c = torch.empty(case["m"], case["n"], dtype=torch.bfloat16, device="cuda")
    return dict(a=a[0], a_scale=a[1], b=b[0], b_scale=b[1], c=c)


def _prepare_cache(case, seed):
    n, h, d = case["seqs"], case["kv_heads"], case["head_dim"]
    length, new, page_size = case["length"], case["new"], case["page_size"]
    cols = -(-length // page_size)
    lengths = torch.full((n,), length, device="cuda")
    state = dict(cache=_cache(case, n * cols + 3, seed))
    state["table"] = table = _table(case, lengths, cols, n * cols + 3, seed)
    at = torch.arange(length - new, length, device="cuda")
    slots = table[:, at // page_size].long() * page_size + at % page_size
    state["slots"] = slots.flatten().to(torch.int32)
    state["starts"] = (torch.arange(n + 1, device="cuda") * length).to(torch.int32)
    # the new K and V are columns of one fused projection's output rows
    rows = _channels((n * new, 3, h, d), seed, 5).to(torch.bfloat16)
    state["k"], state["v"] = rows[:, 1], rows[:, 2]
    for name in ("k_out", "v_out"):  # a batch padded at its end
        state[name] = torch.zeros(n * length + 5, h, d, dtype=torch.bfloat16, device="cuda")
    return state


def _prepare_decode(case, seed):
    order = torch.randperm(case["seqs"], generator=_generator(seed, 8), device="cuda")
    lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order]
    pages = sum(-(-n // case["page_size"]) for n in _lengths(case)) + 3
    cols = max(1, -(-case["max_len"] // case["page_size"]))
    q = _normal((case["seqs"], case["q_heads"], case["head_dim"]), seed, 11).to(torch.bfloat16)
    # queries of a size that gives scores of a few units over the cache's channels
    q = q / 2
    return dict(cache=_cache(case, pages, seed), table=_table(case, lengths, cols, pages, seed),
                lengths=lengths, q=q, out=torch.empty_like(q),
                lse=torch.empty(case["seqs"], case["q_heads"], device="cuda"),
                scratch=torch.empty(SCRATCH, dtype=torch.uint8, device="cuda"))


def _frequencies(case):
    """Radians a position for each pair, the slow pairs stretched over a context `factor`
    times as long: the user's own table, in 64 bits."""
    r = case["rotary_dim"]
    i = torch.arange(r // 2, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / r)
    # pairs of over 32 turns in 4096 tokens keep their speed, those under one are slowed
    turns = 4096 * freq / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return freq * (keep + (1 - keep) / case["factor"])


def _prepare_rotary(case, seed):
    t, h, g, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    # columns of one fused projection's output rows
    rows = _normal((t, h + 2 * g, d), seed, 1).to(_dtype(case))
    at = torch.randint(0, case["spread"], (t,), generator=_generator(seed, 2), device="cuda")
    q, k = rows[:, :h], rows[:, h:h + g]
    return dict(q=q, k=k, positions=(case["first"] + at).to(torch.int32),
                freq=_frequencies(case).cuda(), scale=0.1 * math.log(case["factor"]) + 1.0,
                q_out=torch.empty(q.shape, dtype=q.dtype, device="cuda"),
                k_out=torch.empty(k.shape, dtype=k.dtype, device="cuda"))


def prepare(case, seed):
    state = dict(quantize=_prepare_quantize, product=_prepare_product, cache=_prepare_cache,
                 decode=_prepare_decode, rotary=_prepare_rotary)[case["kind"]](case, seed)
    return dict(state, case=case)


# ---- one pass, plain ----------------------------------------------------------------------

def _plain_quantize(state):
    codes, scales = _pack_matrix(state["x"].float())
    state["codes"].copy_(codes)
    state["scales"].copy_(scales)
    x = _unpack_matrix(state["codes"], state["scales"])
    state["out"].copy_(x[:, :state["x"].shape[1]])
    return state["out"]


def _plain_product(state):
    a = _unpack_matrix(state["a"], state["a_scale"])
    b = _unpack_matrix(state["b"], state["b_scale"])
    state["c"].copy_(torch.matmul(a, b.T))
    return state["c"]


def _rows_of(cache, name, page, place):
    """Rows [..., kv_heads, head_dim] of a cache in 32 bits."""
    x = _values(cache[name][page, place])
    scale = _scale_of(cache[name + "_scale"].transpose(1, 2)[page, place])
    return (x.unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)


def _plain_cache(state):
    cache, n = state["cache"], state["case"]["page_size"]
    slot = state["slots"].long()
    for name in ("k", "v"):
        code, scale = _encode(state[name].float().unflatten(-1, (-1, BLOCK)))
        cache[name][slot // n, slot % n] = _two_to_a_byte(code).flatten(-2)
        cache[name + "_scale"].transpose(1, 2)[slot // n, slot % n] = scale
    starts = state["starts"].long()
    row = torch.arange(state["k_out"].shape[0], device="cuda")
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp_max(starts.numel() - 2)
    inside = row < starts[-1]
    at = torch.where(inside, row - starts[seq], 0)
    page = state["table"][seq, at // n].long()
    for name in ("k", "v"):
        x = _rows_of(cache, name, page, at % n).to(torch.bfloat16)
        out = state[name + "_out"]
        out.copy_(torch.where(inside[:, None, None], x, out))
    return dict(k=state["k_out"], v=state["v_out"])


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
    k = _rows_of(cache, "k", page, at % n).permute(0, 2, 3, 1)
    s = torch.matmul(q, k) * d ** -0.5
    del k
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    v = _rows_of(cache, "v", page, at % n).permute(0, 2, 1, 3)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    shape = (case["seqs"], case["q_heads"])
    state["out"].copy_(o.reshape(*shape, d))
    state["lse"].copy_(lse.reshape(shape))
    return dict(out=state["out"], lse=state["lse"])


def _plain_rotary(state):
    case = state["case"]
    r = case["rotary_dim"]
    angle = state["positions"].double()[:, None, None] * state["freq"]
    cos = (torch.cos(angle) * state["scale"]).float()
    sin = (torch.sin(angle) * state["scale"]).float()
    if case["inverse"]:
        sin = -sin
    for name in ("q", "k"):
        x, out = state[name].float(), state[name + "_out"]
        if case["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
        pair = (a * cos - b * sin, b * cos + a * sin)
        turned = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
        out[..., :r] = turned.to(out.dtype)
        out[..., r:] = state[name][..., r:]
    return dict(q=state["q_out"], k=state["k_out"])


# ---- one pass, by the framework -----------------------------------------------------------

def _own(state):
    from fe2o3_amd import kernels
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        kernels.quantize_mxfp4(state["x"], state["codes"], state["scales"], sync=False)
        kernels.dequantize_mxfp4(state["codes"], state["scales"], state["out"], sync=False)
        return state["out"]
    if kind == "product":
        kernels.gemm_mxfp4_nt(state["a"], state["a_scale"], state["b"], state["b_scale"],
                              state["c"], sync=False)
        return state["c"]
    if kind == "rotary":
        kernels.rotary(state["q"], state["k"], state["positions"], state["freq"],
                       q_out=state["q_out"], k_out=state["k_out"],
                       interleaved=case["interleaved"], inverse=case["inverse"],
                       scale=state["scale"], sync=False)
        return dict(q=state["q_out"], k=state["k_out"])
    held = state["cache"]
    cache = kernels.KvCache(held["k"], held["v"], held["k_scale"], held["v_scale"])
    if kind == "cache":
        kernels.kv_cache_write(cache, state["k"], state["v"], state["slots"], sync=False)
        kernels.kv_cache_read(cache, state["table"], state["starts"], state["k_out"],
                              state["v_out"], sync=False)
        return dict(k=state["k_out"], v=state["v_out"])
    kernels.paged_attention_decode(cache, state["q"], state["table"], state["lengths"],
                                   state["out"], state["lse"], state["scratch"],
                                   max_length=case["max_len"], window=case["window"],
                                   scale=case["head_dim"] ** -0.5, sync=False)
    return dict(out=state["out"], lse=state["lse"])


def run(state):
    if own:
        return _own(state)
    return dict(quantize=_plain_quantize, product=_plain_product, cache=_plain_cache,
                decode=_plain_decode, rotary=_plain_rotary)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        packed = rows * -(-cols // BLOCK) * (BLOCK // 2 + 1)
        return dict(bytes=2 * (rows * cols * (2 if case["dtype"] == "bf16" else 4) + packed),
                    flops=4 * rows * cols)
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        packed = (m + n) * -(-k // BLOCK) * (BLOCK // 2 + 1)
        return dict(bytes=packed + 2 * m * n, flops=2 * m * n * k)
    h, d = case["kv_heads"], case["head_dim"]
    if kind == "rotary":
        heads = case["q_heads"] + h
        return dict(bytes=case["tokens"] * (2 * heads * d * (2 if case["dtype"] == "bf16" else 4)
                                            + 4),
                    flops=3 * case["tokens"] * heads * case["rotary_dim"])
    # one token's K and V as the cache holds them, and as bf16
    cached = 2 * h * (d // 2 + d // BLOCK)
    plain = 2 * h * 2 * d
    if kind == "cache":
        new, all_rows = case["seqs"] * case["new"], case["seqs"] * case["length"]
        return dict(bytes=(new + all_rows) * (plain + cached) + 4 * new,
                    flops=2 * (new + all_rows) * 2 * h * d)
    lengths = _lengths(case)
    keys = [min(n, case["window"]) if case["window"] else n for n in lengths]
    tables = 4 * sum(1 - (-n // case["page_size"]) for n in keys)
    heads = case["seqs"] * case["q_heads"]
    return dict(bytes=sum(keys) * cached + heads * (4 * d + 4) + tables,
                flops=4 * sum(keys) * case["q_heads"] * d)


# ---- the definitions in 64 bits ---------------------------------------------------------------

def _nearest64(x):
    """Each value's nearest on its block's grid of 4 bits, blocks [..., 32] in 64 bits."""
    top = x.abs().amax(-1, keepdim=True)
    # the exponent by a search that has no rounding: frexp's mantissa lies in [0.5, 1)
    exponent = torch.frexp(top)[1].double() - 1
    scale = torch.exp2(torch.where(top > 0, exponent - 2, -127.0).clamp_min(-127.0))
    y = (x / scale).clamp(-6.0, 6.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1.0))) - 1)
    return torch.round(y / step) * step * scale


def _decoded64(packed, scale_bytes):
    """Blocks' values [..., blocks, 32] of packed codes [..., blocks, 16] in 64 bits."""
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).double()
    sign = torch.where(code >= 8, -1.0, 1.0)
    c = code % 8
    magnitude = torch.where(c < 2, c / 2, (1 + (c % 2) / 2) * torch.exp2(torch.floor(c / 2) - 1))
    return sign * magnitude * torch.exp2(scale_bytes.double() - 127)[..., None]


def _matrix64(codes, scales):
    rows, panels = codes.shape[0], scales.shape[0]
    blocks = codes.view(rows, panels, 8, BLOCK // 2)
    return _decoded64(blocks, scales[:, :rows].transpose(0, 1)).reshape(rows, panels * PANEL)


def _row64(state, name, seq, count):
    """The first `count` rows of one sequence, [count, kv_heads, head_dim] in 64 bits."""
    cache, n = state["cache"], state["case"]["page_size"]
    pages = state["table"][seq, :-(-count // n)].long()
    codes = cache[name][pages].unflatten(-1, (-1, BLOCK // 2))
    x = _decoded64(codes, cache[name + "_scale"][pages].transpose(1, 2)).flatten(-2)
    return x.reshape(-1, *x.shape[2:])[:count]


def exact(case, seed):
    kind = case["kind"]
    state = prepare(case, seed)
    if kind == "quantize":
        x = state["x"].double()
        pad = -x.shape[1] % BLOCK
        x = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, BLOCK))
        return _nearest64(x).flatten(-2)[:, :case["cols"]].contiguous()
    if kind == "product":
        a, b = _matrix64(state["a"], state["a_scale"]), _matrix64(state["b"], state["b_scale"])
        return a @ b.T.contiguous()
    if kind == "rotary":
        r, out = case["rotary_dim"], {}
        phase = torch.outer(state["positions"].double(), state["freq"])[:, None]
        turn = torch.polar(torch.full_like(phase, state["scale"]), phase)
        if case["inverse"]:
            turn = turn.conj()
        for name in ("q", "k"):
            x = state[name].double().contiguous()
            part = x[..., :r]
            if case["interleaved"]:
                z = torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * turn
                x[..., :r] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(part[..., :r // 2], part[..., r // 2:]) * turn
                x[..., :r] = torch.cat((z.real, z.imag), -1)
            out[name] = x
        return out
    if kind == "cache":
        out, n, new, length = {}, case["seqs"], case["new"], case["length"]
        for name in ("k", "v"):
            rows = state[name + "_out"].double()
            x = _nearest64(state[name].double().unflatten(-1, (-1, BLOCK))).flatten(-2)
            for seq in range(n):
                rows[seq * length:(seq + 1) * length] = _row64(state, name, seq, length)
                rows[(seq + 1) * length - new:(seq + 1) * length] = x[seq * new:(seq + 1) * new]
            out[name] = rows
        return out
    lengths = state["lengths"].tolist()
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
