"""Serving operators around the attention of a decoder block, measured: rotary
positions, keys and values appended to a paged cache held in 4 bits (rotated
on the way), and attention over that cache.  `run` computes each in its plain
form (elementary torch operations) or, with `own`, through the library.

The cache is one device buffer of pages (uint8).  A page holds `page` rows of
every KV head; per head a record of K codes, K scales, V codes, V scales:

    [page][head_len / 2] bytes, [page][head_len / 32] fp16, then V the same

A row is cut into blocks of 32 values, value = scale * (code - 8).  Byte k of
a block (k = 0..15) has value k's code in its low nibble and value k + 16's in
its high nibble.  Byte k of block b stands at byte (k / 4) * 4 nb + 4 b + k % 4
of a K row and at byte (k / 2) * 2 nb + 2 b + k % 2 of a V row (nb blocks a
row).  The scale is -m / 8 in fp16 (m the block's largest value or, where its
magnitude is larger, its smallest), held to fp16's finite range; the code is
rint(value * (1 / scale)) + 8, in 0..15.  A block with an infinity or a NaN
has a NaN scale.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
DEVICE = "cuda"


# ------------------------------------------------------------------ the cases
def listed():
    # Head shapes: 16/16 x 128 and theta 1e4 (the OLMoE configuration), 32/8 x
    # 128 and theta 1e6 (Mixtral), and generic ones.  Lengths: the 512 and 2048
    # token prompts and the 8192-token context of those configurations,
    # batches of them, and long contexts.
    return [
        # one token of one sequence, every call of a decode step: latency
        dict(name="rope-one-token", kind="rope", type="f32", tokens=1, heads=16, kv_heads=16, head_len=128,
             rot=128, layout="pairs", theta=1e4, scaling="none", max_pos=8192),
        # a 2048-token prompt, Mixtral's heads, out of the fused QKV product
        dict(name="rope-prompt", kind="rope", type="f32", tokens=2048, heads=32, kv_heads=8, head_len=128,
             rot=128, layout="pairs", theta=1e6, scaling="none", max_pos=32768),
        # a packed batch of far positions, half of each head rotated, frequencies scaled by parts
        dict(name="rope-long-context", kind="rope", type="bf16", tokens=16383, heads=32, kv_heads=4, head_len=128,
             rot=64, layout="halves", theta=1e4, scaling="parts", max_pos=1 << 20),
        # the new rows of a decode batch: one token for each of 64 sequences
        dict(name="append-decode", kind="append", type="bf16", seqs=64, q=1, ragged=False, kv_min=1, kv_max=8192,
             heads=32, kv_heads=8, head_len=128, page=64, rot=128, layout="pairs", theta=1e6, scaling="none",
             max_pos=32768, pad=0),
        # the reference model's 512-token prompt in fp32, as its own engine has it
        dict(name="append-prompt", kind="append", type="f32", seqs=1, q=512, ragged=False, kv_min=512, kv_max=512,
             heads=16, kv_heads=16, head_len=128, page=32, rot=128, layout="pairs", theta=1e4, scaling="none",
             max_pos=8192, pad=0),
        # ragged chunks of several prompts in one batch, padded at its end
        dict(name="append-chunks", kind="append", type="f16", seqs=7, q=4099, ragged=True, kv_min=4099, kv_max=20011,
             heads=28, kv_heads=4, head_len=64, page=16, rot=32, layout="halves", theta=5e5, scaling="bands",
             max_pos=131072, pad=117),
        # decode of one OLMoE sequence: 2049 rows in the cache
        dict(name="attn-one-sequence", kind="attn", type="f32", seqs=1, q=1, ragged=False, kv_min=2049, kv_max=2049,
             heads=16, kv_heads=16, head_len=128, page=64, causal=True, window=0, pad=0),
        # a decode batch with Mixtral's heads, sequences of every length
        dict(name="attn-decode-batch", kind="attn", type="bf16", seqs=64, q=1, ragged=False, kv_min=1, kv_max=8192,
             heads=32, kv_heads=8, head_len=128, page=64, causal=True, window=0, pad=3),
        # decode over long contexts: the cache read is all the time
        dict(name="attn-decode-long", kind="attn", type="bf16", seqs=4, q=1, ragged=False, kv_min=98304, kv_max=131072,
             heads=32, kv_heads=8, head_len=128, page=128, causal=True, window=0, pad=0),
        # several drafted tokens of each sequence verified at once, in a sliding window
        dict(name="attn-drafted-window", kind="attn", type="f16", seqs=17, q=6, ragged=True, kv_min=5, kv_max=9973,
             heads=32, kv_heads=4, head_len=64, page=32, causal=True, window=4096, pad=0),
        # a 2048-token prompt against itself, Mixtral's heads
        dict(name="attn-prompt", kind="attn", type="bf16", seqs=1, q=2048, ragged=False, kv_min=2048, kv_max=2048,
             heads=32, kv_heads=8, head_len=128, page=64, causal=True, window=0, pad=0),
        # a decode step's attention as an engine runs it: rotate, append, attend (and read the new rows back)
        dict(name="step-decode-batch", kind="step", type="bf16", seqs=32, q=1, ragged=False, kv_min=512, kv_max=4096,
             heads=32, kv_heads=8, head_len=128, page=64, rot=128, layout="pairs", theta=1e6, scaling="none",
             max_pos=32768, causal=True, window=0, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "append", "append", "attn", "attn", "attn", "step"])
    head_len = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8])
    while heads * head_len > 8192:
        heads -= kv_heads
    c = dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), heads=heads, kv_heads=kv_heads, head_len=head_len)
    if kind != "attn":
        c |= dict(rot=rng.choice([head_len, head_len, head_len // 2, head_len - 6]), layout=rng.choice(["pairs", "halves"]),
                  theta=rng.choice([1e4, 5e5, 1e6]), scaling=rng.choice(["none", "linear", "parts", "bands"]),
                  max_pos=rng.choice([32768, 131072, 1 << 20]))
    if kind == "rope":
        return c | dict(tokens=min(_log(rng, 1, 16384), max(1, (1 << 26) // ((heads + kv_heads) * head_len))))
    c |= dict(page=rng.choice([16, 32, 64, 128]), ragged=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 29]))
    if kind != "append":
        c |= dict(causal=kind == "step" or rng.random() < 0.8, window=0)
    if kind == "step":
        c["type"] = rng.choice(["f16", "bf16"])
    rows = (1 << 28) // (kv_heads * head_len)  # of the cache, over all sequences
    if kind != "append" and rng.random() < 0.6:  # decode, drafted tokens
        seqs, q = _log(rng, 1, 96), _log(rng, 1, 8)
        kv_max = _log(rng, q, 131072)
    else:  # prompts and chunks of them
        seqs, q = _log(rng, 1, 9), _log(rng, 1, 2000)
        kv_max = _log(rng, q, min(32000, q + 9000))
    seqs = max(1, min(seqs, rows // kv_max))
    while kind != "append" and seqs * q * kv_max * heads * head_len > 2 ** 33 and q > 1:
        q = max(1, q // 2)
    while kind == "append" and seqs * q * heads * head_len > 2 ** 25 and q > 1:
        q = max(1, q // 2)
    c |= dict(seqs=seqs, q=q, kv_max=kv_max, kv_min=_log(rng, 1, kv_max))
    if kind == "attn" and c["causal"] and rng.random() < 0.3:
        c["window"] = _log(rng, 1, kv_max)
    return c


def _lengths(c):
    """Rows of each sequence in the batch and in the cache (the batch's among them): of the case alone."""
    n = c["seqs"]
    order = sorted(range(n), key=lambda b: b * 2654435761 % 2 ** 32)
    q = [max(1, c["q"] * (b + 1) // n) if c["ragged"] else c["q"] for b in range(n)]
    kv = [round(c["kv_max"] * (c["kv_min"] / c["kv_max"]) ** (order[b] / max(1, n - 1))) for b in range(n)]
    return q, [max(k, s) for k, s in zip(kv, q)]


def _pairs(c):
    """(query, row) pairs that a case attends, and the cache rows that it has to read."""
    pairs = rows = 0
    for n, kv in zip(*_lengths(c)):
        if not c["causal"]:
            pairs, rows = pairs + n * kv, rows + kv
            continue
        first = kv - n  # query i sees rows 0 .. first + i
        if c["window"]:
            w = c["window"]
            low = max(0, min(n, w - first - 1))  # queries whose window reaches before row 0
            pairs += low * (first + 1) + low * (low - 1) // 2 + (n - low) * w
            rows += min(kv, n + w - 1)
        else:
            pairs += n * (first + 1) + n * (n - 1) // 2
            rows += kv
    return pairs, rows


def work(c):
    es, H, KVH, D = BYTES[c["type"]], c["heads"], c["kv_heads"], c["head_len"]
    if c["kind"] == "rope":
        n = c["tokens"] * (H + KVH)
        return {"bytes": 2 * n * D * es + 4 * c["tokens"], "flops": 3 * n * c["rot"]}
    q, kv = _lengths(c)
    tokens, held = sum(q), 2 * KVH * (D // 2 + D // 16)  # bytes of one row's K and V in the cache
    got = {"bytes": 0, "flops": 0}
    if c["kind"] != "attn":  # q, k, v read; q and the rows written
        got["bytes"] += tokens * ((H + 2 * KVH) * D * es + held)
        got["flops"] += tokens * (3 * (H + KVH) * c["rot"] + 8 * KVH * D)
        # rotated q written; the new rows read back as values
        got["bytes"] += tokens * (H * D * es + held + 2 * KVH * D * es)
    if c["kind"] != "append":
        pairs, rows = _pairs(c)
        got["bytes"] += rows * held + tokens * (2 * H * D * es + 4 * H)
        got["flops"] += 4 * pairs * H * D
    return got


# ------------------------------------------------------------------ the inputs
def _views(pool, c):
    """K codes, K scales, V codes, V scales of the pages: [page, head, row, ...] views."""
    P, D = c["page"], c["head_len"]
    kc, sc = P * D // 2, P * D // 16
    at = pool.view(-1, c["kv_heads"], 2, kc + sc)
    codes = [at[:, :, i, :kc].unflatten(-1, (P, D // 2)) for i in (0, 1)]
    scales = [at[:, :, i, kc:].view(torch.float16).unflatten(-1, (P, D // 32)) for i in (0, 1)]
    return codes[0], scales[0], codes[1], scales[1]


def _quantize(x):
    """fp32 rows [..., head_len] as codes and scales."""
    b = x.unflatten(-1, (-1, 32))
    hi, lo = b.amax(-1), b.amin(-1)
    scale = (torch.where(hi >= -lo, hi, lo) * -0.125).clamp(-65504.0, 65504.0).half()
    scale = torch.where(b.isfinite().all(-1), scale, torch.nan)
    inv = torch.where(scale == 0, 0.0, 1.0 / scale.float())
    codes = (torch.round(b * inv[..., None]) + 8).clamp(0, 15)
    return torch.where(scale.isnan()[..., None], 8.0, codes).to(torch.uint8), scale


def _pack(codes, width):
    """Codes [..., nb, 32] as the bytes of a row: `width` bytes of each block side by side (4: K, 2: V)."""
    by = codes[..., :16] | (codes[..., 16:] << 4)
    return by.unflatten(-1, (16 // width, width)).transpose(-3, -2).flatten(-3)


def _values(by, scale, width):
    """The fp32 values that the bytes of rows stand for."""
    nb = scale.shape[-1]
    by = by.unflatten(-1, (16 // width, nb, width)).transpose(-3, -2).flatten(-2)
    codes = torch.cat([by & 15, by >> 4], -1)
    return ((codes.float() - 8) * scale.float()[..., None]).flatten(-2)


def _fill(pool, c, g):
    """Pages of keys and values as a model has them: a few channels of the keys stand out."""
    kc, ks, vc, vs = _views(pool, c)
    KVH, P, D = c["kv_heads"], c["page"], c["head_len"]
    stand_out = 1 + 3 * (torch.rand(KVH, 1, D, generator=g, device=DEVICE) < 0.05)
    step = max(1, (1 << 24) // (KVH * P * D))
    for i in range(0, pool.shape[0], step):
        n = min(step, pool.shape[0] - i)
        for codes, scales, width, by in ((kc, ks, 4, stand_out), (vc, vs, 2, 1.0)):
            q, s = _quantize(torch.randn(n, KVH, P, D, generator=g, device=DEVICE) * by)
            codes[i:i + n], scales[i:i + n] = _pack(q, width), s


def _frequencies(c):
    """Radians a position of each rotated pair, in 64 bits, and the factor on cosine and sine."""
    rot, theta = c["rot"], c["theta"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = theta ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        return f / 4.0, 1.0
    if c["scaling"] == "parts":  # fast pairs stay, slow ones are divided, a ramp over the pairs between
        pair = lambda turns: rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / 16.0 * ramp + f * (1 - ramp), 0.1 * math.log(16.0) + 1.0
    if c["scaling"] == "bands":  # by the turns that a pair makes over the original context
        turns = 8192 * f / (2 * math.pi)
        s = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - s) * f / 8.0 + s * f, 1.0
    return f, 1.0


def _rope_arguments(c, m):
    """moe_rope_desc's fields for _frequencies(c)."""
    a = dict(rot=c["rot"], theta=c["theta"], max_position=c["max_pos"],
             layout=m.ROPE_PAIRS if c["layout"] == "pairs" else m.ROPE_HALVES)
    if c["scaling"] == "linear":
        a |= dict(scaling=m.ROPE_LINEAR, factor=4.0)
    if c["scaling"] == "parts":
        a |= dict(scaling=m.ROPE_PARTS, factor=16.0, orig_context=8192, beta_fast=32.0, beta_slow=1.0)
    if c["scaling"] == "bands":
        a |= dict(scaling=m.ROPE_BANDS, factor=8.0, orig_context=8192, low_freq=1.0, high_freq=4.0)
    return a


def _library():
    """The framework's package (its folder's name is no identifier)."""
    if "moe_b200" not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.c_b200", "__init__.py")
        spec = importlib.util.spec_from_file_location("moe_b200", at)
        sys.modules["moe_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["moe_b200"])
    m = sys.modules["moe_b200"]
    m.init(0)
    return m


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"case": c}
    if c["kind"] != "attn":
        f, s["factor"] = _frequencies(c)
        s["freq"] = f.to(DEVICE)
    H, KVH, D, dt = c["heads"], c["kv_heads"], c["head_len"], TYPES[c["type"]]
    if c["kind"] == "rope":
        n = tokens = c["tokens"]
        s["pos"] = torch.randint(0, c["max_pos"], (n,), generator=g, device=DEVICE, dtype=torch.int32)
    else:
        q, kv = _lengths(c)
        n = sum(q)
        tokens = n + c["pad"]
        need = [-(-k // c["page"]) for k in kv]
        wide = max(need) + 2
        pages = sum(need) + 3
        perm = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        table = torch.full((len(kv), wide), -1, device=DEVICE, dtype=torch.int32)
        ends = torch.cumsum(torch.tensor(need), 0)
        mask = torch.arange(wide)[None] < torch.tensor(need)[:, None]
        table[mask.to(DEVICE)] = perm[:int(ends[-1])]
        rec = KVH * 2 * c["page"] * (D // 2 + D // 16)
        s["pool"] = torch.empty(pages, rec, device=DEVICE, dtype=torch.uint8)
        _fill(s["pool"], c, g)
        start = torch.cumsum(torch.tensor([0] + q), 0)
        s |= {"table": table, "q_start": start.to(DEVICE, torch.int32), "kv_len": torch.tensor(kv, device=DEVICE, dtype=torch.int32),
              "rows": n, "max_q": max(q), "max_kv": max(kv)}
    # q, k, v side by side, as one product leaves them
    qkv = torch.randn(tokens, (H + 2 * KVH) * D, generator=g, device=DEVICE)
    qkv[:, H * D:(H + KVH) * D] *= 1 + 2 * (torch.rand(KVH * D, generator=g, device=DEVICE) < 0.05)
    s["qkv"] = qkv.mul_(1.5).to(dt)
    del qkv
    new = lambda *shape, d=dt: torch.zeros(shape, device=DEVICE, dtype=d)  # noqa: E731
    if c["kind"] != "attn":
        s["q_out"] = new(tokens, H, D)
    if c["kind"] == "rope":
        s["k_out"] = new(tokens, KVH, D)
    if c["kind"] in ("append", "step"):
        s["k_rows"], s["v_rows"] = new(tokens, KVH, D), new(tokens, KVH, D)
    if c["kind"] in ("attn", "step"):
        s["out"], s["lse"] = new(tokens, H, D), new(tokens, H, d=torch.float32)
    if own:
        m = _library()
        s["m"] = m
        if c["kind"] != "attn":
            s["rope"] = m.Rope(**_rope_arguments(c, m))
        if c["kind"] != "rope":
            s["cache"] = m.KVCache(pages, c["page"], KVH, D, m.Q4_0, pages=s["pool"].data_ptr())
            s["batch"] = m.KVBatch(len(kv), tokens, s["max_q"], s["max_kv"], s["q_start"].data_ptr(),
                                   s["kv_len"].data_ptr(), s["table"].data_ptr(), wide)
            if c["kind"] != "append":
                s["work"] = torch.empty(max(16, s["cache"].workspace_bytes(s["batch"], H)), device=DEVICE, dtype=torch.uint8)
    return s


def _heads(s):
    """q, k, v of the fused rows, [token, head, head_len]."""
    c = s["case"]
    H, KVH, D = c["heads"], c["kv_heads"], c["head_len"]
    x = s["qkv"].unflatten(-1, (H + 2 * KVH, D))
    return x[:, :H], x[:, H:H + KVH], x[:, H + KVH:]


# ------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    m, c = s["m"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream or 1  # 1: CUDA's legacy default stream
    kinds = {torch.float32: m.F32, torch.float16: m.F16, torch.bfloat16: m.BF16}
    rows = lambda x: m.Rows(x.data_ptr(), kinds[x.dtype], x.shape[1], x.stride(0), x.stride(1))  # noqa: E731
    q, k, v = (rows(x) for x in _heads(s))
    scale = c["head_len"] ** -0.5
    if c["kind"] == "rope":
        s["rope"].forward(c["tokens"], c["head_len"], s["pos"].data_ptr(), q, rows(s["q_out"]), k, rows(s["k_out"]), stream=stream)
        return {"q": s["q_out"], "k": s["k_out"]}
    if c["kind"] == "attn":
        s["cache"].attention(s["batch"], q, rows(s["out"]), scale, causal=c["causal"], window=c["window"],
                             lse=s["lse"].data_ptr(), workspace=s["work"].data_ptr(), workspace_bytes=s["work"].numel(), stream=stream)
        return {"out": s["out"], "lse": s["lse"]}
    s["cache"].append(s["batch"], k, v, rope=s["rope"], q=q, q_out=rows(s["q_out"]), stream=stream)
    s["cache"].gather(s["batch"], rows(s["k_rows"]), rows(s["v_rows"]), stream=stream)
    got = {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}
    if c["kind"] == "step":
        s["cache"].attention(s["batch"], rows(s["q_out"]), rows(s["out"]), scale, causal=c["causal"], window=c["window"],
                             lse=s["lse"].data_ptr(), workspace=s["work"].data_ptr(), workspace_bytes=s["work"].numel(), stream=stream)
        got |= {"out": s["out"], "lse": s["lse"]}
    return got


def _turn(x, pos, s):
    """fp32 rows with their first `rot` values rotated."""
    c = s["case"]
    angle = pos.double()[:, None] * s["freq"]
    cos, sin = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]
    r = x[..., :c["rot"]]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["layout"] == "pairs" else r.chunk(2, -1)
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if c["layout"] == "pairs" else torch.cat(y, -1)
    return torch.cat([y, x[..., c["rot"]:]], -1)


def _places(s):
    """Sequence, row in its cache, page and row of the page of each of the batch's tokens."""
    t = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), t, right=True)
    row = s["kv_len"][seq] - s["q_start"][seq + 1] + t
    P = s["case"]["page"]
    return seq, row, s["table"][seq, row // P].long(), row % P


def _run_plain(s):
    c = s["case"]
    dt = TYPES[c["type"]]
    q, k, v = _heads(s)
    if c["kind"] == "rope":
        s["q_out"].copy_(_turn(q.float(), s["pos"], s))
        s["k_out"].copy_(_turn(k.float(), s["pos"], s))
        return {"q": s["q_out"], "k": s["k_out"]}
    if c["kind"] == "attn":
        _attend(s, q)
        return {"out": s["out"], "lse": s["lse"]}
    n = s["rows"]
    _, row, page, at = _places(s)
    s["q_out"][:n] = _turn(q[:n].float(), row, s).to(dt)
    kc, ks, vc, vs = _views(s["pool"], c)
    for x, codes, scales, width in ((_turn(k[:n].float(), row, s), kc, ks, 4), (v[:n].float(), vc, vs, 2)):
        by, scale = _quantize(x)
        codes[page, :, at], scales[page, :, at] = _pack(by, width), scale
    s["k_rows"][:n] = _values(kc[page, :, at], ks[page, :, at], 4).to(dt)
    s["v_rows"][:n] = _values(vc[page, :, at], vs[page, :, at], 2).to(dt)
    got = {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}
    if c["kind"] == "step":
        _attend(s, s["q_out"])
        got |= {"out": s["out"], "lse": s["lse"]}
    return got


def _attend(s, q):
    c = s["case"]
    H, KVH, D, n, B = c["heads"], c["kv_heads"], c["head_len"], s["rows"], c["seqs"]
    G, S, Q = H // KVH, s["max_kv"], s["max_q"]
    seq, row, _, _ = _places(s)
    i = torch.arange(n, device=DEVICE) - s["q_start"][seq]
    x = torch.zeros(B, Q, KVH, G, D, device=DEVICE)
    x[seq, i] = q[:n].float().unflatten(1, (KVH, G))
    x = x.permute(0, 2, 1, 3, 4).reshape(B, KVH, Q * G, D)
    j = torch.arange(S, device=DEVICE)
    page, at = s["table"][:, j // c["page"]].clamp(min=0).long(), (j % c["page"]).expand(B, S)
    kc, ks, vc, vs = _views(s["pool"], c)
    k = _values(kc[page, :, at], ks[page, :, at], 4).transpose(1, 2)  # [B, KVH, S, D]
    score = (x @ k.transpose(-1, -2)).mul_(D ** -0.5).view(B, KVH, Q, G, S)
    del k
    at_row = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1]))[:, None] + torch.arange(Q, device=DEVICE)  # [B, Q]
    seen = (j < s["kv_len"][:, None])[:, None].expand(B, Q, S)
    if c["causal"]:
        seen = seen & (j <= at_row[..., None])
    if c["window"]:
        seen = seen & (j > at_row[..., None] - c["window"])
    score.masked_fill_(~seen[:, None, :, None], -torch.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -torch.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = _values(vc[page, :, at], vs[page, :, at], 2).transpose(1, 2)
    out = (p.view(B, KVH, Q * G, S) @ v).view(B, KVH, Q, G, D)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log()).squeeze(-1)  # -inf where nothing is seen
    s["out"][:n] = out.permute(0, 2, 1, 3, 4).reshape(B, Q, H, D)[seq, i].to(s["out"].dtype)
    s["lse"][:n] = lse.permute(0, 2, 1, 3).reshape(B, Q, H)[seq, i]


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """From the definitions, sequence after sequence, in 64 bits.  The values
    that 4 bits stand for have none: which code a value takes is a decision on
    its fp32 form."""
    c = case
    s = prepare(c, seed)
    H, KVH, D = c["heads"], c["kv_heads"], c["head_len"]
    x = s["qkv"].double().view(-1, H + 2 * KVH, D)
    if c["kind"] == "rope":
        q, k = _rotated64(x[:, :H], s["pos"], c), _rotated64(x[:, H:H + KVH], s["pos"], c)
        return {"q": q, "k": k}
    lens, kv = _lengths(c)
    turned = torch.zeros_like(x[:, :H])
    out, lse = torch.zeros_like(turned), torch.zeros_like(turned[..., 0])
    t = 0
    for b, (n, m) in enumerate(zip(lens, kv)):
        rows = torch.arange(m - n, m, device=DEVICE)
        q = x[t:t + n, :H]
        if c["kind"] != "attn":
            q = turned[t:t + n] = _rotated64(q, rows, c)
        if c["kind"] != "append":
            keys, values = (_held64(s["pool"], s["table"][b], m, c, i) for i in (0, 1))
            if c["kind"] == "step":
                keys[m - n:] = _as_held64(_rotated64(x[t:t + n, H:H + KVH], rows, c))
                values[m - n:] = _as_held64(x[t:t + n, H + KVH:])
                q = q.to(TYPES[c["type"]]).double()
            o, l = _attended64(q, keys, values, rows, c)
            out[t:t + n], lse[t:t + n] = o, l
        t += n
    got = {"q": turned, "k": None, "v": None} if c["kind"] != "attn" else {}
    return got | ({"out": out, "lse": lse} if c["kind"] != "append" else {})


def _rotated64(x, pos, c):
    f, factor = _frequencies(c)
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device=DEVICE).expand(pos.numel(), f.numel()),
                       torch.outer(pos.double(), f.to(DEVICE)))
    rot = c["rot"]
    y = x.clone()
    first = torch.arange(rot // 2, device=DEVICE) * (2 if c["layout"] == "pairs" else 1)
    second = first + (1 if c["layout"] == "pairs" else rot // 2)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _held64(pool, table, n, c, which):
    """n rows of a sequence's keys (0) or values (1), [row, head, head_len], value by value from the layout."""
    P, D, KVH = c["page"], c["head_len"], c["kv_heads"]
    nb, width = D // 32, (4, 2)[which]
    pages = pool[table[:-(-n // P)].long()].view(-1, KVH, 2, P * (D // 2 + D // 16))[:, :, which]
    d = torch.arange(D, device=DEVICE)
    k = d % 16
    place = (k // width) * width * nb + width * (d // 32) + k % width
    row = torch.arange(P, device=DEVICE)[:, None] * (D // 2)
    by = pages[..., (row + place).flatten()].view(-1, KVH, P, D)
    code = torch.where(d % 32 < 16, by % 16, by // 16)
    scale = pages[..., P * D // 2:].contiguous().view(torch.float16).view(-1, KVH, P, nb).double().repeat_interleave(32, -1)
    return ((code.double() - 8) * scale).transpose(1, 2).reshape(-1, KVH, D)[:n]


def _as_held64(x):
    """Values [.., head_len] as the 4 bits hold them."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    i = b.abs().argmax(-1, keepdim=True)
    step = (b.gather(-1, i) / -8).half().double()
    code = torch.round(b / torch.where(step == 0, 1.0, step)).clamp(-8, 7)
    return (code * step).reshape(x.shape)


def _attended64(q, keys, values, rows, c):
    H, KVH, D = c["heads"], c["kv_heads"], c["head_len"]
    j = torch.arange(keys.shape[0], device=DEVICE)
    hidden = torch.zeros(rows.numel(), keys.shape[0], dtype=torch.bool, device=DEVICE)
    if c["causal"]:
        hidden |= j[None] > rows[:, None]
    if c["window"]:
        hidden |= j[None] <= rows[:, None] - c["window"]
    out, lse = torch.empty_like(q), torch.empty_like(q[..., 0])
    for h in range(H):
        kh = h // (H // KVH)
        score = torch.einsum("td,sd->ts", q[:, h], keys[:, kh]) / math.sqrt(D)
        score[hidden] = -math.inf
        lse[:, h] = torch.logsumexp(score, -1)
        weight = torch.exp(score - lse[:, h, None])
        out[:, h] = torch.einsum("ts,sd->td", weight, values[:, kh])
    return out, lse
