"""Attention over the 4-bit cache where an item has many key tiles (rings that turn, pages
fetched again every 32 tiles, runs at their longest), and the weighted sums over long
rows against 64 bits by their norm."""
import numpy as np
import pytest
import torch

import kv_ref as ref
from kv_ref import TYPES, rows
from test_gpu_kv import LEGACY, Case, cuda_i32, f64, m, rand  # noqa: F401

pytestmark = pytest.mark.gpu


def check_tokens(c, q, out, lse, tokens, window=0, scale=None):
    """rows of some tokens of a causal call against 64 bits (token by token: its keys cut
    behind it)"""
    x, o, l = f64(q), f64(out), f64(lse)
    scale = scale or c.D ** -0.5
    for t in tokens:
        b = int(np.searchsorted(c.start, t, side="right")) - 1
        n = c.kv_len[b] - (c.start[b + 1] - t) + 1
        k, v = c.k[b][:n], c.v[b][:n]
        want, wl, size = ref.attention(x[t:t + 1], k, v, scale, True, window)
        tol, tol_l = ref.attention_bounds(q.dtype, size, np.abs(v).max(), n, want, wl)
        err = np.abs(o[t:t + 1] - want)
        assert (err <= tol).all(), f"token {t}: {(err / tol).max():.3g} of its bound"
        assert (np.abs(l[t:t + 1] - wl) <= tol_l).all(), f"token {t}: lse"


def some(rng, start, n=10):
    """the first and last tokens and some between"""
    end = int(start[-1])
    return sorted({0, 1, end - 1, *(int(x) - 1 for x in start[1:]), *(int(x) for x in rng.integers(0, end, n))})


@pytest.mark.parametrize("dtype,D,KVH,G,P,q_len,kv_len,window", [
    ("bf16", 128, 8, 4, 64, [512], [2048], 0),      # items of 256 query rows, runs of some 50 tiles
    ("f16", 64, 8, 4, 16, [512], [2077], 0),        # the same from pages of half a tile
    ("bf16", 128, 8, 4, 32, [300, 512], [300, 2500], 1500),
    ("f32", 128, 8, 8, 128, [600], [2100], 0),      # an item a warp: whole sequences of 66 tiles
    ("f32", 256, 4, 8, 16, [600], [2100], 0),
    ("bf16", 256, 4, 16, 64, [600], [2100], 1700)])
def test_attention_long_items(m, dtype, D, KVH, G, P, q_len, kv_len, window):
    """prompts over long rows: every buffer of a kernel's rings comes round many times, the
    pages' list is fetched anew, V's scales grow on the way (sums are rescaled)"""
    c = Case(m, q_len, kv_len, KVH, D, P, pad=1, seed=D + P)
    q = rand(11, c.T, KVH * G, D, dtype=TYPES[dtype], sd=1.2).cuda()
    tokens = some(np.random.default_rng(P), c.start)
    out, lse = c.attend(q, window=window)
    assert c.cache.status() == 0
    check_tokens(c, q, out, lse, tokens, window)
    for b, n in enumerate(kv_len):
        at = np.arange(n)
        f = np.float32(2.0) ** np.minimum(at // 150 - 9, 5)
        pages, row = c.table[b, at // P], at % P
        sc = c.pool.scales()[pages, :, 1, row].view(np.float16).astype(np.float32)
        c.pool.scales()[pages, :, 1, row] = (sc * f[:, None, None]).astype(np.float16).view(np.uint16)
        c.v[b] = c.pool.sequence(c.table[b], n, 1)
    c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
    out, lse = c.attend(q, window=window)
    assert c.cache.status() == 0
    check_tokens(c, q, out, lse, tokens, window)
    again, lse2 = c.attend(q, window=window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype,D,G", [("f32", 64, 2), ("bf16", 64, 4), ("f16", 128, 4), ("bf16", 256, 3)])
def test_attention_long_decode_items(m, dtype, D, G):
    """decode steps of 128 sequences that share their pages, in runs of more than 32 tiles"""
    KVH, P, n = 8, 32, 2100
    c = Case(m, [1], [n], KVH, D, P, seed=G)
    B = 128
    lens = [n - 7 * b for b in range(B)]
    c.q_len, c.kv_len, c.k, c.v = [1] * B, lens, c.k * B, c.v * B
    c.k, c.v = ([x[:i] for x, i in zip(y, lens)] for y in (c.k, c.v))
    c.table = np.repeat(c.table, B, 0)
    c.start, c.T = np.arange(B + 1, dtype=np.int32), B
    c.dev = [torch.tensor(x, device="cuda") for x in (c.start, np.array(lens, np.int32), c.table)]
    c.batch = m.KVBatch(B, B, 1, n, *[x.data_ptr() for x in c.dev], c.table.shape[1])
    q = rand(12, B, KVH * G, D, dtype=TYPES[dtype], sd=1.2).cuda()
    out, lse = c.attend(q)
    assert c.cache.status() == 0
    check_tokens(c, q, out, lse, range(0, B, 9))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,KVH,G,P,n", [(128, 4, 1, 64, 1), (64, 1, 7, 16, 1), (256, 1, 8, 32, 1), (128, 2, 4, 64, 64),
                                         (64, 1, 8, 32, 33)])
def test_attention_error_of_many_rows(m, dtype, D, KVH, G, P, n):
    """Many keys of equal weight: results are 1 / sqrt(rows) of V.  A weight and its product with
    V's scale (or the weight, and V's value) are rounded to fp16, 2^-11 of their size each with
    signs of their own, so the sums keep the share: sqrt(2) 2^-11 of the results' norm.  Codes
    as subnormals, 2^-16 of a product a sum of 16 rows at most, all of one sign: sqrt(rows) / 16
    * 2^-16 = 2^-14.5 for 2049.  The results' rounding: half of eps.  Scores: 2^-19 of the
    weights.  The rest is below 2^-18."""
    c = Case(m, [n], [2049], KVH, D, P, pad=0)
    q = rand(9, n, KVH * G, D, sd=0.5, dtype=TYPES[dtype]).cuda()
    out, _ = c.attend(q, causal=False)
    k, v = (torch.tensor(x[0], dtype=torch.float64, device="cuda").repeat_interleave(G, 1) for x in (c.k, c.v))
    p = torch.einsum("thd,shd->hts", q.double(), k).mul_(D ** -0.5).softmax(-1)
    want = torch.einsum("hts,shd->thd", p, v)
    err = ((out.double() - want).norm() / want.norm()).item()
    assert err <= 2.0 ** -10.5 + 2.0 ** -14.5 + 2.0 ** -17 + torch.finfo(q.dtype).eps / 2, err


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("top", [65536.0, -65536.0, 65504.0, 70000.0, 524032.0, 1e9])
def test_attention_large_keys(m, top, dtype):
    """keys whose scale is 2^13 and more, with the code that stands for -8 of it"""
    D, KVH, G, n = 128, 1, 4, 70
    c = Case(m, [n], [n], KVH, D, 32, pad=0)
    x = np.random.default_rng(4).standard_normal((n, KVH, D)).astype(np.float32) * (abs(top) / 8)
    x = np.clip(x, -abs(top), abs(top))
    x[::3, :, ::32] = top
    for r in range(n):
        c.pool.put(c.table[0, r // 32], r % 32, 0, x[r])
    c.k[0] = c.pool.sequence(c.table[0], n, 0)
    c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
    q = rand(5, n, KVH * G, D, dtype=TYPES[dtype]).cuda()
    scale = 2.0 / min(abs(top), 524032.0)
    out, lse = c.attend(q, scale=scale)
    assert c.cache.status() == 0
    c.check(q, out, lse, scale=scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,P", [(128, 32), (64, 16), (128, 128)])
def test_attention_small_key_scales(m, D, P, dtype):
    """Key scales of 2^-14 .. 2^-11 in prompts.  What a row that a query does not see holds
    (behind the sequence's end; or behind the query, where others see it) changes no bit of its
    result: zeros, NaN, fp16's largest scale."""
    KVH, G, n, kv = 2, 4, 83, 83
    c = Case(m, [n], [kv], KVH, D, P, pad=0, extra=0, spare=0)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((kv, KVH, D)).astype(np.float32) * 2.0 ** -11
    x *= 2.0 ** rng.integers(-1, 2, (kv, KVH, 1))
    for r in range(kv):
        c.pool.put(c.table[0, r // P], r % P, 0, x[r])
    c.k[0] = c.pool.sequence(c.table[0], kv, 0)
    q = rand(5, n, KVH * G, D, dtype=TYPES[dtype]).cuda()
    scale = D ** -0.5 * 2.0 ** 11
    clean = c.pool.data.copy()
    got = []
    for bits in (0, 0x7fff, 0x7bff, 0x7c00):
        c.pool.data[...] = clean
        for r in range(kv, -(-kv // P) * P):
            c.pool.scales()[c.table[0, r // P], :, :, r % P] = bits
        c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
        out, lse = c.attend(q, scale=scale)
        assert c.cache.status() == 0
        c.check(q, out, lse, scale=scale)
        got.append((out, lse))
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])
    for bits in (0x7fff, 0x7bff, 0x7000):
        c.pool.data[...] = clean
        c.pool.scales()[c.table[0, 70 // P], :, 0, 70 % P] = bits
        c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
        out, lse = c.attend(q, scale=scale)
        assert torch.equal(out[:70], got[0][0][:70]) and torch.equal(lse[:70], got[0][1][:70])
        assert c.cache.status() == 0


@pytest.mark.parametrize("dtype,q_len,kv,B", [("f32", 1, 20, 100), ("bf16", 2, 32, 70), ("f16", 64, 32, 40)])
def test_attention_reports_every_sequence(m, dtype, q_len, kv, B):
    """lengths out of range in a sequence behind the first 32, of a call whose items are whole
    sequences: reported, and the others are right"""
    D, KVH, G = 64, 1, 4
    c = Case(m, [q_len] * B, [kv] * B, KVH, D, 16, pad=2)
    q = rand(5, c.T, G, D, dtype=TYPES[dtype]).cuda()
    for b, bad in ((B - 1, kv + 1), (33, -1)):
        c.dev[1].fill_(kv)
        c.dev[1][b] = bad
        out, lse = c.attend(q)
        assert c.cache.status() == -1 and c.cache.status() == 0
        c.check(q, out, lse, seqs=[0, 1, 31, 32, B - 2])
        a, z = c.start[b], c.start[b + 1]
        assert (out[a:z] == 5.0).all() and (lse[a:z] == 6.0).all()
    c.dev[1].fill_(kv)
    c.dev[0][B - 1] -= 1   # a query more for the last sequence than max_q
    c.attend(q)
    assert c.cache.status() == -1 and c.cache.status() == 0


def long_rows(m, n, D, KVH, P, k, v):
    """a cache of one sequence of n rows, its page table, and the rows that it holds"""
    cache = m.KVCache(n // P, P, KVH, D)
    table = torch.randperm(n // P, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()[None]
    one = [cuda_i32([0, n]), cuda_i32([n])]
    b = m.KVBatch(1, n, n, n, one[0].data_ptr(), one[1].data_ptr(), table.data_ptr(), n // P)
    cache.append(b, rows(m, k), rows(m, v), stream=LEGACY)
    cache.gather(b, rows(m, k), rows(m, v), stream=LEGACY)
    return cache, table, k, v


def attend_long(m, cache, table, q, q_len, B, n, causal):
    """B sequences over the same n rows"""
    T, H, D = q.shape
    tables = table.expand(B, -1).contiguous()
    dev = [torch.arange(0, T + 1, q_len, dtype=torch.int32, device="cuda"),
           torch.full((B,), n, dtype=torch.int32, device="cuda")]
    b = m.KVBatch(B, T, q_len, n, *[x.data_ptr() for x in dev], tables.data_ptr(), table.shape[1])
    out, lse = torch.empty_like(q), torch.empty(T, H, device="cuda")
    size = cache.workspace_bytes(b, H)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    cache.attention(b, rows(m, q), rows(m, out), D ** -0.5, causal=causal, lse=lse.data_ptr(),
                    workspace=ws.data_ptr(), workspace_bytes=size, stream=LEGACY)
    assert cache.status() == 0
    return out, lse


MANY_ITEMS = [("f32", 64, 8, 1200, 1), ("f16", 64, 8, 1, 1200), ("f16", 64, 8, 2400, 1)]   # whole rows an item
LONG_RUNS = [("f32", 64, 2, 1, 256), ("f16", 64, 8, 300, 1)]                               # runs of 256 tiles


@pytest.mark.parametrize("dtype,D,G,q_len,B", MANY_ITEMS + LONG_RUNS)
def test_attention_unsplit_long_rows(m, dtype, D, G, q_len, B):
    """131072 rows in items of thousands of tiles, values of one sign: the tensor cores cut what
    they add to a sum, 2 units of 2^-23 a product at most where 16 addends are each cut 3 bits
    below it, so a chain of N of them loses up to N units of the last sum, half of it on the way
    there.  Chains end after 256 products whatever the rows: 2^-15, and weights as in
    attention_bounds (2^-19).  16-bit results are compared by the mean of their relative errors: each is
    off by up to half of eps, evenly; there are 8 * 64 independent ones, so the mean of these is
    off by eps / 2 / sqrt(3 * 512) and, at 5 deviations, by eps / 15."""
    KVH, n, P = 8, 131072, 256
    dt = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(2)
    k = torch.randn(n, KVH, D, device="cuda", generator=g)
    v = torch.rand(n, KVH, D, device="cuda", generator=g) + torch.rand(1, KVH, D, device="cuda", generator=g)
    cache, table, k, v = long_rows(m, n, D, KVH, P, k, v)
    T = q_len * B
    q = (torch.randn(T, KVH * G, D, device="cuda", generator=g) * 0.1).to(dt)
    out, lse = attend_long(m, cache, table, q, q_len, B, n, False)
    tokens = torch.tensor([0, 7, T // 2, T - 1], device="cuda")
    rel, dl = [], []
    for h in range(KVH):
        kk, vv = k[:, h].double(), v[:, h].double()
        x = q[tokens][:, h * G:(h + 1) * G].double()
        s = torch.einsum("tgd,sd->tgs", x, kk).mul_(D ** -0.5)
        want = torch.einsum("tgs,sd->tgd", s.softmax(-1), vv)
        rel.append((out[tokens][:, h * G:(h + 1) * G].double() - want) / want)
        dl.append((lse[tokens][:, h * G:(h + 1) * G].double() - s.logsumexp(-1)).abs().max())
    rel = torch.cat(rel, 1)
    assert max(dl) <= 2.0 ** -15
    if dtype == "f32":
        assert rel.abs().max() <= 2.0 ** -15 + 2.0 ** -18, rel.abs().max()
    else:
        eps = torch.finfo(dt).eps
        assert rel.mean().abs() <= 2.0 ** -15 + 2.0 ** -18 + eps / 15, rel.mean()
        assert rel.abs().max() <= 2.0 ** -15 + 2.0 ** -11 + eps / 2 * 1.01, rel.abs().max()


@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("dtype,D,G,q_len,B", MANY_ITEMS + [("bf16", 128, 8, 2400, 1), ("bf16", 256, 8, 1200, 1)])
def test_attention_unsplit_growth(m, dtype, D, G, q_len, B, rising):
    """items of 384 tiles whose sums move to their records on the way, while the scores and
    V's scales grow (or fall) along the rows"""
    KVH, n, P = 8, 12288, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    at = torch.arange(n, device="cuda", dtype=torch.float32)
    at = (at if rising else at.flip(0))[:, None, None]
    k = torch.randn(n, KVH, D, device="cuda", generator=g)
    k[..., :1] = at / 512 - 12
    v = torch.randn(n, KVH, D, device="cuda", generator=g) * 2.0 ** torch.floor(at / 1000 - 9)
    cache, table, k, v = long_rows(m, n, D, KVH, P, k, v)
    T = q_len * B
    q = torch.randn(T, KVH * G, D, device="cuda", generator=g)
    q[..., 0] = torch.tensor([4.0, -3.0, 0.02, 1.0] * (KVH * G // 4), device="cuda")
    q = q.to(TYPES[dtype])
    out, lse = attend_long(m, cache, table, q, q_len, B, n, True)
    k, v, x, o, l = f64(k), f64(v), f64(q), f64(out), f64(lse)
    for t in (0, 31, T // 2, T - 1):
        seen = n - q_len + t % q_len + 1
        want, wl, size = ref.attention(x[t:t + 1], k[:seen], v[:seen], D ** -0.5)
        tol, tol_l = ref.attention_bounds(q.dtype, size, np.abs(v[:seen]).max(), min(seen, 4096), want, wl)
        err = np.abs(o[t:t + 1] - want)
        assert (err <= tol).all(), f"token {t}: {(err / tol).max():.3g} of its bound"
        assert (np.abs(l[t:t + 1] - wl) <= tol_l).all(), f"token {t}: lse"
