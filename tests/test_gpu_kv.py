"""Rotary positions, the paged 4-bit cache and attention over it
(moe_rope_*, moe_kv_*) against plain forms in 64 bits (kv_ref.py).

Tolerances.  Rotation: cosine and sine rounded to fp32 (2^-24 each), two
products and a sum rounded once: 3 * 2^-24 (|a| + |b|), then half a step of the
rows' type.  The cache: codes, scales and read-back values exactly, from the
rotation's own fp32 results.  Attention: kv_ref.attention_bounds."""
import numpy as np
import pytest
import torch

import kv_ref as ref
from kv_ref import TYPES, rows

pytestmark = pytest.mark.gpu

LEGACY = 1   # cudaStreamLegacy: torch's default stream


@pytest.fixture
def m(moe):
    torch.backends.cuda.matmul.allow_tf32 = False
    return moe


def rand(seed, *shape, dtype=torch.float32, sd=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * sd).to(dtype)


def cuda_i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def f64(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------ rotation
def check_turned(got, x, pos, freq, layout, mag=1.0):
    want, size = ref.rotate(f64(x), pos, freq, layout, mag)
    tol = 3 * 2.0 ** -24 * size + np.abs(want) * torch.finfo(got.dtype).eps / 2 + 1e-38
    tol[..., 2 * len(freq):] = 0
    err = np.abs(f64(got) - want)
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,H,KVH,D,rot", [(1, 16, 16, 128, 128), (5, 4, 1, 64, 64), (3, 3, 3, 64, 30),
                                            (7, 8, 2, 128, 64), (2, 5, 5, 256, 250), (701, 2, 1, 128, 122),
                                            (2, 2, 2, 34, 34), (1, 1, 1, 2, 2)])
def test_rope(m, T, H, KVH, D, rot, dtype, layout):
    dt = TYPES[dtype]
    x = rand(T + D, T, H + KVH, D, dtype=dt).cuda()
    q, k = x[:, :H], x[:, H:]
    pos = np.random.default_rng(rot).integers(0, 8192, T)
    pos[0] = 8191
    r = m.Rope(rot, 1e4, 8192, m.ROPE_PAIRS if layout == "pairs" else m.ROPE_HALVES)
    qo, ko = torch.empty(T, H, D, dtype=dt, device="cuda"), torch.empty(T, KVH, D, dtype=dt, device="cuda")
    p = cuda_i32(pos)
    r.forward(T, D, p.data_ptr(), rows(m, q), rows(m, qo), rows(m, k), rows(m, ko), stream=LEGACY)
    assert r.status() == 0
    freq = ref.frequencies(rot, 1e4)
    check_turned(qo, q, pos, freq, layout)
    check_turned(ko, k, pos, freq, layout)
    # in place, one tensor, head-major strides
    y = x.transpose(0, 1).contiguous().transpose(0, 1)
    r.forward(T, D, p.data_ptr(), rows(m, y), rows(m, y), stream=LEGACY)
    assert r.status() == 0
    assert torch.equal(y[:, :H], qo) and torch.equal(y[:, H:], ko)


@pytest.mark.parametrize("kw", [
    dict(scaling="linear", factor=4.0), dict(scaling="parts", factor=16.0, orig=4096.0),
    dict(scaling="parts", factor=8.0, orig=1024.0, fast=16.0, slow=2.0),
    dict(scaling="bands", factor=8.0, orig=8192.0), dict(divisors=np.linspace(1, 9, 32))])
def test_rope_scaling_far_positions(m, kw):
    """frequencies of every scaling, up to the largest positions that a plan takes"""
    T, D, rot = 9, 64, 64
    freq = ref.frequencies(rot, 5e5, **kw)
    args = dict(factor=kw.get("factor", 1.0), orig_context=kw.get("orig", 0.0),
                freq_divisors=kw.get("divisors"))
    mag = 1.0
    if kw.get("scaling") == "parts":
        args |= dict(scaling=m.ROPE_PARTS, beta_fast=kw.get("fast", 0.0), beta_slow=kw.get("slow", 0.0))
        mag = 0.1 * np.log(kw["factor"]) + 1.0
    if kw.get("scaling") == "bands":
        args |= dict(scaling=m.ROPE_BANDS, low_freq=1.0, high_freq=4.0)
    if kw.get("scaling") == "linear":
        args |= dict(scaling=m.ROPE_LINEAR)
    r = m.Rope(rot, 5e5, 1 << 24, m.ROPE_HALVES, **args)
    pos = np.array([0, 1, 1023, 1024, 1025, 65537, 1 << 20, (1 << 24) - 2, (1 << 24) - 1])
    x = rand(3, T, 2, D).cuda()
    out, p = torch.empty_like(x), cuda_i32(pos)
    r.forward(T, D, p.data_ptr(), rows(m, x), rows(m, out), stream=LEGACY)
    assert r.status() == 0
    check_turned(out, x, pos, freq, "halves", mag)
    r2 = m.Rope(rot, 5e5, 1 << 20, m.ROPE_HALVES, magnitude=0.5)
    r2.forward(1, D, p.data_ptr(), rows(m, x[:1]), rows(m, out[:1]), stream=LEGACY)
    assert torch.equal(out[:1], x[:1] * 0.5)   # position 0, magnitude a power of two


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("T,H,KVH,D,rot", [(2500, 3, 1, 64, 64), (6001, 1, 1, 128, 64), (20000, 1, 0, 64, 32),
                                            (2500, 1, 1, 256, 250), (9000, 2, 0, 66, 66)])
def test_rope_many_tokens(m, T, H, KVH, D, rot, layout):
    """tokens enough that a CTA takes 2, 4, 8 .. of them; rows at odd offsets and in place
    have the aligned rows' bits"""
    x = rand(T, T, H + KVH, D, dtype=torch.bfloat16).cuda()
    pos = np.random.default_rng(T).integers(0, 4096, T)
    p = cuda_i32(pos)
    r = m.Rope(rot, 1e4, 4096, m.ROPE_PAIRS if layout == "pairs" else m.ROPE_HALVES)

    def turn(a, b):
        k = (rows(m, a[:, H:]), rows(m, b[:, H:])) if KVH else (None, None)
        r.forward(T, D, p.data_ptr(), rows(m, a[:, :H]), rows(m, b[:, :H]), *k, stream=LEGACY)
        assert r.status() == 0

    out = torch.full_like(x, 5.0)
    turn(x, out)
    check_turned(out, x, pos, ref.frequencies(rot, 1e4), layout)
    wide = torch.full((T, (H + KVH) * D + 3), 5.0, dtype=x.dtype, device="cuda")
    odd = wide[:, 1:-2].unflatten(1, (H + KVH, D))
    odd.copy_(x)
    turn(odd, odd)
    assert torch.equal(odd, out) and (wide[:, 0] == 5.0).all() and (wide[:, -2:] == 5.0).all()


def test_rope_positions_out_of_range(m):
    """such a token stays unwritten and is reported once; the others turn"""
    r = m.Rope(64, 1e4, 100)
    x = rand(1, 4, 2, 64).cuda()
    out, pos = torch.full_like(x, 7.0), cuda_i32([5, 100, -1, 99])
    r.forward(4, 64, pos.data_ptr(), rows(m, x), rows(m, out), stream=LEGACY)
    assert r.status() == -1 and r.status() == 0
    assert (out[1:3] == 7.0).all()
    check_turned(out[[0, 3]], x[[0, 3]], [5, 99], ref.frequencies(64, 1e4), "pairs")


def test_rope_broadcast_and_special_values(m):
    """one row for all tokens and heads (strides 0); infinities and NaN stay in their pair;
    values behind rot come back bit for bit"""
    r = m.Rope(32, 1e4, 4096, m.ROPE_HALVES)
    x = rand(2, 1, 1, 64).cuda()
    x[0, 0, 3], x[0, 0, 40], x[0, 0, 41] = float("inf"), float("nan"), -0.0
    out = torch.empty(6, 3, 64, device="cuda")
    pos = cuda_i32([0, 1, 2, 3, 4, 5])
    q = m.Rows(x.data_ptr(), m.F32, 3, 0, 0)
    r.forward(6, 64, pos.data_ptr(), q, rows(m, out), stream=LEGACY)
    assert r.status() == 0
    o = f64(out)
    bad = ~np.isfinite(o)
    bad[:, :, [3, 19, 40]] = False
    assert not bad.any() and np.isnan(o[:, :, 40]).all() and not np.isfinite(o[1:, :, 3]).any()
    assert torch.equal(out[..., 41].view(torch.int32), x[0, 0, 41].view(torch.int32).expand(6, 3))


def test_rope_refusals(m):
    r = m.Rope(64, 1e4, 100)
    x = rand(1, 4, 2, 64).cuda()
    pos = cuda_i32([1] * 4)
    R = rows(m, x)

    def no(code, *a, n=4, d=64, p=pos.data_ptr()):
        with pytest.raises(m.MoeError) as e:
            r.forward(n, d, p, *a, stream=LEGACY)
        assert e.value.code == code

    no(-1, R, None)
    no(-1, R, R, R)
    no(-1, R, R, n=-1)
    no(-1, R, R, d=62)
    no(-1, R, R, d=65)
    no(-1, R, R, p=None)
    no(-2, m.Rows(x.data_ptr(), 1, 2, 128, 64), R)
    no(-2, R, m.Rows(x.data_ptr(), m.F16, 2, 128, 64))
    no(-1, R, m.Rows(x.data_ptr(), m.F32, 1, 128, 64))
    no(-1, m.Rows(x.data_ptr() + 2, m.F32, 2, 128, 64), R)
    no(-1, R, m.Rows(x.data_ptr(), m.F32, 2, 127, 64))
    no(-1, R, m.Rows(x.data_ptr(), m.F32, 2, 128, 0))
    no(-1, R, m.Rows(x.data_ptr(), m.F32, 2, 0, 64))
    no(-1, m.Rows(x.data_ptr(), m.F32, 2, -128, 64), R)
    r.forward(0, 64, None, R, R, stream=LEGACY)
    assert r.status() == 0


def test_rope_refuses_rows_past_64_bits(m):
    """tokens times their stride beyond 64 bits: rows of one place for all heads are refused"""
    r = m.Rope(64, 1e4, 100)
    x, pos = rand(1, 4, 2, 64).cuda(), cuda_i32([1] * 4)
    for n, ts, hs in (((1 << 23) + 1, 1 << 40, 0), (1 << 30, 1 << 40, 0), ((1 << 24) + 1, 1 << 40, 63),
                      ((1 << 24) + 1, 1 << 38, 1 << 39)):
        with pytest.raises(m.MoeError) as e:
            r.forward(n, 64, pos.data_ptr(), rows(m, x), m.Rows(x.data_ptr(), m.F32, 2, ts, hs), stream=LEGACY)
        assert e.value.code == -1
    # head-major rows that just fit, and one value less
    y = torch.empty(2 * 4 * 64, device="cuda")
    r.forward(4, 64, pos.data_ptr(), rows(m, x), m.Rows(y.data_ptr(), m.F32, 2, 64, 256), stream=LEGACY)
    with pytest.raises(m.MoeError):
        r.forward(4, 64, pos.data_ptr(), rows(m, x), m.Rows(y.data_ptr(), m.F32, 2, 64, 255), stream=LEGACY)
    assert r.status() == 0


# ------------------------------------------------------------------ a batch and its cache
class Case:
    """Sequences with random keys and values in a shuffled pool; `fill` "nan" puts a NaN
    scale wherever no row of a sequence stands."""

    def __init__(self, m, q_len, kv_len, KVH, D, P, pad=0, extra=2, fill="nan", seed=0, spare=2):
        self.m, self.q_len, self.kv_len, self.KVH, self.D, self.P = m, q_len, kv_len, KVH, D, P
        rng = np.random.default_rng(seed)
        need = [-(-k // P) for k in kv_len]
        self.n_pages = sum(need) + extra
        perm = rng.permutation(self.n_pages)
        self.table = np.full((len(kv_len), max(need + [0]) + spare), -7, np.int32)
        self.pool = ref.Pool(self.n_pages, P, KVH, D, fill, seed)
        at = 0
        self.k, self.v = [], []
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
            for which in (0, 1):
                x = rng.standard_normal((kv_len[b], KVH, D)).astype(np.float32)
                x *= 1 + 3 * (rng.random((1, KVH, D)) < 0.05)
                for r in range(kv_len[b]):
                    self.pool.put(self.table[b, r // P], r % P, which, x[r])
                (self.k, self.v)[which].append(self.pool.sequence(self.table[b], kv_len[b], which))
        self.start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.T = int(self.start[-1]) + pad
        self.dev = [torch.tensor(x, device="cuda") for x in (self.start, np.array(kv_len, np.int32), self.table)]
        self.pages = torch.tensor(self.pool.data.reshape(-1), device="cuda")
        self.cache = m.KVCache(self.n_pages, P, KVH, D, pages=self.pages.data_ptr())
        self.batch = m.KVBatch(len(kv_len), self.T, max(q_len + [0]), max(kv_len + [0]),
                               *[x.data_ptr() for x in self.dev], self.table.shape[1])

    def attend(self, q, causal=True, window=0, scale=None, lse=True, stream=LEGACY, out=None):
        H = q.shape[1]
        out = torch.full_like(q, 5.0) if out is None else out
        l = torch.full(q.shape[:2], 6.0, device="cuda")
        n = self.cache.workspace_bytes(self.batch, H)
        self.ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")   # NaN everywhere
        self.cache.attention(self.batch, rows(self.m, q), rows(self.m, out), scale or self.D ** -0.5,
                             causal=causal, window=window, lse=l.data_ptr() if lse else None,
                             workspace=self.ws.data_ptr(), workspace_bytes=n, stream=stream)
        return out, l

    def check(self, q, out, lse, causal=True, window=0, scale=None, seqs=None):
        """every sequence's rows (or those of `seqs`) against 64 bits; padding untouched"""
        x, o, l = f64(q), f64(out), f64(lse)
        for b in seqs if seqs is not None else range(len(self.q_len)):
            a, z = self.start[b], self.start[b + 1]
            want, wl, size = ref.attention(x[a:z], self.k[b], self.v[b], scale or self.D ** -0.5, causal, window)
            vmax = np.abs(self.v[b]).max() if len(self.v[b]) else 0.0
            tol, tol_l = ref.attention_bounds(q.dtype, size, vmax, max(1, self.kv_len[b]), want, wl)
            err = np.abs(o[a:z] - want)
            assert (err <= tol).all(), f"sequence {b}: {err.max():.3g}, {(err / tol).max():.3g} of its bound"
            assert (np.isneginf(l[a:z]) == np.isneginf(wl)).all()
            fine = np.isfinite(wl)
            assert (np.abs(l[a:z][fine] - wl[fine]) <= tol_l[fine]).all(), f"sequence {b}: lse"
        end = self.start[-1]
        assert (o[end:] == 5.0).all() and (l[end:] == 6.0).all()


# ------------------------------------------------------------------ append, gather
@pytest.mark.parametrize("layout,rot", [("none", 0), ("pairs", 1.0), ("halves", 1.0), ("halves", 0.5),
                                        ("pairs", -6), ("halves", -6)])
@pytest.mark.parametrize("dtype,D,P,KVH,G,q_len,kv_len,pad", [
    ("f32", 128, 16, 2, 2, [1], [1], 0),
    ("bf16", 128, 64, 2, 4, [1, 1, 1, 1, 1], [7, 64, 65, 1, 200], 2),
    ("f16", 64, 16, 3, 1, [17, 0, 1, 33], [17, 5, 16, 50], 1),
    ("f32", 256, 32, 1, 5, [3, 40], [31, 70], 0),
    ("bf16", 64, 128, 1, 7, [130], [300], 3)])
def test_append_gather(m, dtype, D, P, KVH, G, q_len, kv_len, pad, layout, rot):
    dt, H = TYPES[dtype], KVH * G
    rot = int(D * rot) if 0 < rot <= 1 else D + int(rot) if rot < 0 else 0
    c = Case(m, q_len, kv_len, KVH, D, P, pad=pad, fill=None)
    qkv = rand(1, c.T, H + 2 * KVH, D, dtype=dt, sd=2.0)
    qkv[0, :, :32] = 0.0                              # blocks of zeros
    if c.T > 2:
        qkv[1, H + 2 * KVH - 1, 5] = float("nan")     # a poisoned value block
        qkv[2, H + KVH, 1] = 1e-7 if dt == torch.float32 else 0.0
    qkv = qkv.cuda()
    q, k, v = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
    r = None
    if rot:
        r = m.Rope(rot, 1e4, 512, m.ROPE_PAIRS if layout == "pairs" else m.ROPE_HALVES)
    qo = torch.full((c.T, H, D), 5.0, dtype=dt, device="cuda")
    c.cache.append(c.batch, rows(m, k), rows(m, v), rope=r, q=rows(m, q), q_out=rows(m, qo), stream=LEGACY)
    assert c.cache.status() == 0
    n = int(c.start[-1])
    pos = np.concatenate([np.arange(kv - ql, kv) for ql, kv in zip(q_len, kv_len)]).astype(np.int64)
    # the queries, and the keys in fp32, by the rotation alone (tested above)
    kf, qf = k[:n].float().contiguous(), q[:n].contiguous()
    if r:
        p = cuda_i32(pos)
        r.forward(n, D, p.data_ptr(), rows(m, kf), rows(m, kf), stream=LEGACY)
        r.forward(n, D, p.data_ptr(), rows(m, qf), rows(m, qf), stream=LEGACY)
    bits = lambda t: t.contiguous().view({4: torch.int32, 2: torch.int16}[t.element_size()])  # noqa: E731
    assert torch.equal(bits(qo[:n]), bits(qf)) and (qo[n:] == 5.0).all()
    # the pages: the new rows' bytes and no others
    kf, vf = kf.cpu().numpy(), v[:n].float().cpu().numpy()
    t = 0
    for b, (ql, kv) in enumerate(zip(q_len, kv_len)):
        for row in range(kv - ql, kv):
            c.pool.put(c.table[b, row // P], row % P, 0, kf[t])
            c.pool.put(c.table[b, row // P], row % P, 1, vf[t])
            t += 1
    got = c.pages.cpu().numpy().reshape(c.pool.data.shape)
    nan = lambda a: (a.view(np.uint16) & 0x7fff) > 0x7c00  # noqa: E731
    sc = slice(P * D // 2, None)
    assert np.array_equal(got[..., :P * D // 2], c.pool.data[..., :P * D // 2])
    gs, ws = got[..., sc].copy(), c.pool.data[..., sc].copy()
    assert np.array_equal(nan(gs), nan(ws)) and np.array_equal(gs.view(np.uint16)[~nan(gs)], ws.view(np.uint16)[~nan(gs)])
    # read back, as values of every type
    for odt in (torch.float32, dt):
        ko = torch.full((c.T, KVH, D), 5.0, dtype=odt, device="cuda")
        vo = torch.full_like(ko, 5.0)
        c.cache.gather(c.batch, rows(m, ko), rows(m, vo), stream=LEGACY)
        assert c.cache.status() == 0
        t = 0
        for b, (ql, kv) in enumerate(zip(q_len, kv_len)):
            for row in range(kv - ql, kv):
                for x, which in ((ko, 0), (vo, 1)):
                    want = torch.tensor(c.pool.get(c.table[b, row // P], row % P, which)).to(odt)
                    assert torch.equal(x[t].cpu().nan_to_num(9e9), want.nan_to_num(9e9))
                t += 1
        assert (ko[n:] == 5.0).all() and (vo[n:] == 5.0).all()


@pytest.mark.parametrize("layout,rot", [("none", 0), ("pairs", 64), ("halves", 64), ("halves", 22)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_append_gather_odd_offsets(m, dtype, layout, rot):
    """rows that are not 16-byte aligned, queries turned in place: the aligned call's bits"""
    D, KVH, H, dt = 64, 3, 6, TYPES[dtype]
    q_len, kv_len = [5, 1, 37], [9, 70, 37]
    a, b = (Case(m, q_len, kv_len, KVH, D, 16, pad=2, fill=None) for _ in range(2))
    x = rand(5, a.T, H + 2 * KVH, D, dtype=dt).cuda()
    wide = torch.full((a.T, (H + 2 * KVH) * D + 5), 5.0, dtype=dt, device="cuda")
    odd = wide[:, 3:-2].unflatten(1, (H + 2 * KVH, D))
    odd.copy_(x)
    r = m.Rope(rot, 1e4, 512, m.ROPE_PAIRS if layout == "pairs" else m.ROPE_HALVES) if rot else None
    qo = x[:, :H].clone()
    for c, y, o in ((a, x, qo), (b, odd, odd[:, :H])):
        c.cache.append(c.batch, rows(m, y[:, H:H + KVH]), rows(m, y[:, H + KVH:]), rope=r,
                       q=rows(m, y[:, :H]), q_out=rows(m, o), stream=LEGACY)
        assert c.cache.status() == 0
    assert torch.equal(a.pages, b.pages) and torch.equal(odd[:, :H], qo)
    assert torch.equal(odd[:, H:], x[:, H:]) and (wide[:, :3] == 5.0).all() and (wide[:, -2:] == 5.0).all()
    ko, vo = x[:, H:H + KVH].clone(), x[:, H + KVH:].clone()
    a.cache.gather(a.batch, rows(m, ko), rows(m, vo), stream=LEGACY)
    b.cache.gather(b.batch, rows(m, odd[:, H:H + KVH]), rows(m, odd[:, H + KVH:]), stream=LEGACY)
    assert torch.equal(odd[:, H:H + KVH], ko) and torch.equal(odd[:, H + KVH:], vo)


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("T,D,KVH", [(2500, 64, 2), (6001, 128, 1), (20001, 64, 1)])
def test_append_gather_many_tokens(m, T, D, KVH, layout):
    """tokens enough that a CTA takes 2, 4, 8 .. of them, ragged sequences inside them: the
    bytes of a call a sequence"""
    rng = np.random.default_rng(T)
    q_len = [1, 0, 1, 700, 3, 33]
    q_len = [int(x) for x in q_len + [T - sum(q_len)]]
    before = [int(x) for x in rng.integers(0, 90, len(q_len))]
    kv_len = [x + y for x, y in zip(q_len, before)]
    P, H = 64, KVH
    need = [-(-x // P) for x in kv_len]
    perm = rng.permutation(sum(need))
    table = np.full((len(kv_len), max(need)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(q_len)])
    dev = [cuda_i32(start), cuda_i32(kv_len), torch.tensor(table, device="cuda")]
    x = rand(1, T, H + 2 * KVH, D, dtype=torch.bfloat16).cuda()
    r = m.Rope(D, 1e4, 32768, m.ROPE_PAIRS if layout == "pairs" else m.ROPE_HALVES)
    got = []
    for whole in (True, False):
        cache = m.KVCache(sum(need), P, KVH, D)
        out = torch.full((T, H + 2 * KVH, D), 5.0, dtype=x.dtype, device="cuda")
        for i in [None] if whole else [j for j in range(len(q_len)) if q_len[j]]:
            a, n = (0, T) if whole else (int(start[i]), q_len[i])
            one = dev if whole else [cuda_i32([0, n]), dev[1][i:], dev[2][i:]]
            batch = m.KVBatch(len(q_len) if whole else 1, n, max(q_len), max(kv_len),
                              *[y.data_ptr() for y in one], table.shape[1])
            y, o = x[a:a + n], out[a:a + n]
            cache.append(batch, rows(m, y[:, H:H + KVH]), rows(m, y[:, H + KVH:]), rope=r,
                         q=rows(m, y[:, :H]), q_out=rows(m, o[:, :H]), stream=LEGACY)
            cache.gather(batch, rows(m, o[:, H:H + KVH]), rows(m, o[:, H + KVH:]), stream=LEGACY)
        assert cache.status() == 0
        got.append(out)
    assert torch.equal(*got)
    # and the values themselves, the keys after the rotation
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, q_len)])
    p, kt = cuda_i32(pos.tolist()), x[:, H:H + KVH].float().contiguous()
    r.forward(T, D, p.data_ptr(), rows(m, kt), rows(m, kt), stream=LEGACY)
    for i, want in ((H, kt), (H + KVH, x[:, H + KVH:].float())):
        want = want.cpu().numpy()
        y = torch.tensor(ref.values(*ref.quantize(want))).to(torch.bfloat16)
        assert torch.equal(got[0][:, i:i + KVH].cpu(), y)


def test_quantizer_edges(m):
    """scales at both ends of fp16, ties of the largest magnitude, rounding to even, a
    block with an infinity"""
    D = 64
    c = Case(m, [8], [8], 1, D, 16, fill=None)
    x = np.zeros((8, 1, D), np.float32)
    x[0, 0, :32] = np.linspace(-8, 7, 32)           # halves between codes
    x[0, 0, 32:] = np.linspace(8, -8, 32)           # +8 and -8: the positive one counts
    x[1, 0, :32] = 1e9                              # above 8 * 65504
    x[1, 0, 32:] = -1e9
    x[2, 0, :32] = 1e-7                             # scale rounds to a subnormal, or 0
    x[2, 0, 32:] = 2.0 ** -22
    x[3, 0, 4] = np.inf
    x[3, 0, 40] = -np.inf
    x[4, 0, 4] = np.nan
    x[5, 0] = np.arange(D) / 64 - 0.5
    x[6, 0, 0], x[6, 0, 63] = -3.0, 3.0
    x[7, 0] = 524032.0                              # 8 * 65504
    d = torch.tensor(x).cuda()
    c.cache.append(c.batch, rows(m, d), rows(m, d), stream=LEGACY)
    out = torch.empty_like(d)
    for which in (0, 1):
        c.cache.gather(c.batch, **{("k_out", "v_out")[which]: rows(m, out)}, stream=LEGACY)
        want = ref.values(*ref.quantize(x))
        assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want[3]).all() and np.isnan(want[4, 0, :32]).all() and np.isfinite(want[4, 0, 32:]).all()
    assert want[1, 0, 0] == 8 * 65504 and want[1, 0, 63] == -8 * 65504 and want[7, 0, 0] == 524032


def test_append_positions(m):
    """positions of their own; one outside the tables leaves the token out and is reported"""
    D = 64
    c = Case(m, [3], [5], 1, D, 16, fill=None)
    before = c.pages.clone()
    x = rand(3, 3, 2, D).cuda()
    r = m.Rope(D, 1e4, 1000)
    pos, qo = cuda_i32([700, 1000, -1]), torch.full((3, 1, D), 5.0, device="cuda")
    k = x[:, 1:]
    c.cache.append(c.batch, rows(m, k), rows(m, k), rope=r, pos=pos.data_ptr(), q=rows(m, x[:, :1]),
                   q_out=rows(m, qo), stream=LEGACY)
    assert c.cache.status() == -1 and c.cache.status() == 0
    check_turned(qo[:1], x[:1, :1], [700], ref.frequencies(D, 1e4), "pairs")
    assert (qo[1:] == 5.0).all()
    c.pool.put(c.table[0, 0], 2, 1, x[0, 1:].cpu().numpy())
    out = torch.empty(3, 1, D, device="cuda")
    c.cache.gather(c.batch, v_out=rows(m, out), stream=LEGACY)
    assert np.array_equal(out[0].cpu().numpy(), c.pool.get(c.table[0, 0], 2, 1))
    # only the first token's row changed
    changed = (c.pages != before).view(c.pool.data.shape).nonzero()
    assert set(changed[:, 0].tolist()) == {int(c.table[0, 0])}


# ------------------------------------------------------------------ attention
LENGTHS = {
    "one": ([1], [1]), "decode": ([1] * 6, [1, 31, 32, 33, 130, 257]), "split": ([1, 1], [1500, 3]),
    "mixed": ([3, 1, 0, 20, 5], [3, 64, 9, 41, 70]), "prompt": ([75], [75]), "tail": ([40], [333]),
    "short": ([9, 1, 2], [4, 0, 2])}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,KVH,G,P", [(128, 2, 4, 64), (64, 1, 7, 16), (128, 2, 1, 32), (256, 1, 2, 16),
                                       (64, 2, 8, 128), (128, 1, 16, 256), (256, 1, 12, 32)])
def test_attention(m, D, KVH, G, P, dtype, lengths):
    """short: more queries than rows (the first see nothing), a sequence without rows"""
    q_len, kv_len = LENGTHS[lengths]
    c = Case(m, q_len, kv_len, KVH, D, P, pad=3, seed=D + G)
    q = rand(7, c.T, KVH * G, D, dtype=TYPES[dtype], sd=1.5).cuda()
    out, lse = c.attend(q)
    assert c.cache.status() == 0
    c.check(q, out, lse)
    again, lse2 = c.attend(q)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 17), (True, 64), (True, 1000)])
@pytest.mark.parametrize("dtype,D,KVH,G,P", [("f32", 128, 1, 2, 16), ("bf16", 64, 2, 8, 32), ("f16", 128, 2, 1, 64)])
def test_attention_masks(m, dtype, D, KVH, G, P, causal, window):
    c = Case(m, [1, 30, 6, 2], [300, 30, 200, 1], KVH, D, P, pad=1, seed=3)
    q = rand(8, c.T, KVH * G, D, dtype=TYPES[dtype]).cuda()
    if window:
        # rows and pages behind every query's window: unseen, and no longer there
        for b, (n, kv) in enumerate(zip(c.q_len, c.kv_len)):
            low = max(0, kv - n - window + 1)
            for row in range(low):
                c.pool.scales()[c.table[b, row // P], :, :, row % P] = 0x7fff
            c.table[b, :low // P] = -1
        c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
        c.dev[2].copy_(torch.tensor(c.table))
    out, lse = c.attend(q, causal, window)
    assert c.cache.status() == 0
    c.check(q, out, lse, causal, window)


def test_attention_strides_scale_no_lse(m):
    """query heads inside fused rows at odd offsets, head-major results, another scale, negative scale"""
    D, KVH, G = 64, 2, 3
    c = Case(m, [2, 5], [50, 90], KVH, D, 16, pad=2)
    H = KVH * G
    for dt in (torch.float32, torch.bfloat16):
        wide = rand(4, c.T, H * D + 35, dtype=dt).cuda()
        q = wide[:, 33:33 + H * D].unflatten(1, (H, D))
        for scale in (0.3, -0.2):
            out = torch.full((H, c.T, D), 5.0, dtype=dt, device="cuda").transpose(0, 1)
            o, lse = c.attend(q, scale=scale, out=out)
            assert c.cache.status() == 0
            c.check(q, o, lse, scale=scale)
            o2, l2 = c.attend(q, scale=scale, lse=False)
            assert torch.equal(o2, o) and (l2 == 6.0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_in_place_shared_pages(m, dtype):
    """results over their queries; two sequences that hold the same pages"""
    D, KVH, G = 128, 2, 4
    c = Case(m, [1, 1, 40, 1], [700, 700, 90, 0], KVH, D, 32, pad=2)
    c.table[1] = c.table[0]
    c.k[1], c.v[1] = c.k[0], c.v[0]
    c.dev[2].copy_(torch.tensor(c.table))
    q = rand(9, c.T, KVH * G, D, dtype=TYPES[dtype]).cuda()
    q[c.start[-1]:] = 5.0
    out, lse = c.attend(q)
    same = q.clone()
    same, lse2 = c.attend(same, out=same)
    assert c.cache.status() == 0
    c.check(q, out, lse)
    assert torch.equal(same, out) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,KVH,G,P,q_len,kv_len,causal,window", [
    (128, 1, 4, 64, [64], [64], True, 0),              # one whole item of 256 query rows
    (128, 2, 4, 32, [65, 96], [2065, 96], True, 0),    # rows of a second item; several runs
    (64, 1, 8, 16, [33, 200], [33, 1000], True, 0),    # pages of half a tile
    (128, 1, 1, 128, [300, 1, 7], [300, 900, 7], True, 0),   # a prompt beside decode steps
    (64, 2, 5, 256, [27, 130, 2], [50, 600, 2], True, 100),
    (128, 1, 16, 32, [9, 40], [40, 333], False, 0),
    (64, 1, 129, 64, [3, 1], [70, 70], True, 0)])      # rows of a token over two items
def test_attention_many_queries(m, D, KVH, G, P, q_len, kv_len, causal, window, dtype):
    """sequences of 128 query rows of a KV head and more, alone and beside small ones; K scales
    over all of fp16's range (above 2^13 and subnormal), V scales that grow from tile to
    tile; what no query sees may hold anything"""
    c = Case(m, q_len, kv_len, KVH, D, P, pad=2, seed=sum(kv_len))
    q = rand(3, c.T, KVH * G, D, dtype=TYPES[dtype], sd=1.2).cuda()
    out, lse = c.attend(q, causal, window)
    assert c.cache.status() == 0
    c.check(q, out, lse, causal, window)
    # K of a row, V of a tile far apart
    rng = np.random.default_rng(1)
    for b, n in enumerate(kv_len):
        for r in range(n):
            at = (c.table[b, r // P], slice(None), slice(None), r % P)
            f = np.array([2.0 ** rng.integers(-16, 17), 2.0 ** min(r // 32 - 9, 9)], np.float32)
            sc = c.pool.scales()[at].view(np.float16).astype(np.float32)
            c.pool.scales()[at] = np.clip(sc * f[:, None], -65504, 65504).astype(np.float16).view(np.uint16)
        c.k[b], c.v[b] = (c.pool.sequence(c.table[b], n, w) for w in (0, 1))
    c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
    top = max(float(np.abs(k).max()) for k in c.k)
    out, lse = c.attend(q, causal, window, scale=3.0 / top)
    assert c.cache.status() == 0
    c.check(q, out, lse, causal, window, scale=3.0 / top)
    again, lse2 = c.attend(q, causal, window, scale=3.0 / top)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_many_queries_strides_in_place(m, dtype):
    """query rows at odd offsets, head-major results; results over the queries; a negative scale;
    nothing seen by the first queries; no log-sum-exp"""
    D, KVH, G = 64, 2, 4
    c = Case(m, [70, 200], [130, 150], KVH, D, 16, pad=2)
    H = KVH * G
    wide = rand(4, c.T, H * D + 35, dtype=TYPES[dtype]).cuda()
    q = wide[:, 33:33 + H * D].unflatten(1, (H, D))
    q[c.start[-1]:] = 5.0
    plain, lse = c.attend(q.contiguous(), scale=-0.2)
    c.check(q, plain, lse, scale=-0.2)
    out = torch.full((H, c.T, D), 5.0, dtype=q.dtype, device="cuda").transpose(0, 1)
    o, _ = c.attend(q, scale=-0.2, out=out)
    assert torch.equal(o, plain)
    o, l2 = c.attend(q, scale=-0.2, out=q, lse=False)
    assert torch.equal(q, plain) and (l2 == 6.0).all()
    assert c.cache.status() == 0


def test_attention_many_queries_poisoned(m):
    """a NaN scale of K or of a block of V reaches the queries that see its row, there its
    block, and no others"""
    D, G, kv = 128, 4, 100
    c = Case(m, [kv], [kv], 1, D, 32, pad=0)
    q = rand(5, kv, G, D, dtype=torch.bfloat16).cuda()
    clean, _ = c.attend(q)
    for which, block, row in ((1, 2, 40), (0, 1, 70)):
        old = c.pool.data.copy()
        c.pool.scales()[c.table[0, row // 32], :, which, row % 32, block] = 0x7e00
        c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
        out, _ = c.attend(q)
        assert torch.equal(out[:row], clean[:row])
        part = out[row:, :, 32 * block:32 * block + 32] if which else out[row:]
        assert part.isnan().all()
        if which:
            keep = [e for e in range(D) if e // 32 != block]
            assert torch.equal(out[row:, :, keep], clean[row:, :, keep])
        c.pool.data[...] = old


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_len,kv_len,causal", [
    ([64], [0], True), ([64], [0], False), ([200], [100], True),   # queries before the first row
    ([300, 3, 64, 128], [70, 40, 0, 128], True), ([300], [1], True)])
def test_attention_many_queries_nothing_seen(m, q_len, kv_len, causal, D, dtype):
    """items of 256 query rows without a key tile: zeros and -infinity, alone and beside
    sequences that see rows"""
    c = Case(m, q_len, kv_len, 2, D, 32, pad=1, seed=1)
    q = rand(2, c.T, 8, D, dtype=TYPES[dtype]).cuda()
    for _ in range(3):
        out, lse = c.attend(q, causal)
        assert c.cache.status() == 0
        c.check(q, out, lse, causal)


@pytest.mark.parametrize("D,KVH,G,P", [(128, 4, 1, 64), (64, 1, 7, 16), (256, 1, 8, 32)])
def test_attention_fp32_error(m, D, KVH, G, P):
    """Many keys of equal weight: results are 1 / sqrt(n) of V, and an error of the weighted
    sums counts sqrt(n)-fold.  Of a weight: 2^-20 of the score's size (as in
    attention_bounds) with a sign of its own, so it keeps its share; sums cut to 24 bits:
    2^-22 of V's size a product, less than 2^-19 / sqrt(n) of the whole.  Together below
    2^-18 = 3.8e-6 of the results' norm; sums of 17 bits would be above 8e-6."""
    n = 2049
    c = Case(m, [1], [n], KVH, D, P, pad=0)
    q = rand(9, 1, KVH * G, D, sd=0.5).cuda()
    out, _ = c.attend(q)
    want = ref.attention(f64(q), c.k[0], c.v[0], D ** -0.5)[0]
    err = np.linalg.norm(f64(out) - want) / np.linalg.norm(want)
    assert err <= 2.0 ** -18, err


def test_attention_extreme_values(m):
    """queries and cache scales far from 1 (the kernel's fp16 operands are brought to
    its range by powers of two), blocks of values of very different size"""
    D = 128
    c = Case(m, [2], [140], 1, D, 32, fill="nan")
    x = np.random.default_rng(5).standard_normal((140, 1, D)).astype(np.float32)
    size = np.array([1e-3, 1.0, 3e4, 1e-5], np.float32).repeat(32)
    for dt, up in ((torch.float32, 1e-20), (torch.float32, 1e18), (torch.bfloat16, 1e12), (torch.float16, 1e-4)):
        c.k, c.v = [[]], [[]]
        for r in range(140):
            c.pool.put(c.table[0, r // 32], r % 32, 0, x[r] * 1e-3)
            c.pool.put(c.table[0, r // 32], r % 32, 1, x[139 - r] * size)
        for which in (0, 1):
            (c.k, c.v)[which][0] = c.pool.sequence(c.table[0], 140, which)
        c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
        q = (rand(6, 2, 4, D, dtype=torch.float32) * up).to(dt).cuda()
        scale = float(np.float32(100.0 / up))
        out, lse = c.attend(q, scale=scale)
        assert c.cache.status() == 0
        # block by block: each block's error against its own size
        want, wl, s = ref.attention(f64(q), c.k[0], c.v[0], scale)
        for b in range(4):
            e = slice(32 * b, 32 * b + 32)
            tol, tol_l = ref.attention_bounds(dt, s, np.abs(c.v[0][..., e]).max(), 140, want[..., e], wl)
            assert (np.abs(f64(out)[..., e] - want[..., e]) <= tol).all(), (dt, up, b)
        assert (np.abs(f64(lse) - wl) <= tol_l).all()


def test_attention_peaks_and_growth(m):
    """scores whose maximum rises along the sequence, row by row and by far (rescaling), and
    one that towers at the start"""
    D, n = 64, 400
    for order in (1, -1):
        c = Case(m, [1], [n], 1, D, 64)
        k = np.zeros((n, 1, D), np.float32)
        k[:, 0, 0] = (np.arange(n) - n / 2)[::order] / 2.0
        k[:, 0, 1:] = np.random.default_rng(1).standard_normal((n, D - 1)) * 0.1
        for r in range(n):
            c.pool.put(c.table[0, r // 64], r % 64, 0, k[r])
        c.k[0] = c.pool.sequence(c.table[0], n, 0)
        c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
        for dt in TYPES.values():
            q = rand(2, 1, 4, D).cuda()
            q[0, :, 0] = torch.tensor([1.0, -1.0, 0.01, 5.0])
            out, lse = c.attend(q.to(dt), scale=1.0)
            assert c.cache.status() == 0
            c.check(q.to(dt), out, lse, scale=1.0)


def test_attention_poisoned(m):
    """a NaN or an infinity in a query makes that query's head NaN and no other; a poisoned
    key row every query that sees it; a poisoned value block its 32 values"""
    D = 64
    c = Case(m, [3], [40], 2, D, 16)
    q = rand(3, 3, 4, D).cuda()
    clean, _ = c.attend(q)
    bad = q.clone()
    bad[1, 2, 7], bad[2, 0, 9] = float("nan"), float("-inf")
    out, lse = c.attend(bad)
    nan = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    nan[1, 2] = nan[2, 0] = True
    assert torch.equal(out.isnan().all(-1), nan) and torch.equal(out.isnan().any(-1), nan)
    assert torch.equal(out[~nan], clean[~nan]) and torch.equal(lse.isnan(), nan)
    s = c.pool.scales()
    s[c.table[0, 2], 0, 0, 39 % 16, 1] = 0x7fff       # row 39's keys, KV head 0: seen by query 2 alone
    s[c.table[0, 0], 1, 1, 3, 0] = 0x7fff             # row 3's values, KV head 1, first block
    c.pages.copy_(torch.tensor(c.pool.data.reshape(-1)))
    out, lse = c.attend(q)
    nan = torch.zeros(3, 4, D, dtype=torch.bool, device="cuda")
    nan[2, :2] = True
    nan[:, 2:, :32] = True
    assert torch.equal(out.isnan(), nan) and torch.equal(out[~nan], clean[~nan])
    assert c.cache.status() == 0


def test_attention_bad_arrays(m):
    """pages outside the cache count as unseen rows, sequences with impossible lengths are
    left out; both are reported, the others are right, nothing else is written"""
    D = 64
    c = Case(m, [1, 1, 2, 1], [40, 100, 70, 20], 1, D, 16, pad=1, spare=6)
    q = rand(3, c.T, 4, D).cuda()
    c.dev[2][0, 1] = c.n_pages
    c.dev[2][1, 5] = -3
    out, lse = c.attend(q)
    assert c.cache.status() == -1 and c.cache.status() == 0
    c.check(q, out, lse, seqs=[2, 3])
    c.k[0], c.v[0] = np.delete(c.k[0], slice(16, 32), 0), np.delete(c.v[0], slice(16, 32), 0)
    c.k[1], c.v[1] = np.delete(c.k[1], slice(80, 96), 0), np.delete(c.v[1], slice(80, 96), 0)
    c.check(q, out, lse, seqs=[0, 1])
    # append there: the token is left out
    c.dev[2][0, 2] = 1 << 30
    before = c.pages.clone()
    k = rand(4, c.T, 1, D).cuda()
    c.cache.append(c.batch, rows(m, k), rows(m, k), stream=LEGACY)
    assert c.cache.status() == -1
    assert torch.equal(c.pages[c.table[0, 0] * 16 * 72:][:16 * 72], before[c.table[0, 0] * 16 * 72:][:16 * 72])
    c.pages.copy_(before)   # the other sequences' tokens were appended
    # lengths: above max_kv, negative, below the queries (append only), q_start falling or beyond n_tokens
    for start, kv, good in ([[0, 1, 2, 4, 5], [40, 101, 70, 20], [3]], [[0, 1, 2, 4, 5], [40, -1, 70, 20], [3]],
                            [[0, 1, 2, 4, 99], [40, 100, 70, 20], []], [[0, 1, 0, 2, 3], [40, 100, 70, 20], []],
                            [[-1, 1, 2, 4, 5], [40, 100, 70, 20], [3]], [[0, 1, 2, 5, 6], [40, 100, 70, 20], []]):
        c.dev[0].copy_(torch.tensor(start))
        c.dev[1].copy_(torch.tensor(kv))
        c.dev[2].copy_(torch.tensor(c.table))
        out, lse = c.attend(q)
        assert c.cache.status() == -1, (start, kv)
        if good:
            c.check(q, out, lse, seqs=good)
        before = c.pages.clone()
        c.cache.append(c.batch, rows(m, k), rows(m, k), stream=LEGACY)
        assert c.cache.status() == -1, (start, kv)
        c.pages.copy_(before)


def test_many_sequences(m):
    """more sequences than the kernel's planning takes in one round, some without queries"""
    n = 300
    rng = np.random.default_rng(0)
    kv = [int(x) for x in rng.integers(0, 60, n)]
    ql = [min(k, int(x)) for k, x in zip(kv, rng.integers(0, 3, n))]
    c = Case(m, ql, kv, 1, 64, 16, pad=2)
    q = rand(5, c.T, 2, 64, dtype=torch.bfloat16).cuda()
    out, lse = c.attend(q)
    assert c.cache.status() == 0
    c.check(q, out, lse)


def test_long_cache_offsets(m):
    """a pool of over 4 GiB: the pages at its end are as good as those at its start (the
    rows' offsets pass 32 bits)"""
    D, KVH, P = 128, 8, 256
    per = m.kv_page_bytes(P, KVH, D)
    n = (1 << 32) // per + 40
    pages = torch.empty(n * per, dtype=torch.uint8, device="cuda")
    cache = m.KVCache(n, P, KVH, D, pages=pages.data_ptr())
    kv, ql = 300, 300
    x = rand(1, ql, 3 * KVH, D).cuda()
    out, ws = [], torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    for table in ([1, 0], [n - 1, n - 2]):
        t = [cuda_i32([0, ql]), cuda_i32([kv]), cuda_i32(table)]
        b = m.KVBatch(1, ql, ql, kv, *[a.data_ptr() for a in t], 2)
        q = x[:, :KVH].contiguous()
        o, l = torch.empty_like(q), torch.empty(ql, KVH, device="cuda")
        cache.append(b, rows(m, x[:, KVH:2 * KVH]), rows(m, x[:, 2 * KVH:]), stream=LEGACY)
        cache.attention(b, rows(m, q), rows(m, o), 0.1, lse=l.data_ptr(), workspace=ws.data_ptr(),
                        workspace_bytes=ws.numel(), stream=LEGACY)
        g = torch.empty_like(q)
        cache.gather(b, k_out=rows(m, g), stream=LEGACY)
        assert cache.status() == 0
        out.append((o, l, g))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    k = out[1][2].cpu().numpy()
    assert np.array_equal(k, ref.values(*ref.quantize(x[:, KVH:2 * KVH].cpu().numpy())))


# ------------------------------------------------------------------ together
def test_generation_steps_in_a_graph(m):
    """a ragged prompt appended and attended, then decode steps captured once and replayed
    with the lengths moved on the device; each step against 64 bits on the rows
    that the cache holds"""
    D, KVH, G, P = 128, 2, 4, 16
    H, B, steps = KVH * G, 3, 5
    prompt, room = [7, 33, 1], 64
    r = m.Rope(D, 1e6, 4096)
    cache = m.KVCache(B * room // P, P, KVH, D)
    table = torch.tensor(np.random.default_rng(1).permutation(B * room // P).reshape(B, -1).astype(np.int32)).cuda()
    kv = cuda_i32(prompt)
    stream = torch.cuda.Stream()

    class Call:
        def __init__(self, q_len, seed):
            self.start = cuda_i32(np.concatenate([[0], np.cumsum(q_len)]))
            T = sum(q_len)
            self.q_len, self.batch = q_len, m.KVBatch(B, T, max(q_len), room, self.start.data_ptr(), kv.data_ptr(),
                                                      table.data_ptr(), room // P)
            self.qkv = rand(seed, T, H + 2 * KVH, D, dtype=torch.bfloat16).cuda()
            self.q, self.out = (torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            self.lse = torch.empty(T, H, device="cuda")
            self.ws = torch.empty(max(16, cache.workspace_bytes(self.batch, H)), dtype=torch.uint8, device="cuda")

        def run(self):
            x = self.qkv
            s = torch.cuda.current_stream().cuda_stream
            cache.append(self.batch, rows(m, x[:, H:H + KVH]), rows(m, x[:, H + KVH:]), rope=r,
                         q=rows(m, x[:, :H]), q_out=rows(m, self.q), stream=s)
            cache.attention(self.batch, rows(m, self.q), rows(m, self.out), D ** -0.5, lse=self.lse.data_ptr(),
                            workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel(), stream=s)

        def check(self):
            torch.cuda.synchronize()
            assert cache.status() == 0
            lens = kv.tolist()
            whole = cuda_i32(np.concatenate([[0], np.cumsum(lens)]))
            n = sum(lens)
            b = m.KVBatch(B, n, max(lens), room, whole.data_ptr(), kv.data_ptr(), table.data_ptr(), room // P)
            k, v = (torch.empty(n, KVH, D, device="cuda") for _ in range(2))
            cache.gather(b, rows(m, k), rows(m, v), stream=LEGACY)
            k, v, w = f64(k), f64(v), whole.tolist()
            a = 0
            for i, ql in enumerate(self.q_len):
                kk, vv = k[w[i]:w[i + 1]], v[w[i]:w[i + 1]]
                # the newest rows are this call's keys, turned to the row they stand at
                x = f64(self.qkv[a:a + ql, H:H + KVH])
                turned, _ = ref.rotate(x, np.arange(lens[i] - ql, lens[i]), ref.frequencies(D, 1e6), "pairs")
                step = np.abs(turned).reshape(ql, KVH, -1, 32).max(-1).repeat(32, -1) / 8 * 1.01
                assert (np.abs(kk[-ql:] - turned) <= step).all()
                want, wl, size = ref.attention(f64(self.q[a:a + ql]), kk, vv, D ** -0.5)
                tol, tol_l = ref.attention_bounds(torch.bfloat16, size, np.abs(vv).max(), lens[i], want, wl)
                assert (np.abs(f64(self.out[a:a + ql]) - want) <= tol).all()
                assert (np.abs(f64(self.lse[a:a + ql]) - wl) <= tol_l).all()
                a += ql

    with torch.cuda.stream(stream):
        first = Call(prompt, 1)
        first.run()
        first.check()
        step = Call([1] * B, 2)
        kv += 1
        step.run()   # before the capture: kernel attributes
        step.check()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            kv.add_(1)
            step.run()
        for i in range(steps):
            step.qkv.copy_(rand(10 + i, B, H + 2 * KVH, D, dtype=torch.bfloat16))
            g.replay()
            step.check()
    assert kv.tolist() == [p + 1 + steps for p in prompt]


def test_two_streams(m):
    """two batches over one cache at once, each with its workspace, on streams of their own"""
    D = 64
    c = Case(m, [1] * 8, [700] * 8, 1, D, 32)
    q = [rand(s, 8, 8, D, dtype=torch.bfloat16).cuda() for s in (1, 2)]
    want = [c.attend(x)[0].clone() for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    n = c.cache.workspace_bytes(c.batch, 8)
    ws = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for _ in q]
    out = [torch.empty_like(x) for x in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, o, w, s in zip(q, out, ws, streams):
            c.cache.attention(c.batch, rows(m, x), rows(m, o), D ** -0.5, workspace=w.data_ptr(),
                              workspace_bytes=n, stream=s.cuda_stream)
    assert c.cache.status() == 0
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_cache_refusals(m):
    D = 64
    c = Case(m, [1, 1], [40, 1500], 2, D, 16)
    x = rand(1, 2, 8, D).cuda()
    q, k = rows(m, x[:, :4]), rows(m, x[:, 4:6])
    o = torch.empty(2, 4, D, device="cuda")
    n = c.cache.workspace_bytes(c.batch, 4)
    assert n > 0
    ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")

    def no(code, fn, *a, **kw):
        with pytest.raises(m.MoeError) as e:
            fn(*a, **kw)
        assert e.value.code == code, str(e.value)

    at = c.cache.attention
    ok = dict(workspace=ws.data_ptr(), workspace_bytes=n, stream=LEGACY)
    at(c.batch, q, rows(m, o), 0.1, **ok)
    no(-1, at, c.batch, q, rows(m, o), 0.1, stream=LEGACY)
    no(-1, at, c.batch, q, rows(m, o), 0.1, **(ok | dict(workspace_bytes=n - 1)))
    no(-1, at, c.batch, q, rows(m, o), 0.1, **(ok | dict(workspace=ws.data_ptr() + 8)))
    no(-1, at, c.batch, q, rows(m, o), float("nan"), **ok)
    no(-1, at, c.batch, q, rows(m, o), 0.1, window=-1, **ok)
    no(-1, at, c.batch, q, rows(m, o), 0.1, window=4, causal=False, **ok)
    no(-1, at, c.batch, rows(m, x[:, :3]), rows(m, o[:, :3]), 0.1, **ok)
    no(-1, at, c.batch, q, rows(m, o[:, :2]), 0.1, **ok)
    no(-2, at, c.batch, q, rows(m, o.half()), 0.1, **ok)
    no(-1, at, c.batch, q, m.Rows(o.data_ptr(), m.F32, 4, 64, 64), 0.1, **ok)
    no(-1, c.cache.workspace_bytes, c.batch, 3)
    for field, bad in (("n_seqs", -1), ("n_tokens", -1), ("max_q", -1), ("max_kv", -1), ("max_kv", 1 << 20),
                       ("table_stride", -1), ("table_stride", 3), ("q_start", None), ("kv_len", None),
                       ("page_table", None)):
        b = type(c.batch).from_buffer_copy(c.batch)
        setattr(b, field, bad)
        no(-1, at, b, q, rows(m, o), 0.1, **ok)
        no(-1, c.cache.append, b, k, k, stream=LEGACY)
        no(-1, c.cache.gather, b, rows(m, torch.empty(2, 2, D, device="cuda")), stream=LEGACY)
    ap = c.cache.append
    no(-1, ap, c.batch, k, None, stream=LEGACY)
    no(-1, ap, c.batch, k, rows(m, x[:, :1]), stream=LEGACY)
    no(-1, ap, c.batch, k, k, q=q, stream=LEGACY)
    no(-2, ap, c.batch, k, rows(m, x[:, :2].half()), stream=LEGACY)
    no(-1, ap, c.batch, k, k, rope=m.Rope(128, 1e4, 100), stream=LEGACY)
    no(-1, ap, c.batch, k, k, q=rows(m, x[:, :3]), q_out=rows(m, o[:, :3]), stream=LEGACY)
    no(-1, c.cache.gather, c.batch, stream=LEGACY)
    # empty batches: nothing to do
    for field in ("n_seqs", "n_tokens"):
        b = type(c.batch).from_buffer_copy(c.batch)
        setattr(b, field, 0)
        at(b, q, rows(m, o), 0.1, **ok)
        ap(b, k, k, stream=LEGACY)
    assert c.cache.status() == 0
    assert c.cache.pages == c.pages.data_ptr()


def test_own_pages_and_library_stream(m):
    """a cache with pages of its own (zeroed), on the library's stream"""
    cache = m.KVCache(3, 16, 1, 64)
    t = [cuda_i32([0, 2]), cuda_i32([18]), cuda_i32([2, 0])]
    b = m.KVBatch(1, 2, 2, 32, *[a.data_ptr() for a in t], 2)
    k = rand(1, 2, 1, 64).cuda()
    out = torch.empty(2, 1, 64, device="cuda")
    torch.cuda.synchronize()
    cache.gather(b, rows(m, out))
    m.check(m.lib().moe_sync())
    assert (out == 0).all()
    cache.append(b, rows(m, k), rows(m, k))
    cache.gather(b, rows(m, out))
    m.check(m.lib().moe_sync())
    assert np.array_equal(out.cpu().numpy(), ref.values(*ref.quantize(k.cpu().numpy())))
    assert cache.status() == 0


def test_unaligned_arrays_refused(m):
    """positions, lengths and page tables off their 4 bytes are refused by every call"""
    c = Case(m, [1, 1], [40, 50], 1, 64, 16)
    x = rand(1, 2, 4, 64).cuda()
    q, k = rows(m, x), rows(m, x[:, :1])
    out = rows(m, torch.empty_like(x))
    ws = torch.empty(max(16, c.cache.workspace_bytes(c.batch, 4)), dtype=torch.uint8, device="cuda")
    pos, r = cuda_i32([1, 2, 3]), m.Rope(64, 1e4, 100)

    def no(fn, *a, **kw):
        with pytest.raises(m.MoeError) as e:
            fn(*a, stream=LEGACY, **kw)
        assert e.value.code == -1

    for field in ("q_start", "kv_len", "page_table"):
        b = type(c.batch).from_buffer_copy(c.batch)
        setattr(b, field, getattr(b, field) + 2)
        no(c.cache.attention, b, q, out, 0.1, workspace=ws.data_ptr(), workspace_bytes=ws.numel())
        no(c.cache.append, b, k, k)
        no(c.cache.gather, b, k)
    no(c.cache.append, c.batch, k, k, rope=r, pos=pos.data_ptr() + 1)
    no(r.forward, 2, 64, pos.data_ptr() + 2, q, out)
    assert c.cache.status() == 0 and r.status() == 0
