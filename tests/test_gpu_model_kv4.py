"""Whole models over the 4-bit cache (moe_model_set_kv): prefill and decode through
moe_kv_append and moe_kv_attention.

The fp32 cache is the reference; the 4-bit one differs from it by its
rounding, so what is checked is that the two forms of the same computation agree:
a decode step's row equals the prefill's row of the same token over the same
cached rows, a rotated cache equals the one that was filled with the newest rows
alone, graphs equal eager steps, and the fp32 cache gives what it gave before.

Tolerance of two forms: the projections of a prefill and of a decode step agree to
2e-5 of a row's rms (fp16 hi/lo products), so a cached value falls on the other
side of a code's border with probability 2 * 2e-5 rms / step, and is then off by a
step; with a step of 0.27 rms (an eighth of a block's largest of 32 normal values,
2.2 rms) that is 1.5e-4 of the values off by 0.27 rms: sqrt(1.5e-4 * 0.27^2) =
3.3e-3 of the cached keys and of the values, each.  An attention output moves by
about as much for either (a score's spread is 1), sqrt(2) * 3.3e-3 = 4.7e-3, and a
final row by no more: rel-L2 5e-3."""
import threading

import numpy as np
import pytest
import torch

from test_gguf import gguf_module

pytestmark = pytest.mark.gpu

RTOL = 5e-3


def close(got, want, what):
    rel = np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)
    assert rel <= RTOL, f"{what}: rel-L2 {rel:.3g}"


def build(moe, tmp_path, arch, d, context, layers=1, seed=41):
    gg = gguf_module()
    path = str(tmp_path / f"{arch}{d}{context}.gguf")
    if arch == "olmoe":
        gg.write_olmoe(path, layers, d, d // 128, 8, 2, 256, 512, seed=seed, context=context, norm_sd=0.1)
    else:
        gg.write_mixtral(path, layers, d, d // 128, d // 512, 4, 2, 512, 512, seed=seed, context=context, norm_sd=0.1)
    return moe.Model.from_gguf(gg.GGUFReader(path))


@pytest.mark.parametrize("arch,d", [("olmoe", 512), ("olmoe", 2048), ("mixtral", 512), ("mixtral", 2048)])
def test_decode_continues_prefill(moe, tmp_path, arch, d):
    """one layer: the cached rows follow from tokens and positions alone, so the step's row
    and the prefill's last row are the same computation (d 2048: the fused step in a graph)"""
    model = build(moe, tmp_path, arch, d, 256)
    before = model.info()[2]
    tok = np.random.default_rng(1).integers(0, 512, 91)
    f32 = model.prefill(tok)
    model.reset()
    model.set_kv(moe.Q4_0)
    assert model.info()[2] < before
    full = model.prefill(tok)
    assert not np.array_equal(full, f32)
    # 4-bit keys and values: nearer to the fp32 cache's rows than to anything else
    assert np.linalg.norm(full - f32) < 0.25 * np.linalg.norm(f32)
    model.reset()
    model.prefill(tok[:70], rows=False)
    for i in range(70, 91):
        close(model.decode(int(tok[i]), i), full[i], f"row {i}")
    assert model.status() == 0 and model.info()[0] == 91
    # back to fp32: what it gave before
    model.reset()
    model.set_kv(moe.F32)
    assert model.info()[2] == before
    assert np.array_equal(model.prefill(tok), f32)


@pytest.mark.parametrize("context", [64, 200, 65])
def test_rotation(moe, tmp_path, context):
    """a full cache keeps its newest context / 2 rows (kvcache.c:29-55)"""
    model = build(moe, tmp_path, "olmoe", 512, context)
    model.set_kv(moe.Q4_0)
    tok = np.random.default_rng(2).integers(0, 512, context + 3)
    keep = context // 2
    model.prefill(tok[:context], rows=False)
    after = [model.decode(int(t), context - 1) for t in tok[context:]]
    assert model.info()[0] == keep + 3
    model.reset()
    model.prefill(tok[context - keep:context], np.arange(context - keep, context), rows=False)
    for i, t in enumerate(tok[context:]):
        close(model.decode(int(t), context - 1), after[i], f"row {i} after the rotation")
    assert model.status() == 0


def test_generate(moe, tmp_path):
    """greedy generation replays one graph: the picks of eager decode steps, twice alike, across
    a rotation"""
    model = build(moe, tmp_path, "olmoe", 2048, 64, layers=2)
    model.set_kv(moe.Q4_0)
    tok = np.random.default_rng(3).integers(0, 512, 30)
    a = model.generate(tok, 45)
    assert model.mode()["graph"] and model.mode()["fused"]
    model.reset()
    assert np.array_equal(model.generate(tok, 45), a)
    model.reset()
    model.prefill(tok, rows=False)
    got = [int(np.argmax(model.logits(29)))]
    for i in range(20):
        model.decode(got[-1], 30 + i, row=False)
        got.append(int(np.argmax(model.logits(0))))
    assert got == list(a[:21])
    assert model.status() == 0


def test_refusals(moe, tmp_path):
    model = build(moe, tmp_path, "olmoe", 512, 64)
    for bad, code in ((moe.Q8_0, -2), (99, -2)):
        with pytest.raises(moe.MoeError) as e:
            model.set_kv(bad)
        assert e.value.code == code
    model.prefill([1, 2, 3], rows=False)
    with pytest.raises(moe.MoeError) as e:
        model.set_kv(moe.Q4_0)
    assert e.value.code == -1
    model.reset()
    model.set_kv(moe.Q4_0)
    model.set_kv(moe.Q4_0)
    with pytest.raises(moe.MoeError):
        model.prefill(np.arange(65) % 100)
    with pytest.raises(moe.MoeError):
        model.prefill([1], [64])
    model.prefill([1, 2], rows=False)
    assert model.status() == 0 and moe.lib().moe_model_set_kv(None, 0) == -1


def test_set_kv_beside_other_work(moe, tmp_path):
    """the cache's type changed while another thread keeps the legacy stream busy: the calls
    behind it start from what set_kv left, bit for bit"""
    model = build(moe, tmp_path, "olmoe", 2048, 256)
    tok = np.random.default_rng(5).integers(0, 512, 40)

    def calls():
        got = []
        for kind in (moe.Q4_0, moe.F32):
            model.reset()
            model.set_kv(kind)
            got += [model.prefill(tok[:39]), model.decode(int(tok[39]), 39)]
            model.reset()
            model.set_kv(moe.Q4_0 if kind == moe.F32 else moe.F32)
            got.append(model.decode(int(tok[0]), 0))
        assert model.status() == 0
        return got

    quiet = calls()
    stop = threading.Event()

    def work():
        a = torch.randn(2048, 2048, device="cuda", dtype=torch.bfloat16)
        while not stop.is_set():
            for _ in range(20):
                a @ a
            torch.cuda.current_stream().synchronize()

    t = threading.Thread(target=work)
    t.start()
    try:
        for _ in range(4):
            assert all(np.array_equal(x, y) for x, y in zip(calls(), quiet))
    finally:
        stop.set()
        t.join()
