"""The 8-bit cache's oracle against torch's own casts, brute force and the
bounds that its definition gives; the library's and the wrappers' refusals
(nothing here needs a GPU)."""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

from conftest import ROOT

import _kvdec as K
import paged8_kernel as P8
from oracle import paged8_oracle as O

FAKE = ctypes.c_void_p(0x1000)   # never dereferenced: every call is refused before a launch


def _empty(num_pages, KVH, ps, block, D=16):
    c = {n + "_pages": np.zeros((num_pages, KVH, ps, D), np.uint8) for n in "kv"}
    c.update({n + "_scales": np.ones((num_pages, KVH, ps // block), np.float32) for n in "kv"})
    return c


def test_e4m3_codes_are_torchs():
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(O.e4m3_table().astype(np.float32), table, equal_nan=True)
    x = np.concatenate([np.random.default_rng(0).uniform(-448, 448, 4000),
                        np.random.default_rng(1).standard_normal(4000) * 0.01,
                        (table[:127][:, None] + np.array([0, 2**-11, 2**-7, 0.125, 8.0])).ravel().clip(-448, 448)])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.encode(x, "e4m3"), want)
    mid = (table[1:127] + table[:126]) / 2   # ties
    want = torch.from_numpy(mid).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.encode(mid, "e4m3"), want)
    assert list(O.encode([np.nan, np.inf, -np.inf], "e4m3")) == [O.NAN_CODE] * 3


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_scale_is_the_least_that_fits(code):
    rng = np.random.default_rng(3)
    for amax in list(np.exp2(rng.uniform(-90, 120, 300))) + [O.TOP[code], O.TOP[code] * (1 + 2**-20), 1.0, 3e38]:
        s = float(O.need_scale(amax, code))
        assert amax <= s * O.TOP[code] and amax > s / 2 * O.TOP[code]
        assert np.frexp(s)[0] == 0.5
    assert O.need_scale(0.0, code) == np.float32(2.0**-100) == O.need_scale(1e-40, code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_growing_block_loses_less_than_a_step(code):
    """Tokens of growing size, one call each: every token's value stays within
    one step of the block's final scale (int8), or of its own size (e4m3: half
    a step of 2^-3 from the rounding, and the subnormals' 2^-9 of the scale)."""
    rng = np.random.default_rng(5)
    cache, table = _empty(1, 1, 16, 16), np.zeros((1, 1), np.int32)
    rows = []
    for i in range(16):
        x = rng.standard_normal((1, 1, 16)) * 2.0**(i * 0.7)
        rows.append(x[0, 0])
        cache = O.write(cache, x, x, table, [i + 1], None, code, "HND")
    s = float(cache["k_scales"][0, 0, 0])
    got = O.read(cache, table, [16], [0, 16], 16, code, "HND")[0][:, 0]
    for x, y in zip(rows, got):
        step = s if code == "int8" else np.maximum(np.abs(x) * 2**-4, s * 2**-9)
        assert (np.abs(x - y) < step * (1 + 1e-9)).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_whole_equals_blockwise(code):
    """A prompt in one call, and split at block boundaries: the same cache; and
    attention over it is brute force over the values read back."""
    rng = np.random.default_rng(7)
    B, KVH, ps, block = 2, 2, 32, 16
    table = np.array([[3, 0, 5], [1, 4, 2]], np.int32)
    lens = [50, 77]
    x = [rng.standard_normal((n, KVH, 16)) for n in lens]
    cu = np.cumsum([0] + lens)
    one = O.write(_empty(6, KVH, ps, block), np.concatenate(x), np.concatenate(x), table, lens, cu, code, "HND")
    two = _empty(6, KVH, ps, block)
    for lo, hi in ((0, 32), (32, 48), (48, 80)):
        part = [a[lo:hi] for a in x]
        y = np.concatenate(part)
        two = O.write(two, y, y, table, [min(hi, n) for n in lens], np.cumsum([0] + [len(p) for p in part]), code, "HND")
    assert all(np.array_equal(one[n], two[n]) for n in one)
    kk, vv = O.read(one, table, lens, cu, sum(lens), code, "HND")
    # a row is within half a step of what was written
    assert np.abs(kk - np.concatenate(x)).max() < 4.5 * 2**-4
    q = rng.standard_normal((2, 4, 16))
    o = O.attention(q, one, table, lens, None, 0.25, code, "HND", window=20, sink=3)
    for b in range(B):
        seen = np.r_[0:3, lens[b] - 20:lens[b]]
        rows = np.arange(cu[b], cu[b + 1])[seen]
        for h in range(4):
            w = np.exp(kk[rows, h // 2] @ q[b, h] * 0.25)
            assert np.allclose(o[b, h], w @ vv[rows, h // 2] / w.sum(), atol=1e-12)


# -- refusals -------------------------------------------------------------------

def test_header_and_binding_agree():
    text = open(os.path.join(ROOT, "include", "kvdec_paged8.h")).read()
    names = sorted(set(re.findall(r"^\s*(?:int|size_t)\s+(kvdec_\w+)\s*\(", text, re.M)))
    assert names == sorted(K.PAGED8_SIGNATURES)
    lib = ctypes.CDLL(K.LIB_PATH)
    assert all(hasattr(lib, n) for n in names)


def _c(**kw):
    a = dict(k_pages=0x1000, v_pages=0x1000, k_scales=0x1000, v_scales=0x1000, block_table=0x1000, seq_lens=0x1000,
             num_pages=10, page_stride=65536, row_stride=1024, head_stride=128, code=K.E4M3, KVH=8, D=128,
             page_size=64, block_size=32, max_blocks=4)
    a.update(kw)
    return K.Paged8Cache(**a)


def _write(c, k=FAKE, v=FAKE, dtype=K.F16, st=(1024, 128, 1024, 128), cu=None, B=4, T=4):
    return K.lib.kvdec_paged8_write(None if c is None else ctypes.byref(c), k, v, dtype, *st, cu, B, T, None)


def _read(c, k=FAKE, v=FAKE, dtype=K.F16, cu=None, B=4, T=4):
    return K.lib.kvdec_paged8_read(ctypes.byref(c), cu, B, T, k, v, dtype, None)


def _attend(c, q=FAKE, o=FAKE, dtype=K.F16, st=(8192, 128), cu=None, B=4, T=4, H=64, window=0, sink=0, ws=FAKE,
            nbytes=1 << 30):
    return K.lib.kvdec_paged8_attention(ctypes.byref(c), q, o, dtype, *st, cu, B, T, H, window, sink, 0.1, ws, nbytes,
                                        None)


NULL, SHAPE, DTYPE, GROUP, WORKSPACE, WINDOW, UNSUPPORTED = -1, -2, -3, -4, -6, -7, -10


@pytest.mark.parametrize("change, rc", [
    (dict(k_pages=None), NULL), (dict(v_pages=None), NULL), (dict(k_scales=None), NULL), (dict(v_scales=None), NULL),
    (dict(block_table=None), NULL), (dict(seq_lens=None), NULL), (dict(code=K.F16), DTYPE), (dict(code=5), DTYPE),
    (dict(D=64), SHAPE), (dict(KVH=0), SHAPE), (dict(num_pages=0), SHAPE), (dict(max_blocks=0), SHAPE),
    (dict(page_size=48), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED), (dict(block_size=8), GROUP),
    (dict(block_size=128), GROUP), (dict(block_size=48), GROUP), (dict(max_blocks=1 << 24), SHAPE),
    (dict(row_stride=1 << 27), SHAPE), (dict(page_stride=-16), SHAPE), (dict(head_stride=120), UNSUPPORTED),
    (dict(k_pages=0x1008), UNSUPPORTED), (dict(v_pages=0x1001), UNSUPPORTED)])
def test_bad_caches(change, rc):
    c = _c(**change)
    assert _write(c) == rc
    assert _read(c) == rc
    assert _attend(c, H=64 if c.KVH else 64) == rc


def test_bad_calls():
    c = _c()
    assert _write(None) == NULL
    assert _write(c, k=None) == NULL and _write(c, v=None) == NULL
    assert _write(c, dtype=K.E4M3) == DTYPE
    assert _write(c, T=5) == SHAPE           # one token a sequence, without offsets
    assert _write(c, B=0, T=0) == SHAPE
    assert _write(c, T=1 << 30, cu=FAKE) == SHAPE
    assert _write(c, k=ctypes.c_void_p(0x1002)) == UNSUPPORTED
    assert _write(c, st=(1024, 128, 1024, 132)) == UNSUPPORTED
    assert _write(c, dtype=K.F32, st=(1024, 130, 1024, 128)) == UNSUPPORTED
    assert _read(c, k=None) == NULL and _read(c, v=None) == NULL
    assert _read(c, dtype=9) == DTYPE
    assert _read(c, T=5) == SHAPE
    assert _read(c, v=ctypes.c_void_p(0x1004)) == UNSUPPORTED
    assert _attend(c, q=None) == NULL and _attend(c, o=None) == NULL
    assert _attend(c, dtype=K.F32) == DTYPE
    assert _attend(c, H=60) == SHAPE and _attend(c, H=0) == SHAPE
    assert _attend(c, T=5) == SHAPE
    assert _attend(c, window=-1) == WINDOW and _attend(c, window=4, sink=-1) == WINDOW
    assert _attend(c, sink=4) == WINDOW      # a sink is a window's
    assert _attend(c, st=(8190, 128)) == UNSUPPORTED
    assert _attend(c, ws=None) == WORKSPACE and _attend(c, nbytes=16) == WORKSPACE
    assert _attend(c, ws=ctypes.c_void_p(0x1008)) == WORKSPACE


def test_workspace_bytes():
    f = K.lib.kvdec_paged8_workspace_bytes
    assert f(0, 1, 64, 8, 100) == 0 == f(1, 0, 64, 8, 100) == f(1, 1, 60, 8, 100) == f(1, 1, 64, 8, 0)
    assert f(1, 1, 64, 8, 1 << 30) == 0
    # bounded whatever the batch, the new tokens and the lengths
    for B, T, H, KVH, n in ((1, 1, 8, 8, 16), (32, 32, 64, 8, 163840), (1, 2048, 64, 8, 8192), (8, 40, 64, 8, 4096),
                            (1, 1, 64, 1, 1 << 20), (1 << 20, 1 << 20, 64, 8, (1 << 30) - 1)):
        assert 0 < f(B, T, H, KVH, n) < 1 << 28


def test_wrappers_refuse():
    cache = P8.new_paged8_cache(4, n_kv_heads=2, page_size=32, block_size=16, device="cpu")
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="must live on the GPU"):
        P8.write_paged8_cache(x, x, *cache, table, lens)
    with pytest.raises(ValueError, match="must live on the GPU"):
        P8.read_paged8_cache(*cache, table, lens)
    with pytest.raises(ValueError, match="must live on the GPU"):
        P8.paged8_attention(x, *cache, table, lens)
    with pytest.raises(ValueError, match="kv_layout"):
        P8.paged8_attention(x, *cache, table, lens, kv_layout="DHN")
    for bad in (dict(page_size=24), dict(block_size=8), dict(block_size=64, page_size=32), dict(dtype=torch.float16),
                dict(kv_layout="HDN")):
        with pytest.raises(ValueError):
            P8.new_paged8_cache(4, device="cpu", **bad)
    k, v, ks, vs = P8.new_paged8_cache(3, n_kv_heads=2, page_size=64, block_size=16, dtype=torch.int8,
                                       kv_layout="HND", device="cpu")
    assert k.shape == v.shape == (3, 2, 64, 128) and k.dtype == torch.int8
    assert ks.shape == vs.shape == (3, 2, 4) and bool((ks == 1).all())
