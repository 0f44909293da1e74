"""The paged 8-bit cache on the GPU vs the CPU oracle: written codes and scales
bit for bit, rows read back exactly, attention within one rounding of the
output."""

import numpy as np
import pytest
import torch

from helpers import SCALE, say
from oracle import paged8_oracle as O

pytestmark = pytest.mark.gpu

D = 128
TORCH_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NAMES = ("k_pages", "v_pages", "k_scales", "v_scales")


def make_cache(rng, num_pages, KVH, ps, block, code, layout, spread=1.0, k_far=True):
    """A cache of quantized noise whose blocks differ in magnitude (numpy)."""
    c = {}
    for n in "kv":
        x = rng.standard_normal((num_pages, KVH, ps // block, block, D))
        if n == "k" and k_far:
            x[..., rng.permutation(D)[:3]] *= 6
        x *= np.exp2(spread * rng.standard_normal(x.shape[:3]))[..., None, None]
        s = np.vectorize(lambda a: O.need_scale(a, code), otypes=[np.float32])(np.abs(x).max((3, 4)))
        codes = O.encode(x / s[..., None, None].astype(np.float64), code).reshape(num_pages, KVH, ps, D)
        c[n + "_pages"] = codes if layout == "HND" else np.ascontiguousarray(codes.swapaxes(1, 2))
        c[n + "_scales"] = s
    return c


def put(c, code, device):
    return tuple(torch.from_numpy(np.ascontiguousarray(c[n])).to(device).view(TORCH_CODE[code])
                 if n.endswith("pages") else torch.from_numpy(c[n].copy()).to(device) for n in NAMES)


def take(cache):
    return {n: (t.view(torch.uint8) if n.endswith("pages") else t).cpu().numpy() for n, t in zip(NAMES, cache)}


def make_table(rng, lens, ps, num_pages, extra=1):
    """Distinct random pages for every sequence, -1 behind them."""
    blocks = [-(-max(n, 0) // ps) for n in lens]
    table = np.full((len(lens), max(blocks + [1]) + extra), -1, np.int32)
    perm = rng.permutation(num_pages)
    assert sum(blocks) <= num_pages
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = perm[at:at + n]
        at += n
    return table


def i32(x, device):
    return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


def rows_of(rng, T, KVH, dtype, scale=1.0):
    return (torch.from_numpy(rng.standard_normal((T, KVH, D)).astype(np.float32)) * scale).to(DT[dtype])


def same_cache(got, want, what=""):
    for n in NAMES:
        a, b = got[n], want[n]
        if n.endswith("pages"):
            bad = np.argwhere(a != b)
        else:
            bad = np.argwhere(~((a == b) | (np.isnan(a) & np.isnan(b))))
        assert len(bad) == 0, f"{what} {n}: {len(bad)} differ, first at {bad[0]}: {a[tuple(bad[0])]} {b[tuple(bad[0])]}"


def check_out(o, ref, dtype, vmax, single=False):
    """Each output within half a step of its type of the 64-bit result, plus
    what the arithmetic before that rounding may add: logits of 128 fp32 terms
    (under 2^-13 of a weight's size for the logits here: 128 * 2^-24 of their
    absolute sum of at most 16) move weights by at most 2.5e-5 of their sum, and
    so the output by twice that of the largest |v|; `single`: many query rows,
    whose weights are rounded to fp16 once (2^-11 of each)."""
    o, ref = o.double().cpu().numpy(), np.asarray(ref)
    assert np.array_equal(np.isnan(o), np.isnan(ref))
    o, ref = np.nan_to_num(o), np.nan_to_num(ref)
    # half a step at the larger of the two magnitudes
    top = np.maximum(np.abs(o), np.abs(ref))
    half = np.maximum(top * torch.finfo(DT[dtype]).eps / 2, 2.0**-25)
    slack = 5e-5 * max(1.0, vmax) + (2.0**-11 * vmax if single else 0.0)
    worst = (np.abs(o - ref) - half).max(initial=-1.0)
    assert worst <= slack, f"{worst:.3g} beyond half a step, slack {slack:.3g}"


def vmax_of(c, code):
    s = c["v_scales"][np.isfinite(c["v_scales"])].max()
    return float(s) * O.TOP[code]


# -- writing and reading -----------------------------------------------------------

# (lengths after the write, new tokens): from nothing, mid-block starts, block and
# page edges, sequences without new tokens, more new tokens than length
RAGGED = ([40, 17, 96, 5, 33, 0, 64, 200, 31, 10], [40, 3, 32, 0, 1, 0, 47, 130, 16, 12])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, layout, ps, block", [
    ("fp16", "NHD", 16, 16), ("bf16", "HND", 32, 16), ("fp32", "NHD", 32, 32), ("bf16", "NHD", 64, 32),
    ("fp16", "HND", 64, 64), ("fp32", "HND", 128, 128), ("bf16", "NHD", 256, 128), ("fp16", "NHD", 128, 64)])
def test_write_and_read(code, dtype, layout, ps, block, device):
    from paged8_kernel import read_paged8_cache, write_paged8_cache
    rng = np.random.default_rng(ps + block)
    lens, new = RAGGED
    KVH, T = 3, sum(new) + 4   # 4 rows of no sequence
    c = make_cache(rng, 40, KVH, ps, block, code, layout, spread=2.0)
    table = make_table(rng, lens, ps, 40)
    cu = np.cumsum([0] + new)
    k, v = rows_of(rng, T, KVH, dtype, 3.0), rows_of(rng, T, KVH, dtype)
    want = O.write(c, k.double().numpy(), v.double().numpy(), table, lens, cu, code, layout)
    cache = put(c, code, device)
    say(f"write {code} {dtype} {layout} page {ps} block {block}")
    write_paged8_cache(k.to(device), v.to(device), *cache, i32(table, device), i32(lens, device), i32(cu, device),
                       kv_layout=layout)
    torch.cuda.synchronize()
    same_cache(take(cache), want, "write")
    for out in ("fp16", "bf16", "fp32"):
        gk, gv = read_paged8_cache(*cache, i32(table, device), i32(lens, device), i32(cu, device), num_tokens=T,
                                   dtype=DT[out], kv_layout=layout)
        for got, ref in zip((gk, gv), O.read(want, table, lens, cu, T, code, layout)):
            assert torch.equal(got.cpu(), torch.from_numpy(ref).float().to(DT[out]))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [16, 64, 128])
def test_token_steps_grow_the_scale(code, block, device):
    """One token a call; magnitudes rise and fall, so scales grow inside a block
    and start anew with the next."""
    from paged8_kernel import read_paged8_cache, write_paged8_cache
    rng = np.random.default_rng(block)
    B, KVH, ps, start = 3, 2, 128, [0, 13, 120]
    c = make_cache(rng, 8, KVH, ps, block, code, "NHD")
    table = make_table(rng, [256] * B, ps, 8)
    cache, tab = put(c, code, device), i32(table, device)
    for i in range(24):
        size = 2.0**((i * 5) % 9 - 4)
        k, v = rows_of(rng, B, KVH, "bf16", size), rows_of(rng, B, KVH, "bf16", 1 / size)
        lens = [s + i + 1 for s in start]
        c = O.write(c, k.double().numpy(), v.double().numpy(), table, lens, None, code)
        write_paged8_cache(k.to(device), v.to(device), *cache, tab, i32(lens, device))
        torch.cuda.synchronize()
        same_cache(take(cache), c, f"step {i}")
    gk, gv = read_paged8_cache(*cache, tab, i32(lens, device))
    for got, ref in zip((gk, gv), O.read(c, table, lens, None, B, code)):
        assert torch.equal(got.cpu(), torch.from_numpy(ref).float().to(torch.float16))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_extremes(code, device):
    """Zeros, fp32's smallest and largest values, infinities and NaN: in a block
    of their own, behind earlier tokens, and written over."""
    from paged8_kernel import write_paged8_cache
    rng = np.random.default_rng(9)
    KVH, ps, block = 1, 32, 16
    c = make_cache(rng, 8, KVH, ps, block, code, "NHD")
    lens = [32, 20, 32, 7, 18, 9]
    new = [32, 7, 16, 7, 2, 1]
    table, cu = make_table(rng, [32] * 6, ps, 8), np.cumsum([0] + new)
    x = rng.standard_normal((sum(new), KVH, D)).astype(np.float32)
    x[0:16] = 0
    x[16:32] *= 1e-41
    x[33, 0, 5] = np.inf
    x[36, 0, 7] = -np.inf
    x[39:55] *= 8e37
    x[56, 0, 0] = np.nan
    x[62, 0, 127] = -np.nan
    want = O.write(c, x, -x, table, lens, cu, code)
    cache = put(c, code, device)
    t, args = torch.from_numpy(x).to(device), (i32(table, device), i32(lens, device), i32(cu, device))
    say(f"extremes {code}")
    write_paged8_cache(t, -t, *cache, *args)
    torch.cuda.synchronize()
    same_cache(take(cache), want, "first")
    # again, later tokens in the marked blocks, then from their first tokens
    for first, more in ((0, 1), (1, 3)):
        lens2 = [min(n + more, 32) for n in lens]
        new2 = [b - a for a, b in zip(lens, lens2)] if first == 0 else lens2
        cu2 = np.cumsum([0] + new2)
        y = rng.standard_normal((sum(new2), KVH, D)).astype(np.float32)
        want = O.write(want, y, y, table, lens2, cu2, code)
        t = torch.from_numpy(y).to(device)
        write_paged8_cache(t, t, *cache, i32(table, device), i32(lens2, device), i32(cu2, device))
        torch.cuda.synchronize()
        same_cache(take(cache), want, f"again {first}")


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_scales_that_are_no_power_of_two(code, device):
    """Another program's scales: the quotients are then fl32(x / scale)."""
    from paged8_kernel import write_paged8_cache
    rng = np.random.default_rng(10)
    c = make_cache(rng, 4, 2, 16, 16, code, "HND")
    for n in ("k_scales", "v_scales"):
        c[n] = (c[n] * rng.uniform(1, 2, c[n].shape)).astype(np.float32)
    table = make_table(rng, [16, 16], 16, 4)
    x = rows_of(rng, 2, 2, "fp32", 0.3)
    cache = put(c, code, device)
    write_paged8_cache(x.to(device), x.to(device), *cache, i32(table, device), i32([9, 16], device), kv_layout="HND")
    torch.cuda.synchronize()
    got = take(cache)
    for b, row in enumerate((8, 15)):
        p = table[b, 0]
        for h in range(2):
            s = got["k_scales"][p, h, 0]
            assert s >= c["k_scales"][p, h, 0]
            q = (x[b, h].numpy() / s).astype(np.float32)
            assert np.array_equal(got["k_pages"][p, h, row], O.encode(q, code))


@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_write_without_pages(layout, device):
    """Bad page ids, positions past the table and below 0, lengths past the
    table, offsets out of order: their rows are dropped, and read as zeros."""
    from paged8_kernel import read_paged8_cache, write_paged8_cache
    rng = np.random.default_rng(11)
    KVH, ps, block, N = 2, 16, 16, 9
    c = make_cache(rng, N, KVH, ps, block, "int8", layout)
    table = np.array([[0, N, 1], [-1, 2, 3], [4, 5, -7], [6, 7, 2**31 - 1], [8, -1, -1]], np.int32)
    lens, new = [48, 40, 60, 1000, 5], [48, 40, 20, 48, 9]
    cu = np.cumsum([0] + new)
    T = int(cu[-1]) + 3
    k, v = rows_of(rng, T, KVH, "fp16"), rows_of(rng, T, KVH, "fp16")
    want = O.write(c, k.double().numpy(), v.double().numpy(), table, lens, cu, "int8", layout)
    cache = put(c, "int8", device)
    say("write without pages")
    args = (i32(table, device), i32(lens, device), i32(cu, device))
    write_paged8_cache(k.to(device), v.to(device), *cache, *args, kv_layout=layout)
    torch.cuda.synchronize()
    same_cache(take(cache), want)
    gk, gv = read_paged8_cache(*cache, *args, num_tokens=T, kv_layout=layout)
    for got, ref in zip((gk, gv), O.read(want, table, lens, cu, T, "int8", layout)):
        assert torch.equal(got.cpu(), torch.from_numpy(ref).float().to(torch.float16))
    # offsets in no order name no rows for certain, and harm nothing
    bad = i32([7, 90, 3, 2**31 - 1, -5, 40], device)
    write_paged8_cache(k.to(device), v.to(device), *cache, args[0], args[1], bad, kv_layout=layout)
    read_paged8_cache(*cache, args[0], args[1], bad, num_tokens=T, kv_layout=layout)
    torch.cuda.synchronize()


def test_strided_and_unaligned_rows(device):
    """Views of a fused projection are read in place; rows off 16-byte
    boundaries are copied first.  The cache may be a strided view too."""
    from paged8_kernel import paged8_attention, read_paged8_cache, write_paged8_cache
    rng = np.random.default_rng(12)
    B, H, KVH, ps = 4, 8, 2, 32
    lens = [5, 33, 64, 20]
    c = make_cache(rng, 8, KVH, ps, 16, "e4m3", "NHD")
    table = make_table(rng, lens, ps, 8)
    qkv = torch.from_numpy(rng.standard_normal((B, H + 2 * KVH, D)).astype(np.float32)).half().to(device)
    q, k, v = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
    assert not k.is_contiguous()
    want = O.write(c, k.double().cpu().numpy(), v.double().cpu().numpy(), table, lens, None, "e4m3")
    ref = O.attention(q.double().cpu().numpy(), want, table, lens, None, SCALE, "e4m3")
    tab, n = i32(table, device), i32(lens, device)
    odd = torch.zeros(B * (H + 2 * KVH) * D + 1, dtype=torch.float16, device=device)
    odd[1:] = qkv.flatten()
    o2 = odd[1:].view_as(qkv)
    wide = [torch.zeros(8, ps, KVH, 256, dtype=torch.uint8, device=device) for _ in range(2)]
    for step, (qq, kk, vv) in enumerate(((q, k, v), (o2[:, :H], o2[:, H:H + KVH], o2[:, H + KVH:]))):
        cache = put(c, "e4m3", device)
        if step:   # pages that are a slice of a wider tensor
            for w, p in zip(wide, cache):
                w[..., 16:144] = p.view(torch.uint8)
            cache = tuple(w.view(torch.float8_e4m3fn)[..., 16:144] for w in wide) + cache[2:]
        write_paged8_cache(kk, vv, *cache, tab, n)
        torch.cuda.synchronize()
        same_cache(take(cache), want)
        check_out(paged8_attention(qq, *cache, tab, n), ref, "fp16", vmax_of(want, "e4m3"))
        got = read_paged8_cache(*cache, tab, n, dtype=torch.float32)
        for a, b in zip(got, O.read(want, table, lens, None, B, "e4m3")):
            assert torch.equal(a.cpu(), torch.from_numpy(b).float())
    assert all(bool((w[..., :16] == 0).all()) and bool((w[..., 144:] == 0).all()) for w in wide)


# -- attention ---------------------------------------------------------------------

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, layout, ps, block, H, KVH", [
    ("fp16", "NHD", 16, 16, 8, 1), ("bf16", "HND", 32, 32, 4, 4), ("fp16", "HND", 64, 16, 6, 2),
    ("bf16", "NHD", 128, 128, 16, 1), ("fp16", "NHD", 64, 64, 20, 1), ("bf16", "NHD", 16, 16, 33, 1),
    ("fp16", "HND", 32, 16, 16, 2), ("bf16", "NHD", 64, 32, 64, 1)])
def test_attend_one_token(code, dtype, layout, ps, block, H, KVH, device):
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(H * 10 + KVH)
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 200, 511, 700]
    c = make_cache(rng, sum(-(-n // ps) for n in lens) + 2, KVH, ps, block, code, layout)
    table = make_table(rng, lens, ps, len(c["k_pages"]))
    q = (torch.from_numpy(rng.standard_normal((len(lens), H, D)).astype(np.float32))).to(DT[dtype])
    ref = O.attention(q.double().numpy(), c, table, lens, None, SCALE, code, layout)
    say(f"attend {code} {dtype} {layout} page {ps} block {block} H {H} KVH {KVH}")
    o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32(lens, device), kv_layout=layout)
    torch.cuda.synchronize()
    assert o.dtype == q.dtype and o.shape == q.shape
    assert bool((o[1] == 0).all())
    check_out(o, ref, dtype, vmax_of(c, code), single=H // KVH > 32)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("window, sink", [(None, 0), (1, 0), (7, 4), (40, 4), (64, 33), (300, 1), (33, 1000)])
@pytest.mark.parametrize("many", [False, True])
def test_attend_windows(code, window, sink, many, device):
    """Sink and window, for single tokens and for several: sequences shorter and
    longer than both, windows that end inside tiles and pages."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(20 + sink)
    H, KVH, ps = 12, 4, 16
    lens = [3, 12, 40, 64, 150, 341, 77]
    new = [2, 5, 3, 40, 33, 1, 0] if many else [1] * len(lens)
    c = make_cache(rng, 60, KVH, ps, 16, code, "NHD")
    table = make_table(rng, lens, ps, 60)
    cu = np.cumsum([0] + new) if many else None
    q = torch.from_numpy(rng.standard_normal((sum(new), H, D)).astype(np.float32)).half()
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code, window=window, sink=sink)
    say(f"windows {code} W {window} S {sink} many {many}")
    o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32(lens, device), i32(cu, device),
                         window=window, sink=sink)
    torch.cuda.synchronize()
    check_out(o, ref, "fp16", vmax_of(c, code), single=many)


@pytest.mark.parametrize("code, dtype", [("int8", "bf16"), ("e4m3", "fp16"), ("e4m3", "bf16"), ("int8", "fp16")])
@pytest.mark.parametrize("H, KVH", [(8, 1), (4, 4), (20, 4), (12, 1)])
def test_attend_many_tokens(code, dtype, H, KVH, device):
    """Prompts, chunks, drafts and single tokens in one call; sequences with no
    new tokens, more new tokens than length, and rows of no sequence."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(H)
    lens = [1, 150, 97, 40, 0, 260, 33, 5, 300]
    new = [1, 150, 5, 0, 0, 70, 17, 9, 1]
    T, ps = sum(new) + 5, 32
    c = make_cache(rng, 40, KVH, ps, 32, code, "HND")
    table = make_table(rng, lens, ps, 40)
    cu = np.cumsum([0] + new)
    q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).to(DT[dtype])
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code, "HND")
    say(f"many {code} {dtype} {H} {KVH}")
    o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32(lens, device), i32(cu, device),
                         kv_layout="HND")
    torch.cuda.synchronize()
    assert bool((o[sum(new):] == 0).all()) and bool((o[cu[7]:cu[7] + 4] == 0).all())
    check_out(o, ref, dtype, vmax_of(c, code), single=True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attend_scales_far_apart(code, device):
    """Scales over many powers of two, and ones that are no power of two: each
    output is as exact as its largest contribution."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(31)
    H, KVH, ps = 8, 1, 16
    lens, new = [300, 90, 200], [1, 1, 12]
    c = make_cache(rng, 48, KVH, ps, 16, code, "NHD", spread=0.0)
    c["k_scales"] = (c["k_scales"] * rng.uniform(0.5, 1.5, c["k_scales"].shape)).astype(np.float32)
    c["v_scales"] = np.exp2(rng.uniform(-40, 6, c["v_scales"].shape)).astype(np.float32)
    table, cu = make_table(rng, lens, ps, 48), np.cumsum([0] + new)
    q = torch.from_numpy(rng.standard_normal((sum(new), H, D)).astype(np.float32)).bfloat16()
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code)
    o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32(lens, device), i32(cu, device))
    torch.cuda.synchronize()
    check_out(o, ref, "bf16", vmax_of(c, code), single=True)
    # every block tiny, and every block huge
    for e in (-90, 60):
        c["v_scales"] = np.exp2(rng.integers(e, e + 8, c["v_scales"].shape)).astype(np.float32)
        ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code)
        o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32(lens, device),
                             i32(cu, device))
        back = o.double().cpu().numpy() * 2.0**-e
        top = np.abs(ref).max() * 2.0**-e
        assert np.abs(back - ref * 2.0**-e).max() <= top * (2.0**-8 + 2.0**-11 + 1e-4)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 5])
def test_one_token_outweighs_many(code, new, device):
    """A long cache of equal keys beside one that outweighs each of them by
    2^24.3 and all of them by 200: rounded weights of theirs must not add up to
    an error.  Beside half a step of fp16 under 1 (2^-12) the result, whose values
    are 1 and -1, may be off by
      the weights' steps, 2^-31 of the largest: 2^-32 of each of 50000 at most,
      2^-24 for each sum in fp32 that a wave makes beside the one: of the 25000
      tokens of a wave 32 at a time into the weights' sum and, twice, into the
      product; with several new tokens of 50000, 32 at a time, 16 a product."""
    from paged8_kernel import paged8_attention
    H, KVH, ps, L, B = 8, 1, 64, 100_000, 512     # as many sequences of the same pages as workgroups: long sums
    blocks = -(-L // ps)
    one = {"int8": 1, "e4m3": 0x38}[code]         # the code of 1.0
    kp, vp = np.zeros((blocks, ps, KVH, D), np.uint8), np.full((blocks, ps, KVH, D), one, np.uint8)
    kp[0, 3], vp[0, 3] = one, one | 0x80 if code == "e4m3" else 0xff
    c = dict(k_pages=kp, v_pages=vp, k_scales=np.ones((blocks, KVH, ps // 32), np.float32),
             v_scales=np.ones((blocks, KVH, ps // 32), np.float32))
    table = np.tile(np.arange(blocks, dtype=np.int32), (B, 1))
    q = torch.full((B * new, H, D), 24.3 * np.log(2) / (D * SCALE), dtype=torch.float16)
    x = float(q[0, 0, 0]) * D * SCALE             # the logit of the one
    say(f"one token outweighs many {code} {new}")
    o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32([L] * B, device),
                         i32(new * np.arange(B + 1), device))
    others = np.array([L - new + i for i in range(new)]) * np.exp(-x)
    want = np.tile((others - 1) / (others + 1), B)[:, None, None]
    err = np.abs(o.double().cpu().numpy() - want).max()
    assert err <= 2.0**-12 + 50000 * 2.0**-32 + 3 * (25000 if new == 1 else 50000) / 32 * 2.0**-24, err


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("window", [None, 24])
def test_masked_nan_stays_out(code, window, device):
    """NaN where a row does not look (behind the last token, later tokens,
    tokens that left the window) changes nothing for it; rows that look at one
    are NaN."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(41)
    H, KVH, ps = 4, 2, 32
    lens, new = [100, 61, 75, 64], [1, 20, 36, 1]
    c = make_cache(rng, 16, KVH, ps, 16, code, "HND")
    table, cu = make_table(rng, lens, ps, 16), np.cumsum([0] + new)
    sink = 4 if window else 0
    for b, n in enumerate(lens):   # behind the last token
        p, r = table[b, (n - 1) // ps], (n - 1) % ps + 1
        for x in ("k_pages", "v_pages"):
            c[x][p, :, r:] = O.NAN_CODE if code == "e4m3" else 127
        if code == "int8" and r <= 16:
            c["k_scales"][p, :, 1] = np.nan
            c["v_scales"][p, :, 1] = np.nan
    q = torch.from_numpy(rng.standard_normal((sum(new), H, D)).astype(np.float32)).half()

    def both():
        ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code, "HND", window=window, sink=sink)
        o = paged8_attention(q.to(device), *put(c, code, device), i32(table, device), i32(lens, device),
                             i32(cu, device), window=window, sink=sink, kv_layout="HND")
        return o, ref
    o, ref = both()
    assert not np.isnan(ref).any()
    check_out(o, ref, "fp16", vmax_of(c, code), single=True)
    if code == "e4m3":   # single NaN values: a V channel of one token, a K row
        page, row = table[1, 50 // ps], 50 % ps
        c["v_pages"][page, 0, row, 7] = 0xFF
        c["v_pages"][table[2, 1], 1, 60 % ps, 90] = O.NAN_CODE
        c["k_pages"][table[3, 0], 1, 20, 3] = O.NAN_CODE
        c["v_pages"][table[0, 1], 0, 8, 0] = O.NAN_CODE
    else:                # blocks: tokens 48 .. 63 of sequence 1, 64 .. 79 of sequence 2
        c["v_scales"][table[1, 1], 0, 1] = np.nan
        c["k_scales"][table[2, 2], 1, 0] = np.nan
        c["v_scales"][table[0, 1], 0, 0] = np.nan
    o, ref = both()
    assert np.isnan(ref).any() and not np.isnan(ref).all()
    check_out(o, ref, "fp16", vmax_of(c, code), single=True)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("window", [None, 30])
def test_attend_past_the_table(many, window, device):
    """Lengths past the block table, below 0 and more new tokens than length: keys
    are the table's; bad entries are keys and values of zero."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(57)
    H, KVH, ps = 4, 2, 16
    lens = [70, 48, 1000, 2**31 - 1, -5, 20, 90]
    new = [30, 1, 20, 40, 3, 25, 70] if many else [1] * 7
    c = make_cache(rng, 24, KVH, ps, 16, "int8", "NHD")
    table = rng.permutation(21).reshape(7, 3).astype(np.int32)
    table[1, 1], table[5, 0], table[6, 2] = -1, 24, 2**31 - 1
    cu = np.cumsum([0] + new) if many else None
    q = torch.from_numpy(rng.standard_normal((sum(new), H, D)).astype(np.float32)).half()
    sink = 5 if window else 0
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, "int8", window=window, sink=sink)
    say(f"past the table, many {many} window {window}")
    o = paged8_attention(q.to(device), *put(c, "int8", device), i32(table, device), i32(lens, device), i32(cu, device),
                         window=window, sink=sink)
    torch.cuda.synchronize()
    check_out(o, ref, "fp16", vmax_of(c, "int8"), single=many)


@pytest.mark.parametrize("H, B", [(33, 3), (33, 300), (8, 600)])
@pytest.mark.parametrize("many", [False, True])
def test_attend_short_tables(H, B, many, device):
    """Tables of few tokens, whose rows no workgroups share: groups of more heads
    than the narrow kernel's rows, and of fewer."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(59)
    ps = 16
    lens = [int(n) for n in rng.integers(0, 33, B)]
    new = [int(n) for n in rng.integers(0, 4, B)] if many else [1] * B
    c = make_cache(rng, sum(-(-n // ps) for n in lens) + 1, 1, ps, 16, "int8", "NHD")
    table = make_table(rng, lens, ps, len(c["k_pages"]))
    cu = np.cumsum([0] + new) if many else None
    q = torch.from_numpy(rng.standard_normal((sum(new), H, D)).astype(np.float32)).half()
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, "int8")
    say(f"short tables {H} {B} many {many}")
    o = paged8_attention(q.to(device), *put(c, "int8", device), i32(table, device), i32(lens, device), i32(cu, device))
    torch.cuda.synchronize()
    check_out(o, ref, "fp16", vmax_of(c, "int8"), single=True)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("window, sink", [(2**31 - 1, 0), (2**31 - 40, 3), (2**31, 1), (2**32 + 1, 0), (5, 2**31 - 1),
                                          (5, 2**32 + 3), (2**70, 2**70)])
def test_attend_windows_of_any_size(window, sink, many, device):
    """Windows and sinks at and past the ends of 32 bits, also of sequences with
    more new tokens than length."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(58)
    H, KVH, ps = 4, 2, 16
    lens = [70, 3, 1, 20, 90]
    new = [2, 6, 8, 60, 1] if many else [1] * 5
    c = make_cache(rng, 20, KVH, ps, 16, "e4m3", "NHD")
    table = make_table(rng, lens, ps, 20)
    cu = np.cumsum([0] + new) if many else None
    q = torch.from_numpy(rng.standard_normal((sum(new), H, D)).astype(np.float32)).half()
    # every position is within 100 of the others: so is what the oracle is given
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, "e4m3", window=min(window, 100), sink=min(sink, 100))
    say(f"windows of any size W {window} S {sink} many {many}")
    o = paged8_attention(q.to(device), *put(c, "e4m3", device), i32(table, device), i32(lens, device), i32(cu, device),
                         window=window, sink=sink)
    torch.cuda.synchronize()
    check_out(o, ref, "fp16", vmax_of(c, "e4m3"), single=many)


def test_attend_many_sequences(device):
    """More sequences than a wave has lanes, most of them short or empty."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(51)
    B, H, KVH, ps = 300, 4, 2, 16
    lens = [int(n) for n in rng.integers(0, 40, B)]
    lens[7], lens[130], lens[299] = 900, 333, 512
    c = make_cache(rng, sum(-(-n // ps) for n in lens) + 1, KVH, ps, 16, "int8", "NHD")
    table = make_table(rng, lens, ps, len(c["k_pages"]))
    q = torch.from_numpy(rng.standard_normal((B, H, D)).astype(np.float32)).half()
    ref = O.attention(q.double().numpy(), c, table, lens, None, SCALE, "int8")
    say("many sequences")
    o = paged8_attention(q.to(device), *put(c, "int8", device), i32(table, device), i32(lens, device))
    o2 = paged8_attention(q.to(device), *put(c, "int8", device), i32(table, device), i32(lens, device),
                          i32(np.arange(B + 1), device))
    torch.cuda.synchronize()
    check_out(o, ref, "fp16", vmax_of(c, "int8"))
    check_out(o2, ref, "fp16", vmax_of(c, "int8"))


# sequences, length of the others, (H, KVH), new tokens a sequence (None: one each, no offsets), window, sink
DEALT = [(140, 330, (8, 1), "draft", None, 0),      # three waves' lanes of sequences, 64-row units
         (3, 2500, (8, 2), "draft", None, 0),       # few long ones: many parts each
         (70, 700, (33, 1), None, None, 0),         # one token each, of more rows than the narrow kernel's
         (40, 900, (8, 1), "chunk", None, 0),       # units of 128 and of 64 rows, several a sequence
         (9, 1500, (16, 2), "chunk", 200, 70),
         (20, 300, (8, 8), "chunk", None, 0)]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(DEALT)))
def test_attend_dealt_units(code, case, device):
    """Units too few to fill the GPU, whose tiles are dealt in parts: ragged
    lengths, empty sequences among them, and rows of no sequence."""
    from paged8_kernel import paged8_attention
    B, length, (H, KVH), kind, window, sink = DEALT[case]
    rng = np.random.default_rng(60 + case)
    ps = 16
    lens = [int(n) for n in rng.integers(0, length, B)]
    lens[0], lens[B // 2], lens[-1] = 2 * length, 0, 1
    new = [1] * B
    if kind == "draft":
        new = [int(n) for n in rng.integers(0, 9, B)]
    if kind == "chunk":
        new = [int(n) for n in np.where(rng.random(B) < 0.3, rng.integers(0, 60, B), 1)]
        new[0] = 33
    T = sum(new) + (0 if kind is None else 3)
    c = make_cache(rng, sum(-(-n // ps) for n in lens) + 1, KVH, ps, 16, code, "NHD")
    table, cu = make_table(rng, lens, ps, len(c["k_pages"])), None if kind is None else np.cumsum([0] + new)
    q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).half()
    ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code, window=window, sink=sink)
    say(f"dealt units {code} {DEALT[case]}")
    args = (q.to(device), *put(c, code, device), i32(table, device), i32(lens, device), i32(cu, device))
    o = paged8_attention(*args, window=window, sink=sink)
    again = paged8_attention(*args, window=window, sink=sink)
    torch.cuda.synchronize()
    check_out(o, ref, "fp16", vmax_of(c, code), single=True)
    assert torch.equal(o, again)


def test_pool_past_4_gib(device):
    """Page offsets past 32 bits, in codes and in scales."""
    from paged8_kernel import new_paged8_cache, paged8_attention, read_paged8_cache, write_paged8_cache
    N, KVH, ps = 36000, 8, 128   # 4.7 GB of codes each
    cache = new_paged8_cache(N, KVH, ps, 16, torch.float8_e4m3fn)
    assert cache[0].numel() > 2**32
    rng = np.random.default_rng(61)
    lens = [200, 77]
    table = np.array([[N - 1, 3], [N - 2, -1]], np.int32)
    cu = [0, 200, 277]
    k, v = rows_of(rng, 277, KVH, "bf16"), rows_of(rng, 277, KVH, "bf16")
    args = (i32(table, device), i32(lens, device))
    say("pool past 4 GiB")
    write_paged8_cache(k.to(device), v.to(device), *cache, *args, i32(cu, device))
    q = torch.from_numpy(rng.standard_normal((2, 16, D)).astype(np.float32)).half()
    o = paged8_attention(q.to(device), *cache, *args)
    gk, _ = read_paged8_cache(*cache, *args, i32(cu, device), num_tokens=277, dtype=torch.float32)
    torch.cuda.synchronize()
    small = {n: np.zeros((4, KVH, ps, D), np.uint8) for n in NAMES[:2]}
    small.update({n: np.ones((4, KVH, 8), np.float32) for n in NAMES[2:]})
    t2 = np.array([[0, 1], [2, -1]], np.int32)
    small = O.write(small, k.double().numpy(), v.double().numpy(), t2, lens, cu, "e4m3", "HND")
    assert torch.equal(gk.cpu(), torch.from_numpy(O.read(small, t2, lens, cu, 277, "e4m3", "HND")[0]).float())
    ref = O.attention(q.double().numpy(), small, t2, lens, None, SCALE, "e4m3", "HND")
    check_out(o, ref, "fp16", vmax_of(small, "e4m3"))


# -- together ----------------------------------------------------------------------

@pytest.mark.parametrize("code, dtype", [("e4m3", "bf16"), ("int8", "fp16")])
def test_prompt_then_tokens(code, dtype, device):
    """A serving run: prompts written and attended, then drafts, then tokens,
    each step's attention over what the steps before have written; a graph of
    the token step replayed beside eager calls gives the same bits."""
    from paged8_kernel import new_paged8_cache, paged8_attention, write_paged8_cache
    rng = np.random.default_rng(71)
    B, H, KVH, ps, block = 3, 8, 2, 32, 16
    cache = new_paged8_cache(24, KVH, ps, block, TORCH_CODE[code])
    c = take(cache)
    table = make_table(rng, [160] * B, ps, 24)
    tab = i32(table, device)
    lens = np.zeros(B, int)
    for new in ([40, 17, 64], [5, 3, 4], [1, 1, 1], [1, 0, 1], [1, 1, 1]):
        lens = lens + np.array(new)
        cu, T = np.cumsum([0] + new), sum(new)
        k, v = rows_of(rng, T, KVH, dtype, 2.0), rows_of(rng, T, KVH, dtype)
        q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).to(DT[dtype])
        c = O.write(c, k.double().numpy(), v.double().numpy(), table, lens, cu, code)
        ref = O.attention(q.double().numpy(), c, table, lens, cu, SCALE, code)
        n, off = i32(lens, device), i32(cu, device)
        write_paged8_cache(k.to(device), v.to(device), *cache, tab, n, off)
        o = paged8_attention(q.to(device), *cache, tab, n, off)
        torch.cuda.synchronize()
        same_cache(take(cache), c, f"{new}")
        check_out(o, ref, dtype, vmax_of(c, code), single=True)


def test_graph_replays(device):
    """Two captured graphs of the token step (their own workspaces), replayed in
    turn with other lengths, tables and tokens and eager work in between: each
    replay's bits are the eager call's."""
    from paged8_kernel import new_paged8_cache, paged8_attention, read_paged8_cache, write_paged8_cache
    rng = np.random.default_rng(81)
    B, H, KVH, ps = 4, 16, 2, 32
    made = []
    for _ in range(2):
        cache = new_paged8_cache(40, KVH, ps, 32)
        s = dict(cache=cache, tab=i32(make_table(rng, [300] * B, ps, 40), device), n=i32([1] * B, device),
                 k=torch.zeros(B, KVH, D, dtype=torch.half, device=device))
        s["v"], s["q"] = torch.zeros_like(s["k"]), torch.zeros(B, H, D, dtype=torch.half, device=device)

        def step(s=s):
            write_paged8_cache(s["k"], s["v"], *s["cache"], s["tab"], s["n"])
            return paged8_attention(s["q"], *s["cache"], s["tab"], s["n"])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        s["graph"], s["step"] = torch.cuda.CUDAGraph(), step
        with torch.cuda.graph(s["graph"]):
            s["o"] = step()
        made.append(s)
    for i in range(6):
        for s in made:
            lens = [1 + i, 30 + i, 100 + 31 * i, 0 if i % 2 else 299]
            s["n"].copy_(i32(lens, device))
            for x in ("k", "v", "q"):
                s[x].copy_(torch.from_numpy(rng.standard_normal(s[x].shape).astype(np.float32)))
            before = [t.clone() for t in s["cache"]]
            s["graph"].replay()
            torch.cuda.synchronize()
            got, held = s["o"].clone(), [t.view(torch.uint8).clone() for t in s["cache"]]
            for t, b in zip(s["cache"], before):
                t.view(torch.uint8).copy_(b.view(torch.uint8))
            want = s["step"]()
            torch.cuda.synchronize()
            assert torch.equal(got, want), i
            assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(held, s["cache"]))
            read_paged8_cache(*s["cache"], s["tab"], s["n"])


def test_streams_and_repeats(device):
    """The same bits on every call, also on a side stream while another call
    runs beside it."""
    from paged8_kernel import paged8_attention
    rng = np.random.default_rng(91)
    B, H, KVH, ps = 8, 64, 8, 16
    lens = [int(n) for n in rng.integers(1, 3000, B)]
    c = make_cache(rng, 64, KVH, ps, 16, "e4m3", "NHD")
    table = rng.integers(0, 64, (B, 188)).astype(np.int32)   # pages shared by sequences: reading is fine
    cache, tab, n = put(c, "e4m3", device), i32(table, device), i32(lens, device)
    q = torch.from_numpy(rng.standard_normal((B, H, D)).astype(np.float32)).half().to(device)
    first = paged8_attention(q, *cache, tab, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(paged8_attention(q, *cache, tab, n))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


# -- arguments ---------------------------------------------------------------------

def _calls(device):
    from paged8_kernel import new_paged8_cache
    B, KVH, H, T = 2, 2, 4, 3
    cache = new_paged8_cache(4, KVH, 32, 16, torch.int8)
    return dict(k=torch.zeros(T, KVH, D, dtype=torch.half, device=device),
                v=torch.zeros(T, KVH, D, dtype=torch.half, device=device),
                q=torch.zeros(T, H, D, dtype=torch.half, device=device),
                k_pages=cache[0], v_pages=cache[1], k_scales=cache[2], v_scales=cache[3],
                block_table=torch.zeros(B, 2, dtype=torch.int32, device=device),
                seq_lens=torch.ones(B, dtype=torch.int32, device=device),
                cu_seqlens=torch.tensor([0, 1, 3], dtype=torch.int32, device=device), kv_layout="NHD", window=None,
                sink=0, num_tokens=3, dtype=torch.half)


BAD = {
    "k_pages": [lambda t: t.half(), lambda t: t[..., :64], lambda t: t[0], lambda t: t.cpu(), lambda t: t[:, :24],
                lambda t: t.view(torch.float8_e4m3fn), lambda t: t.transpose(2, 3), lambda t: t[:, ::2]],
    "v_pages": [lambda t: t[:3], lambda t: t.view(torch.float8_e4m3fn)],
    "k_scales": [lambda t: t.half(), lambda t: t[:, :, :1], lambda t: t[:2], lambda t: t.cpu(), lambda t: t[0]],
    "v_scales": [lambda t: t[:, :1], lambda t: t.transpose(1, 2), lambda t: torch.ones(4, 2, 4, device=t.device)],
    "block_table": [lambda t: t.long(), lambda t: t[0], lambda t: t.cpu(), lambda t: t.t()],
    "seq_lens": [lambda t: t.long(), lambda t: t[:1], lambda t: t.cpu()],
    "cu_seqlens": [lambda t: t.long(), lambda t: t[:2], lambda t: t.cpu(), lambda t: None],
    "kv_layout": [lambda t: "DHN", lambda t: None],
}


@pytest.mark.parametrize("name", sorted(BAD))
def test_refusals_of_the_cache(name, device):
    import paged8_kernel as P8
    for change in BAD[name]:
        a = _calls(device)
        a[name] = change(a[name])
        cache = [a[n] for n in (*NAMES, "block_table", "seq_lens", "cu_seqlens")]
        for call in (lambda: P8.write_paged8_cache(a["k"], a["v"], *cache, kv_layout=a["kv_layout"]),
                     lambda: P8.read_paged8_cache(*cache, num_tokens=3, kv_layout=a["kv_layout"]),
                     lambda: P8.paged8_attention(a["q"], *cache, kv_layout=a["kv_layout"])):
            with pytest.raises((ValueError, TypeError)):
                call()


def test_refusals_of_the_rows(device):
    import paged8_kernel as P8
    a = _calls(device)
    cache = [a[n] for n in (*NAMES, "block_table", "seq_lens", "cu_seqlens")]
    k, q = a["k"], a["q"]
    for kk, vv in ((k.long(), k), (k, k.float()), (k[:, :1], k), (k, k[:2]), (k[0], k), (k.cpu(), k.cpu()),
                   (k[..., :64], k[..., :64]), (k.transpose(1, 2), k)):
        with pytest.raises((ValueError, TypeError)):
            P8.write_paged8_cache(kk, vv, *cache)
    for qq in (q.float(), q[:, :3], q[..., :64], q.cpu(), q[0]):
        with pytest.raises((ValueError, TypeError)):
            P8.paged8_attention(qq, *cache)
    for bad in (dict(window=0), dict(window=-3), dict(sink=4), dict(window=4, sink=-1)):
        with pytest.raises(ValueError):
            P8.paged8_attention(q, *cache, **bad)
    for bad in (dict(dtype=torch.int8), dict(num_tokens=-1)):
        with pytest.raises(ValueError):
            P8.read_paged8_cache(*cache, **bad)
    with pytest.raises(ValueError, match="one new token"):
        P8.read_paged8_cache(*cache[:6], num_tokens=5)
    # nothing to do
    P8.write_paged8_cache(k[:0], k[:0], *cache)
    assert P8.paged8_attention(q[:0], *cache).shape == (0, 4, D)
    assert P8.read_paged8_cache(*cache, num_tokens=0)[0].shape == (0, 2, D)
    assert P8.read_paged8_cache(*cache)[0].shape == (3, 2, D)
    none = [*cache[:4], cache[4][:0], cache[5][:0], torch.zeros(1, dtype=torch.int32, device=device)]
    assert bool((P8.paged8_attention(torch.ones_like(q), *none) == 0).all())
    assert bool((P8.read_paged8_cache(*none, num_tokens=2)[1] == 0).all())


def test_fast_path_same_as_checked(device, monkeypatch):
    """The native path and the wrapper's own checks and ctypes make the same
    calls."""
    import _kvdec as K
    import paged8_kernel as P8
    rng = np.random.default_rng(99)
    got = []
    for slow in (False, True):
        if slow:
            monkeypatch.setattr(K, "host", K._Checked())
        rng = np.random.default_rng(99)
        a = _calls(device)
        cache = [a[n] for n in (*NAMES, "block_table", "seq_lens", "cu_seqlens")]
        cache[4] = i32([[0, 1], [2, 3]], device)
        cache[5] = i32([40, 33], device)
        k, q = rows_of(rng, 3, 2, "bf16").to(device), rows_of(rng, 3, 4, "bf16").to(device)
        P8.write_paged8_cache(k, -k, *cache)
        got.append([*(t.view(torch.uint8).clone() for t in cache[:4]), *P8.read_paged8_cache(*cache, num_tokens=3),
                    P8.paged8_attention(q, *cache), P8.paged8_attention(q, *cache, window=9, sink=2)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
